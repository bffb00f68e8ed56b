// Products with 4-bit weights for few rows, and the weights' layout.
//
//     out[t, f] = sum_g s[f, g] sum_{k in g} q[f, k] x[t, k]  (+ bias, + what was there; or silu(.) times a second product)
//
// q is -8 .. 7, g groups of 32 or 64 along K, s a number of five significant bits (q s then has at most eight: it is a bfloat16
// number, so the kernel for many rows multiplies exactly these weights).
//
// Layout (q4.cuh): 128 features x 64 of K are one tile, eight pieces of 16 features one after the other, each piece's codes in the order in
// which the lanes of a warp hold the first operand of mma.sync m16n8k16, then its scales; a warp reads a piece with one 16-byte load a lane and
// the codes go from there into the product without passing through shared memory.
//
// A block of eight warps takes 16 WM features; the warps share out K's tiles, each multiplies its own (codes to bfloat16 by setting
// them below the exponent of 128 and taking 136 away; a group's sum is scaled in float32), and their sums are added in the warps'
// order through shared memory.  Bound by DRAM where there are enough features, by latency otherwise: a block therefore asks for its
// first codes before it waits for the kernel that makes x.
#define CJ_LIB "gemm_q4"
#include "common.cuh"
#include "q4.cuh"

using namespace cj;

namespace {

constexpr int WARPS = 8;

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct Args {
    const __nv_bfloat16* x;
    const uint8_t* w;
    const uint8_t* w_up;
    const float* bias;
    void* out;
    const int* offsets;        // null: one group of all rows
    const int* index;          // null: row s reads row s of x
    long long ldx, ldo;
    int rows, x_rows, features, K, groups, half_out, accumulate;
};

// NTOK: rows of x a block takes at a time; WM: pieces of 16 features a block takes of each weight; HALF: groups of 32; AHEAD: tiles along K whose codes
// a warp has asked for before it multiplies the first
template <int NTOK, int WM, bool GATED, bool HALF, int AHEAD>
__global__ void __launch_bounds__(WARPS * 32, NTOK == 8 && AHEAD == 1 ? 4 : 0) gemm_q4_kernel(const Args a) {
    constexpr int NB = NTOK / 8, W = GATED ? 2 : 1, PIECE = q4::piece_bytes(HALF);
    constexpr int GRP = HALF ? 2 : 1;                      // groups of a tile
    extern __shared__ float red[];                         // [WARPS][W][WM * 16][NTOK + 1]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    const int tiles_k = (a.K + 63) / 64, tiles_f = (a.features + 127) / 128;
    const int piece0 = blockIdx.x * WM;                    // of all pieces of 16 features
    // where this lane's codes and this lane's scales of a piece lie in the first tile along K, of a mixture's first group (pieces past the last tile of
    // features are not there; the last tile's are, filled with zeros)
    const uint8_t* at[W][WM];
#pragma unroll
    for (int i = 0; i < WM; ++i) {
        const int pc = piece0 + i, ft = min(pc >> 3, tiles_f - 1);
        const size_t off = (size_t)ft * tiles_k * q4::tile_bytes(HALF) + (pc & 7) * PIECE;
        at[0][i] = a.w + off;
        if (GATED) at[W - 1][i] = a.w_up + off;
    }
    struct Codes {
        uint4 c[W][WM];
        uint32_t s[W][WM][GRP];
    };
    auto fetch = [&](int kt, Codes& to) {
        if (kt >= tiles_k) return;
        const size_t off = (size_t)kt * q4::tile_bytes(HALF);
#pragma unroll
        for (int i = 0; i < WM; ++i)
#pragma unroll
            for (int u = 0; u < W; ++u) {
                to.c[u][i] = q4::ldg_codes(at[u][i] + off + lane * 16);
#pragma unroll
                for (int h = 0; h < GRP; ++h) to.s[u][i][h] = __ldg((const uint32_t*)(at[u][i] + off + 512 + (h * 8 + g) * 4));
            }
    };
    Codes ring[AHEAD];
    auto fetch_first = [&]() {
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) fetch(warp + d * WARPS, ring[d]);
    };
    // (a group's rows are known only after the wait, and most groups of a few rows' step have none)
    if (!a.offsets) fetch_first();
    cj::after_predecessor();
    cj::release_successor();
    int lo = 0, hi = a.rows;
    if (a.offsets) {
        // The groups that have rows, in their order: this block has the blockIdx.y-th (few rows leave most of 60 experts without one, and blocks
        // that only find that out hold places: experts of 1,408 x 2,048, gated, one row 11.3 us with a block for every group, 7.7 so, eight rows 21.7 and
        // 19.2).  No more groups have rows than there are rows.
        int grp = -1;
        for (int g0 = 0, seen = 0; g0 < a.groups && grp < 0; g0 += 64) {
            int from[2], to[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int idx = g0 + 32 * i + lane;
                from[i] = idx < a.groups ? max(0, a.offsets[idx]) : 0;
                to[i] = idx < a.groups ? min(a.rows, a.offsets[idx + 1]) : 0;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t have = __ballot_sync(0xffffffffu, to[i] > from[i]);
                const uint32_t mine = __ballot_sync(0xffffffffu, to[i] > from[i] && seen + __popc(have & ((1u << lane) - 1)) == (int)blockIdx.y);
                seen += __popc(have);
                if (mine) {
                    const int l = __ffs(mine) - 1;
                    grp = g0 + 32 * i + l;
                    lo = __shfl_sync(0xffffffffu, from[i], l);
                    hi = __shfl_sync(0xffffffffu, to[i], l);
                }
            }
        }
        if (grp < 0) return;
        const size_t off = (size_t)grp * tiles_f * tiles_k * q4::tile_bytes(HALF);
#pragma unroll
        for (int i = 0; i < WM; ++i)
#pragma unroll
            for (int u = 0; u < W; ++u) at[u][i] += off;
    }
    for (int row0 = lo + blockIdx.z * NTOK; row0 < hi; row0 += gridDim.z * NTOK) {
        if (a.offsets || row0 != (int)blockIdx.z * NTOK) fetch_first();
        const __nv_bfloat16* xr[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int s = row0 + n * 8 + g;
            int r = s < hi ? (a.index ? a.index[s] : s) : -1;
            if (r >= a.x_rows) r = -1;
            xr[n] = r >= 0 ? a.x + (size_t)r * a.ldx : nullptr;
        }
        float acc[W][WM][NB][4];
#pragma unroll
        for (int u = 0; u < W; ++u)
#pragma unroll
            for (int i = 0; i < WM; ++i)
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[u][i][n][e] = 0.0f;
        auto fetch_x = [&](int kt, uint2 (&xb)[NB][4]) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int k = kt * 64 + j * 16 + t4 * 4;
                    xb[n][j] = xr[n] && k < a.K ? __ldg((const uint2*)(xr[n] + k)) : make_uint2(0u, 0u);
                }
        };
        uint2 x_next[NB][4];
        fetch_x(warp, x_next);
#pragma unroll 1
        for (int kt0 = warp; kt0 < tiles_k; kt0 += WARPS * AHEAD)
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) {
            const int kt = kt0 + d * WARPS;
            if (kt >= tiles_k) break;
            const Codes now = ring[d];
            uint2 xb[NB][4];
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) xb[n][j] = x_next[n][j];
            fetch(kt + WARPS * AHEAD, ring[d]);
            fetch_x(kt + WARPS, x_next);
#pragma unroll
            for (int u = 0; u < W; ++u)
#pragma unroll
                for (int i = 0; i < WM; ++i) {
                    float part[NB][4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (j % (4 / GRP) == 0) {
#pragma unroll
                            for (int n = 0; n < NB; ++n)
#pragma unroll
                                for (int e = 0; e < 4; ++e) part[n][e] = 0.0f;
                        }
                        const uint32_t wa = j < 2 ? now.c[u][i].x : now.c[u][i].y, wb = j < 2 ? now.c[u][i].z : now.c[u][i].w;
                        uint32_t f[4];
                        f[0] = q4::pair(wa >> (8 * (j & 1)));
                        f[1] = q4::pair(wb >> (8 * (j & 1)));
                        f[2] = q4::pair(wa >> (8 * (j & 1) + 4));
                        f[3] = q4::pair(wb >> (8 * (j & 1) + 4));
#pragma unroll
                        for (int n = 0; n < NB; ++n) mma_bf16(part[n], f, xb[n][j].x, xb[n][j].y);
                        if (j % (4 / GRP) == 4 / GRP - 1) {
                            const uint32_t s = now.s[u][i][j / (4 / GRP)];
                            const float s0 = __uint_as_float(s << 16), s1 = __uint_as_float(s & 0xffff0000u);
#pragma unroll
                            for (int n = 0; n < NB; ++n) {
                                acc[u][i][n][0] = fmaf(part[n][0], s0, acc[u][i][n][0]);
                                acc[u][i][n][1] = fmaf(part[n][1], s0, acc[u][i][n][1]);
                                acc[u][i][n][2] = fmaf(part[n][2], s1, acc[u][i][n][2]);
                                acc[u][i][n][3] = fmaf(part[n][3], s1, acc[u][i][n][3]);
                            }
                        }
                    }
                }
        }
        // ---- the warps' sums: feature i * 16 + g (+ 8), row n * 8 + 2 t4 (+ 1)
        float* mine = red + (size_t)warp * W * WM * 16 * (NTOK + 1);
#pragma unroll
        for (int u = 0; u < W; ++u)
#pragma unroll
            for (int i = 0; i < WM; ++i)
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        mine[((u * WM + i) * 16 + g + 8 * (e >> 1)) * (NTOK + 1) + n * 8 + 2 * t4 + (e & 1)] = acc[u][i][n][e];
        __syncthreads();
        for (int i = threadIdx.x; i < WM * 16 * NTOK; i += WARPS * 32) {
            const int f = i % (WM * 16), n = i / (WM * 16), feature = piece0 * 16 + f, s = row0 + n;
            if (feature >= a.features || s >= hi) continue;
            float y[W];
#pragma unroll
            for (int u = 0; u < W; ++u) {
                y[u] = 0.0f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) y[u] += red[((size_t)(w * W + u) * WM * 16 + f) * (NTOK + 1) + n];
            }
            if (a.bias) y[0] += a.bias[feature];
            const float v = GATED ? gated_act_fast(y[0], y[W - 1], 0.0f, 1.0f, 0.0f) : y[0];
            if (a.half_out) ((__nv_bfloat16*)a.out)[(size_t)s * a.ldo + feature] = __float2bfloat16_rn(v);
            else if (a.accumulate) ((float*)a.out)[(size_t)s * a.ldo + feature] += v;
            else ((float*)a.out)[(size_t)s * a.ldo + feature] = v;
        }
        __syncthreads();
    }
}

// Codes and scales as a quantiser leaves them -> the layout.  One thread a lane of a piece (16 bytes of codes).
__global__ void q4_layout_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales, uint8_t* __restrict__ dst, int features, int K,
                                 int group, int half, long long pieces) {
    const long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const long long pc = idx >> 5;
    if (pc >= pieces) return;
    const int lane = (int)(idx & 31), g = lane >> 2, t4 = lane & 3;
    const int tiles_k = (K + 63) / 64, tiles_f = (features + 127) / 128, groups_k = (K + group - 1) / group;
    const int sub = (int)(pc & 7);
    const long long tile = pc >> 3;
    const int kt = (int)(tile % tiles_k), ft = (int)((tile / tiles_k) % tiles_f);
    const long long grp = tile / tiles_k / tiles_f;
    uint8_t* p = dst + tile * q4::tile_bytes(half != 0) + sub * q4::piece_bytes(half != 0);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int f = ft * 128 + sub * 16 + g + 8 * (i >> 1);
        uint32_t v = 0;
        for (int n = 0; n < 8; ++n) {
            // nibble n: steps 2 (i & 1) and the next; entries 0 .. 3 of each as the pairs that q4::pair takes out together
            const int step = 2 * (i & 1) + ((n >> 1) & 1), e = 2 * (n & 1) + (n >> 2);
            const int k = kt * 64 + step * 16 + t4 * 4 + e;
            const int q = f < features && k < K ? codes[(grp * features + f) * (long long)K + k] : 0;
            v |= (uint32_t)(q + 8) << (4 * n);
        }
        w[i] = v;
    }
    *(uint4*)(p + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    for (int i = lane; i < (half ? 32 : 16); i += 32) {
        const int h = i >> 4, f = ft * 128 + sub * 16 + ((i & 15) >> 1) + 8 * (i & 1), k = kt * 64 + h * 32;
        const float s = f < features && k < K ? scales[(grp * features + f) * (long long)groups_k + k / group] : 0.0f;
        ((__nv_bfloat16*)(p + 512))[i] = __float2bfloat16_rn(s);
    }
}

// A group's scale and codes: s = the smallest number of five significant bits that is at least max |w| / 7, q = w / s rounded to
// the nearest of -8 .. 7 (the even one of two).  A warp a group.
template <typename T>
__global__ void q4_quantise_kernel(const T* __restrict__ w, int8_t* __restrict__ codes, float* __restrict__ scales, long long rows, int K, int group) {
    const int lane = threadIdx.x & 31, groups_k = (K + group - 1) / group;
    const long long idx = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (idx >= rows * groups_k) return;
    const long long row = idx / groups_k;
    const int k0 = (int)(idx % groups_k) * group, n = min(group, K - k0);
    float most = 0.0f;
    bool finite = true;
    for (int i = lane; i < n; i += 32) {
        const float v = fabsf(to_f32(w[row * K + k0 + i]));
        most = fmaxf(most, v);
        finite = finite && v < INFINITY;
    }
    most = warp_max(most);
    // (a group with an entry that is no number has no scale: the caller is told)
    const float s = __all_sync(0xffffffffu, finite) ? q4::scale_up(most / 7.0f) : INFINITY;
    for (int i = lane; i < n; i += 32) {
        const float v = s > 0.0f ? rintf(to_f32(w[row * K + k0 + i]) / s) : 0.0f;
        codes[row * K + k0 + i] = (int8_t)fminf(fmaxf(v, -8.0f), 7.0f);
    }
    if (lane == 0) scales[idx] = s;
}

}  // namespace

// bytes of `groups` weights of [features, K] in the layout; half: groups of 32 along K
CJ_EXPORT long long cj_q4_bytes(int groups, int features, int K, int half) {
    return (long long)groups * ((features + 127) / 128) * ((K + 63) / 64) * q4::tile_bytes(half != 0);
}

// codes int8 [groups, features, K], scales float32 [groups, features, ceil(K / group)] -> dst.  group: 32 (half 1) or a multiple of 64
CJ_EXPORT int cj_q4_layout(const void* codes, const float* scales, void* dst, int groups, int features, int K, int group, cudaStream_t stream) {
    if (!codes || !scales || !dst || groups <= 0 || features <= 0 || K <= 0) return CJ_ERR_ARG;
    if (group != 32 && (group <= 0 || group % 64 != 0)) return CJ_ERR_SIZE;
    const long long pieces = (long long)groups * ((features + 127) / 128) * ((K + 63) / 64) * 8;
    const long long blocks = (pieces * 32 + 255) / 256;
    if (blocks > 0x7fffffffLL) return CJ_ERR_SIZE;
    cj::launch_in_order(q4_layout_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, (const int8_t*)codes, scales, (uint8_t*)dst, features, K,
                        group, group == 32 ? 1 : 0, pieces);
    return launch_status();
}

// w float32 or bf16 [rows, K] -> codes int8 [rows, K], scales float32 [rows, ceil(K / group)]
CJ_EXPORT int cj_q4_quantise(const void* w, int dtype, void* codes, float* scales, long long rows, int K, int group, cudaStream_t stream) {
    if (!w || !codes || !scales || rows <= 0 || K <= 0 || group <= 0) return CJ_ERR_ARG;
    const long long blocks = (rows * ((K + group - 1) / group) * 32 + 255) / 256;
    if (blocks > 0x7fffffffLL) return CJ_ERR_SIZE;
    if (dtype == CJ_F32)
        cj::launch_in_order(q4_quantise_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, stream, (const float*)w, (int8_t*)codes, scales, rows, K, group);
    else if (dtype == CJ_BF16)
        cj::launch_in_order(q4_quantise_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(256), 0, stream, (const __nv_bfloat16*)w, (int8_t*)codes,
                            scales, rows, K, group);
    else return CJ_ERR_DTYPE;
    return launch_status();
}

// x bf16 [x_rows, ldx], w (w_up) in the layout; out float32 or bf16 [rows, ldo].  offsets: null or int32 [groups + 1]; index: null
// or int32 [rows] (an index outside x reads zeros).  K a multiple of four, x and ldx of 8 bytes.  w_up: out = silu(x w) (x w_up).
// n_tok: rows of x a block takes at a time, 8, 16 or 32; ahead: tiles along K whose codes are asked for ahead, 4 or 1 (plain products of eight rows).
CJ_EXPORT int cj_gemm_q4(const void* x, long long ldx, int x_rows, const void* w, const void* w_up, const float* bias, void* out, int out_dtype,
                         long long ldo, int rows, int features, int K, int groups, int half, const int* offsets, const int* index,
                         int accumulate, int n_tok, int ahead, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (!x || !w || !out || features <= 0 || K <= 0 || groups <= 0 || x_rows <= 0) return CJ_ERR_ARG;
    if (out_dtype != CJ_F32 && out_dtype != CJ_BF16) return CJ_ERR_DTYPE;
    if (accumulate && out_dtype != CJ_F32) return CJ_ERR_DTYPE;
    if (w_up && bias) return CJ_ERR_ARG;
    if (!offsets && groups != 1) return CJ_ERR_ARG;
    if ((K & 3) || (ldx & 3) || ((uintptr_t)x & 7) || (((uintptr_t)w | (uintptr_t)w_up) & 15)) return CJ_ERR_ALIGN;
    if (groups > 65535) return CJ_ERR_SIZE;
    const Args a{(const __nv_bfloat16*)x, (const uint8_t*)w, (const uint8_t*)w_up, bias, out, offsets, index, ldx, ldo, rows, x_rows,
                 features, K, groups, out_dtype == CJ_BF16 ? 1 : 0, accumulate};
    const int all = (features + 15) / 16;
    // (the blocks of a group take its rows tile by tile: how many it has is not known here)
    const int row_tiles = offsets ? 1 : min((rows + n_tok - 1) / n_tok, 65535), grid_groups = offsets ? min(groups, rows) : 1;
#define LAUNCH(NTOK, WM, GATED, HALF, AHEAD)                                                                                     \
    {                                                                                                                     \
        constexpr int smem = WARPS * (GATED ? 2 : 1) * WM * 16 * (NTOK + 1) * 4;                                          \
        cudaError_t e = smem <= 48 * 1024 ? cudaSuccess                                                                    \
            : cudaFuncSetAttribute(gemm_q4_kernel<NTOK, WM, GATED, HALF, AHEAD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); \
        if (e != cudaSuccess) return (int)e;                                                                              \
        cj::launch(gemm_q4_kernel<NTOK, WM, GATED, HALF, AHEAD>, dim3((all + WM - 1) / WM, grid_groups, row_tiles), dim3(WARPS * 32), smem, stream, a); \
        return launch_status();                                                                                           \
    }
#define PLAIN(NTOK, WM, AHEAD) { if (half) LAUNCH(NTOK, WM, false, true, AHEAD) else LAUNCH(NTOK, WM, false, false, AHEAD) }
#define GATED(NTOK, WM, AHEAD) { if (half) LAUNCH(NTOK, WM, true, true, AHEAD) else LAUNCH(NTOK, WM, true, false, AHEAD) }
    // rows at a time, pieces of 16 features, tiles ahead
    if (w_up) {
        if (n_tok == 8) GATED(8, 1, 1)
        if (n_tok == 16) GATED(16, 2, 2)
        if (n_tok == 32) GATED(32, 2, 1)
    } else {
        if (n_tok == 8 && ahead == 4) PLAIN(8, 1, 4)
        if (n_tok == 8) PLAIN(8, 1, 1)
        if (n_tok == 16) PLAIN(16, 2, 2)
        if (n_tok == 32) PLAIN(32, 2, 1)
    }
#undef GATED
#undef PLAIN
#undef LAUNCH
    return CJ_ERR_SIZE;
}
