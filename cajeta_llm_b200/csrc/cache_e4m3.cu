// The 8-bit paged cache: keys and values as e4m3 codes with one power of two for each (token, kv head) - appending with the
// rotation on the way, and attention of single rows over it (the prompt form is in attention_e4m3_tc.cu).
//
// A block of tokens that share a scale is one token: an append touches nothing that was written before, and what is cached of a
// prompt does not depend on how it was cut into portions.  The scale is a power of two, held as its exponent + 127 in a byte: a
// code's relative precision (2^-4) does not depend on where in its octave the block's maximum lies, and undoing a power of two is
// exact, so the attention kernels fold it wherever it costs nothing.
#define CJ_LIB "cache_e4m3"
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "e4m3.cuh"

using namespace cj;

namespace {

// ---------------------------------------------------------------------------------------------------------------------------
// Append.  A warp takes a head of q, k or v of a row: HD / 32 neighbouring entries a lane.
//     q, k <- rotated at the row's position p (entry i with i + rot / 2, angle p inv_freq[i]); v as it is
//     e = smallest integer with max |x| <= 448 2^e, within [-100, 119]; code = e4m3(x 2^-e); scale plane: e + 127
// The angle is carried as the rounded product and what the rounding left out (a float32 angle of 30,000 radians is off by up to
// 2^-10, an eighth of a code's step at the block's maximum).  Bound by DRAM for many rows, by the chain load -> rotate ->
// maximum over the warp -> store for few.
// ---------------------------------------------------------------------------------------------------------------------------
template <int HD>
__global__ void __launch_bounds__(256) append_e4m3_kernel(
    const float* __restrict__ qkv, int ld, int q_off, int k_off, int v_off, __nv_bfloat16* __restrict__ q_out, uint8_t* __restrict__ kplane,
    uint8_t* __restrict__ vplane, uint8_t* __restrict__ kexp, uint8_t* __restrict__ vexp, const int* __restrict__ positions,
    const int* __restrict__ row_req, const int* __restrict__ table, int table_rows, int table_stride, int page_tokens, int n_pages,
    int n_heads, int n_kv, int rot, const float* __restrict__ inv_freq, int write_kv) {
    constexpr int VEC = HD / 32;
    __shared__ float cs[HD / 2], sn[HD / 2];
    cj::after_predecessor();
    cj::release_successor();
    const int t = blockIdx.x, lane = threadIdx.x & 31;
    const int pos = positions[t], half = rot >> 1;
    if ((int)threadIdx.x < half) {
        const float p = (float)pos, f = inv_freq[threadIdx.x];
        const float hi = __fmul_rn(p, f), lo = fmaf(p, f, -hi);
        float s, c;
        sincosf(hi, &s, &c);
        cs[threadIdx.x] = fmaf(-lo, s, c);
        sn[threadIdx.x] = fmaf(lo, c, s);
    }
    long long base = -1;                    // row of (page, kv head 0, token) in the planes; -1: no page, nothing is written
    if (write_kv) {
        const int req = row_req[t], at = pos >= 0 ? pos / page_tokens : -1;
        const int page = req >= 0 && req < table_rows && at >= 0 && at < table_stride ? table[(size_t)req * table_stride + at] : -1;
        if (page >= 0 && page < n_pages) base = (long long)page * n_kv * page_tokens + pos % page_tokens;
    }
    __syncthreads();
    const int slots = n_heads + (base >= 0 ? 2 * n_kv : 0);
    const float* row = qkv + (size_t)t * ld;
    const int d0 = lane * VEC;
    for (int slot = blockIdx.y * 8 + (threadIdx.x >> 5); slot < slots; slot += gridDim.y * 8) {
        const int kind = slot < n_heads ? 0 : slot < n_heads + n_kv ? 1 : 2;
        const int h = kind == 0 ? slot : kind == 1 ? slot - n_heads : slot - n_heads - n_kv;
        const float* src = row + (kind == 0 ? q_off : kind == 1 ? k_off : v_off) + h * HD;
        float x[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j += 2) *(float2*)(x + j) = *(const float2*)(src + d0 + j);
        if (kind < 2) {
            if (half % VEC == 0) {
                // all of a lane's entries are of one half: its partners are neighbours too (rot / 2 even: 8-byte loads)
                if (d0 < rot) {
                    const bool low = d0 < half;
                    const int i0 = low ? d0 : d0 - half;
                    float y[VEC];
#pragma unroll
                    for (int j = 0; j < VEC; j += 2) *(float2*)(y + j) = *(const float2*)(src + (low ? d0 + half : i0) + j);
#pragma unroll
                    for (int j = 0; j < VEC; ++j)
                        x[j] = low ? __fsub_rn(__fmul_rn(x[j], cs[i0 + j]), __fmul_rn(y[j], sn[i0 + j]))
                                   : __fadd_rn(__fmul_rn(y[j], sn[i0 + j]), __fmul_rn(x[j], cs[i0 + j]));
                }
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const int d = d0 + j;
                    if (d >= rot) continue;
                    const int i = d < half ? d : d - half;
                    const float y = src[d < half ? d + half : i];
                    x[j] = d < half ? __fsub_rn(__fmul_rn(x[j], cs[i]), __fmul_rn(y, sn[i]))
                                    : __fadd_rn(__fmul_rn(y, sn[i]), __fmul_rn(x[j], cs[i]));
                }
            }
        }
        if (kind == 0) {
            __nv_bfloat162 b[VEC / 2];
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) b[j] = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
            __nv_bfloat16* dst = q_out + ((size_t)t * n_heads + h) * HD + d0;
            if (VEC == 4) *(uint2*)dst = *(uint2*)b;
            else *(uint32_t*)dst = *(uint32_t*)b;
            continue;
        }
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) most = fmaxf(most, fabsf(x[j]));
        const int e = block_exponent(warp_max(most));
        const float down = power_of_two(-e);
        uint32_t code = 0;
#pragma unroll
        for (int j = 0; j < VEC; j += 2)
            code |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[j] * down, x[j + 1] * down), __NV_SATFINITE, __NV_E4M3) << (8 * j);
        const long long at = base + (long long)h * page_tokens;
        uint8_t* dst = (kind == 1 ? kplane : vplane) + at * HD + d0;
        if (VEC == 4) *(uint32_t*)dst = code;
        else *(uint16_t*)dst = (uint16_t)code;
        if (lane == 0) (kind == 1 ? kexp : vexp)[at] = (uint8_t)(e + 127);
    }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Attention of single rows.  A block of four warps takes one row, the query heads of one kv head (up to ROWS at a time) and a
// stretch of the row's keys; each warp walks over its 32-key pieces with a running softmax of its own, codes straight from
// global memory into the registers that the products read (mma.sync m16n8k16, f16 in, float32 out: an e4m3 code is an f16 number
// exactly).  The order of a product's K is free as long as both operands keep it: a lane's share of a key is 32 neighbouring
// bytes, and its share of a value row 16, so every load is 16 bytes and no shared memory lies between.
//     S = q . code_k          rows: heads, columns: keys          s = S scale 2^e_k
//     O = (p 2^(e_v - R)) . code_v   with R the largest exponent of the values so far: the weights stay at most 1 in f16
// Queries come as bfloat16 and are brought to [2^10, 2^11) at their largest entry by a power of two, so that f16 holds all eight
// bits of every entry down to 2^-24 of the largest.  Bound by DRAM: 2 (HD + 1) bytes a key.
// ---------------------------------------------------------------------------------------------------------------------------
constexpr int WARPS = 4;
constexpr int STEP = 32;                   // keys of a warp's step

template <int ROWS>
__device__ __forceinline__ void mma_f16(float (&c)[ROWS == 16 ? 4 : 2], float (&idle)[2], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
    float& c2 = ROWS == 16 ? c[ROWS == 16 ? 2 : 0] : idle[0];
    float& c3 = ROWS == 16 ? c[ROWS == 16 ? 3 : 1] : idle[1];
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c2), "+f"(c3)
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int HD, int ROWS>
__global__ void __launch_bounds__(WARPS * 32, ROWS == 16 ? 2 : 3) decode_e4m3_kernel(
    const __nv_bfloat16* __restrict__ q, __nv_bfloat16* __restrict__ out, const uint8_t* __restrict__ kplane, const uint8_t* __restrict__ vplane,
    const uint8_t* __restrict__ kexp, const uint8_t* __restrict__ vexp, const int* __restrict__ positions, const int* __restrict__ row_req,
    const int* __restrict__ req_start, const int* __restrict__ req_prior, int n_requests, const int* __restrict__ table, int table_stride,
    int page_tokens, int n_pages, int n_heads, int n_kv, int head_batches, int window, float scale_log2, int splits, float* __restrict__ part_acc, float* __restrict__ part_ml) {
    constexpr int NR = ROWS / 8;           // rows of a fragment a lane holds: g, and g + 8
    constexpr int QS = HD / 16;            // steps of 16 of the head's entries
    constexpr int KW = HD / 16;            // words of a key a lane holds
    constexpr int NT = HD / 8;             // column tiles of the output
    cj::after_predecessor();
    cj::release_successor();
    __shared__ float red[WARPS][ROWS][HD + 4];
    __shared__ float sm[WARPS][ROWS], sl[WARPS][ROWS];
    __shared__ int sr[WARPS];
    const int t = blockIdx.x, split = blockIdx.z;
    const int kvh = blockIdx.y / head_batches, hb = blockIdx.y % head_batches;
    const int group = n_heads / n_kv, h0 = kvh * group + hb * ROWS, n_h = min(ROWS, group - hb * ROWS);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    int req, p;
    if (positions) {
        req = row_req[t];
        p = positions[t];
        if (req >= n_requests) req = -1;
    } else {
        // portions: the request whose rows hold this one (none: the row is left alone)
        req = 0;
        while (req < n_requests && t >= req_start[req + 1]) ++req;
        if (req == n_requests || t < req_start[req]) return;
        p = req_prior[req] + t - req_start[req];
    }
    p = req >= 0 ? min(p, table_stride * page_tokens - 1) : -1;
    const int from = window > 0 && p + 1 > window ? p + 1 - window : 0;
    const int n_keys = p - from + 1;
    // equal stretches of whole steps
    const int per = (((n_keys + splits - 1) / splits + STEP - 1) / STEP) * STEP;
    const int first = from + split * per, last = min(p + 1, first + per);
    const int* tab = table + (size_t)max(req, 0) * table_stride;

    uint32_t qa[QS][2 * NR];
    float back[NR];                        // what undoes the queries' power of two, with the scale in units of log 2
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        uint32_t w[2 * QS];
        const int head = g + 8 * r;
#pragma unroll
        for (int i = 0; i < QS / 2; ++i) {
            uint4 u = make_uint4(0u, 0u, 0u, 0u);
            if (head < n_h) u = *(const uint4*)(q + ((size_t)t * n_heads + h0 + head) * HD + t4 * (HD / 4) + i * 8);
            w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
        }
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * QS; ++i) most = fmaxf(most, fmaxf(fabsf(bf16_low(w[i])), fabsf(bf16_high(w[i]))));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = query_exponent(most);
        const float up = power_of_two(e);
        back[r] = scale_log2 * power_of_two(-e);
#pragma unroll
        for (int i = 0; i < QS; ++i) {
            qa[i][r] = pack_f16(bf16_low(w[2 * i]) * up, bf16_high(w[2 * i]) * up);
            qa[i][NR + r] = pack_f16(bf16_low(w[2 * i + 1]) * up, bf16_high(w[2 * i + 1]) * up);
        }
    }

    float o[NT][ROWS == 16 ? 4 : 2], idle[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 2 * NR; ++e) o[i][e] = 0.0f;
    float m[NR], l[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) m[r] = -INFINITY, l[r] = 0.0f;
    int R = -1000;

    for (int k0 = first + warp * STEP; k0 < last; k0 += WARPS * STEP) {
        // lane j looks up key j: its row in the planes (-1: none) and its two exponents
        const int key = k0 + lane;
        int row = -1;
        if (key < last) {
            const int page = tab[key / page_tokens];
            if (page >= 0 && page < n_pages) row = (page * n_kv + kvh) * page_tokens + key % page_tokens;
        }
        uint32_t kw[4][KW];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int at = __shfl_sync(0xffffffffu, row, b * 8 + g);
#pragma unroll
            for (int i = 0; i < KW / 4; ++i) {
                uint4 u = make_uint4(0u, 0u, 0u, 0u);
                if (at >= 0) u = ldg_stream(kplane + (size_t)at * HD + t4 * (HD / 4) + i * 16);
                kw[b][4 * i] = u.x, kw[b][4 * i + 1] = u.y, kw[b][4 * i + 2] = u.z, kw[b][4 * i + 3] = u.w;
            }
        }
        const int ek = row >= 0 ? (int)kexp[row] - 127 : 0, ev = row >= 0 ? (int)vexp[row] - 127 : -1000;
        // the values of this lane's keys: 16 u + {2 t4, 2 t4 + 1, 8 + 2 t4, 9 + 2 t4}, entries [g HD / 8, (g + 1) HD / 8)
        uint32_t vw[2][4][HD / 32];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = __shfl_sync(0xffffffffu, row, u * 16 + (i >> 1) * 8 + 2 * t4 + (i & 1));
                const uint8_t* src = vplane + (size_t)max(at, 0) * HD + g * (HD / 8);
                if (HD == 128) {
                    uint4 x = make_uint4(0u, 0u, 0u, 0u);
                    if (at >= 0) x = ldg_stream(src);
                    vw[u][i][0] = x.x, vw[u][i][1] = x.y, vw[u][i][HD / 32 - 2] = x.z, vw[u][i][HD / 32 - 1] = x.w;
                } else {
                    uint2 x = make_uint2(0u, 0u);
                    if (at >= 0) x = __ldg((const uint2*)src);
                    vw[u][i][0] = x.x, vw[u][i][1] = x.y;
                }
            }

        // ---- scores: s[b][0, 1] of head g and keys 8 b + 2 t4 + {0, 1}, s[b][2, 3] of head g + 8
        float s[4][ROWS == 16 ? 4 : 2];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
#pragma unroll
            for (int e = 0; e < 2 * NR; ++e) s[b][e] = 0.0f;
#pragma unroll
            for (int i = 0; i < QS; ++i) {
                uint32_t b0, b1;
                e4m3x4_to_f16(kw[b][i], b0, b1);
                mma_f16<ROWS>(s[b], idle, qa[i][0], NR == 2 ? qa[i][NR - 1] : 0u, qa[i][NR], NR == 2 ? qa[i][2 * NR - 1] : 0u, b0, b1);
            }
        }
        float mx[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) mx[r] = m[r];
        const float kf = power_of_two(ek);
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float f = __shfl_sync(0xffffffffu, kf, b * 8 + 2 * t4 + e);
                const bool in = __shfl_sync(0xffffffffu, row, b * 8 + 2 * t4 + e) >= 0;
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    const float v = in ? s[b][2 * r + e] * back[r] * f : -INFINITY;
                    s[b][2 * r + e] = v;
                    mx[r] = fmaxf(mx[r], v);
                }
            }
        const int most = max(R, __reduce_max_sync(0xffffffffu, ev));
        float old[NR], use[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
            use[r] = mx[r] == -INFINITY ? 0.0f : mx[r];
            old[r] = exp2f(m[r] - use[r]);
            l[r] *= old[r];
            m[r] = mx[r];
            old[r] *= power_of_two(max(R - most, -126));
        }
        R = most;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 2 * NR; ++e) o[i][e] *= old[e >> 1];
        const float vf = power_of_two(max(ev - R, -126));
        uint32_t pa[4][NR];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float f0 = __shfl_sync(0xffffffffu, vf, b * 8 + 2 * t4), f1 = __shfl_sync(0xffffffffu, vf, b * 8 + 2 * t4 + 1);
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const float p0 = exp2f(s[b][2 * r] - use[r]), p1 = exp2f(s[b][2 * r + 1] - use[r]);
                l[r] += p0 + p1;
                pa[b][r] = pack_f16(p0 * f0, p1 * f1);
            }
        }
        // ---- values: column tile i holds entries g HD / 8 + i of the eight g
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int w = 0; w < HD / 32; ++w) {
                uint32_t lo01 = __byte_perm(vw[u][0][w], vw[u][1][w], 0x5140), lo23 = __byte_perm(vw[u][0][w], vw[u][1][w], 0x7362);
                uint32_t hi01 = __byte_perm(vw[u][2][w], vw[u][3][w], 0x5140), hi23 = __byte_perm(vw[u][2][w], vw[u][3][w], 0x7362);
                uint32_t b0[4], b1[4];
                e4m3x4_to_f16(lo01, b0[0], b0[1]);
                e4m3x4_to_f16(lo23, b0[2], b0[3]);
                e4m3x4_to_f16(hi01, b1[0], b1[1]);
                e4m3x4_to_f16(hi23, b1[2], b1[3]);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    mma_f16<ROWS>(o[4 * w + i], idle, pa[2 * u][0], NR == 2 ? pa[2 * u][NR - 1] : 0u, pa[2 * u + 1][0],
                                  NR == 2 ? pa[2 * u + 1][NR - 1] : 0u, b0[i], b1[i]);
            }
    }

    // ---- the four warps' results, added in their order
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (t4 == 0) sm[warp][g + 8 * r] = m[r], sl[warp][g + 8 * r] = l[r];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            red[warp][g + 8 * r][2 * t4 * NT + i] = o[i][2 * r];
            red[warp][g + 8 * r][(2 * t4 + 1) * NT + i] = o[i][2 * r + 1];
        }
    }
    if (lane == 0) sr[warp] = R;
    __syncthreads();
    for (int i = tid; i < n_h * (HD / 2); i += WARPS * 32) {
        const int row = i / (HD / 2), d = 2 * (i % (HD / 2));
        float M = sm[0][row];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) M = fmaxf(M, sm[w][row]);
        float L = 0.0f;
        float2 a = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (sm[w][row] == -INFINITY) continue;
            const float f = exp2f(sm[w][row] - M), fr = f * power_of_two(max(sr[w], -126));
            L += sl[w][row] * f;
            a.x = fmaf(red[w][row][d], fr, a.x);
            a.y = fmaf(red[w][row][d + 1], fr, a.y);
        }
        const size_t head = (size_t)t * n_heads + h0 + row;
        if (splits == 1) {
            const float inv = M == -INFINITY ? 0.0f : 1.0f / L;
            *(__nv_bfloat162*)(out + head * HD + d) = __floats2bfloat162_rn(a.x * inv, a.y * inv);
        } else {
            *(float2*)(part_acc + (head * splits + split) * HD + d) = a;
            if (d == 0) *(float2*)(part_ml + (head * splits + split) * 2) = make_float2(M, L);
        }
    }
}

// The stretches of every (row, head) added in their order: a warp each.
template <int HD>
__global__ void __launch_bounds__(128) decode_e4m3_merge_kernel(__nv_bfloat16* __restrict__ out, const float* __restrict__ part_acc,
                                                                const float* __restrict__ part_ml, long long n, int splits) {
    cj::after_predecessor();
    cj::release_successor();
    constexpr int VEC = HD / 32;
    const int lane = threadIdx.x & 31;
    const long long idx = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (idx >= n) return;
    const size_t s0 = (size_t)idx * splits;
    float M = -INFINITY;
    for (int s = lane; s < splits; s += 32) M = fmaxf(M, part_ml[(s0 + s) * 2]);
    M = warp_max(M);
    float L = 0.0f, a[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) a[j] = 0.0f;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        const float2 ml = *(const float2*)(part_ml + (s0 + s) * 2);
        const float f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - M);
        L = fmaf(ml.y, f, L);
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const float2 v = *(const float2*)(part_acc + (s0 + s) * HD + lane * VEC + j);
            a[j] = fmaf(v.x, f, a[j]);
            a[j + 1] = fmaf(v.y, f, a[j + 1]);
        }
    }
    const float inv = M == -INFINITY ? 0.0f : 1.0f / L;
#pragma unroll
    for (int j = 0; j < VEC; j += 2)
        *(__nv_bfloat162*)(out + (size_t)idx * HD + lane * VEC + j) = __floats2bfloat162_rn(a[j] * inv, a[j + 1] * inv);
}

}  // namespace

// qkv: float32 [T, ld], columns from q_off, k_off, v_off (even, as ld); q_out: bf16 [T, n_heads, hd]; planes: e4m3 codes
// [pages, n_kv, page_tokens, hd], exponents + 127 [pages, n_kv, page_tokens].  hd: 64 or 128; rotary_dim even, at most hd.
// A row without a request (of table_rows) or a page (of n_pages) is rotated and not written.
CJ_EXPORT int cj_append_e4m3(const float* qkv, int ld, int q_off, int k_off, int v_off, void* q_out, void* kplane, void* vplane,
                             void* kexp, void* vexp, const int* positions, const int* row_req, const int* table, int table_rows, int table_stride,
                             int page_tokens, int n_pages, int T, int n_heads, int n_kv, int hd, int rotary_dim, const float* inv_freq, int write_kv,
                             cudaStream_t stream) {
    if (T <= 0) return 0;
    if (!qkv || !q_out || !positions || n_heads <= 0) return CJ_ERR_ARG;
    if (hd != 64 && hd != 128) return CJ_ERR_SIZE;
    if (rotary_dim < 0 || rotary_dim > hd || (rotary_dim & 1)) return CJ_ERR_SIZE;
    if (rotary_dim > 0 && !inv_freq) return CJ_ERR_ARG;
    if (write_kv && (!kplane || !vplane || !kexp || !vexp || !row_req || !table || page_tokens <= 0 || n_kv <= 0)) return CJ_ERR_ARG;
    if (((ld | q_off | k_off | v_off) & 1) || (((uintptr_t)qkv | (uintptr_t)q_out) & 7)) return CJ_ERR_ALIGN;
    if (write_kv && (((uintptr_t)kplane | (uintptr_t)vplane) & 3)) return CJ_ERR_ALIGN;
    const int slots = n_heads + (write_kv ? 2 * n_kv : 0);
    // few rows: a warp a head; many: a row's heads by one block, so that its angles are worked out once
    const int parts = T >= 256 ? 1 : min((slots + 7) / 8, 64);
    const dim3 grid(T, parts);
    auto kern = hd == 128 ? append_e4m3_kernel<128> : append_e4m3_kernel<64>;
    cj::launch(kern, dim3(grid), dim3(256), 0, stream, qkv, ld, q_off, k_off, v_off, (__nv_bfloat16*)q_out, (uint8_t*)kplane,
               (uint8_t*)vplane, (uint8_t*)kexp, (uint8_t*)vexp, positions, row_req, table, table_rows, table_stride, page_tokens, n_pages, n_heads, n_kv,
               rotary_dim, inv_freq, write_kv);
    return launch_status();
}

// q, out: bf16 [T, n_heads, hd]; the cache as cj_append_e4m3 writes it.  splits > 1: every row's keys are dealt to that many
// blocks; part_acc float32 [T, n_heads, splits, hd] and part_ml [T, n_heads, splits, 2] are scratch.  hd: 64 or 128.
// positions null: the rows are portions of requests, req_start int32 [n_requests + 1], req_prior [n_requests] (one split).
// table: int32 [n_requests, table_stride]; a row of no request sees no key, and a page of no number below n_pages holds none.
CJ_EXPORT int cj_decode_e4m3(const void* q, void* out, const void* kplane, const void* vplane, const void* kexp, const void* vexp,
                             int n_pages, const int* positions, const int* row_req, const int* req_start, const int* req_prior,
                             int n_requests, const int* table, int table_stride, int page_tokens, int T, int n_heads, int n_kv, int hd, int window, float scale, int splits, float* part_acc, float* part_ml,
                             cudaStream_t stream) {
    if (T <= 0) return 0;
    if (!q || !out || !kplane || !vplane || !kexp || !vexp || !table) return CJ_ERR_ARG;
    if (positions ? !row_req : (!req_start || !req_prior || splits != 1)) return CJ_ERR_ARG;
    if (splits < 1 || (splits > 1 && (!part_acc || !part_ml))) return CJ_ERR_ARG;
    if (n_heads <= 0 || n_kv <= 0 || n_heads % n_kv != 0 || page_tokens <= 0 || window < 0 || n_requests <= 0 || n_pages <= 0) return CJ_ERR_SIZE;
    if (hd != 64 && hd != 128) return CJ_ERR_SIZE;
    if (((uintptr_t)q | (uintptr_t)kplane | (uintptr_t)vplane) & 15) return CJ_ERR_ALIGN;
    if ((uintptr_t)out & 3) return CJ_ERR_ALIGN;
    if ((long long)n_pages * n_kv * page_tokens > 0x7fffffffLL || (long long)table_stride * page_tokens > 0x7fffffffLL) return CJ_ERR_SIZE;
    const int group = n_heads / n_kv, rows = group > 8 ? 16 : 8, head_batches = (group + rows - 1) / rows;
    if ((long long)n_kv * head_batches > 65535 || splits > 65535) return CJ_ERR_SIZE;
    const dim3 grid(T, n_kv * head_batches, splits);
    auto kern = hd == 128 ? (rows == 8 ? decode_e4m3_kernel<128, 8> : decode_e4m3_kernel<128, 16>)
                          : (rows == 8 ? decode_e4m3_kernel<64, 8> : decode_e4m3_kernel<64, 16>);
    cj::launch(kern, dim3(grid), dim3(WARPS * 32), 0, stream, (const __nv_bfloat16*)q, (__nv_bfloat16*)out, (const uint8_t*)kplane,
               (const uint8_t*)vplane, (const uint8_t*)kexp, (const uint8_t*)vexp, positions, row_req, req_start, req_prior, n_requests, table,
               table_stride, page_tokens, n_pages, n_heads, n_kv, head_batches, window, scale * 1.4426950408889634f, splits, part_acc, part_ml);
    if (splits > 1) {
        const int status = launch_status();
        if (status != 0) return status;
        const long long n = (long long)T * n_heads;
        auto merge = hd == 128 ? decode_e4m3_merge_kernel<128> : decode_e4m3_merge_kernel<64>;
        cj::launch(merge, dim3((unsigned)((n + 3) / 4)), dim3(128), 0, stream, (__nv_bfloat16*)out, (const float*)part_acc, (const float*)part_ml, n, splits);
    }
    return launch_status();
}
