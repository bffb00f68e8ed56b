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
#include "tc_common.cuh"

using namespace cj;
using tc::bulk_load;
using tc::cluster_sync;
using tc::ex2;
using tc::mbar_expect_tx;
using tc::mbar_init;
using tc::mbar_wait_warp;

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
// stretch of the row's keys; each warp walks over its 32-key pieces with a running softmax of its own and a ring of shared memory of its
// own, filled by bulk copies of a page's run of rows a step ahead (registers that loads are on their way to would make every shuffle and
// exponential wait for them).  An e4m3 code is an f16 number exactly: the products are mma.sync m16n8k16 of f16 numbers, float32 out, with the codes
// as their first operand, so that all 16 rows of a product are keys (or entries) and its columns the heads.  (mma.sync takes e4m3 operands
// too; with them 64 rows of up to 2,048 keys, 16 heads over 16, took 80 us where this took 61.)
//     S^T = code_k . q^T                              s = S scale 2^e_k
//     O^T = code_v^T . (p 2^(m + e_v - N))^T          m: a head's largest score so far, N: its reference of what keys bring, both in octaves
// The order of a product's K, and of its rows, is free as long as both sides keep it: a lane's share of a key is HD / 4 neighbouring bytes and
// of four value rows HD / 8 each (two keys' bytes side by side after a byte permute), 8- and 16-byte loads.  The weights turn from S^T's layout
// into an operand by movmatrix.  Queries are brought to [2^7, 2^8) at their largest entry by a power of two: f16 keeps an entry's eight
// bits down to 2^-21 of that.
// N is an integer, 12 below the largest s + e_v when it was last moved; it moves when a key may bring more than 2^15 of it.  So the factors are at most
// 2^15 in f16 and keep its 11 bits down to 2^-26 of the largest contribution, some down to 2^-36, whatever weight and value make it up, and the rest is what
// float32 weights lose too (those below 2^-126).  A reference of the values' exponents alone, one for a warp, was 2 to 4 % faster (64 rows of up to 2,048 keys
// 60.7 us, 61.6 so; eight of up to 32,768 48 and 50) and lost all others to a large value that the row hardly looks at.  The divisor's weights are not rounded.
// Bound by DRAM, 2 (HD + 1) bytes a key and kv head, where heads have keys of their own (16 over 16: 64 rows of up to 2,048 keys 61.6 us, 72 % of a copy's rate;
// 32 rows of 4,096 107, 76 %); by a step's chain where few blocks hold the keys of many heads (28 over 4: 64 rows of up to 2,048 35 us, 34 %).
// ---------------------------------------------------------------------------------------------------------------------------
constexpr int WARPS = 4;
constexpr int STEP = 32;                   // keys of a warp's step
constexpr int STAGES = 2, BLOCKS = 3;      // steps of a warp's ring, blocks an SM

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {      // an 8 x 8 matrix of f16, two of a row a lane
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *(const uint32_t*)&v;
}

// A row's blocks, up to eight, can be a cluster and add their results through each other's shared memory; otherwise they leave them to a kernel of its own.
constexpr int MOST_CLUSTER = 8;

__device__ __forceinline__ float2 ld_of_block(const float* p, int rank) {      // what lies at p in the shared memory of the cluster's block `rank`
    uint32_t a;
    float2 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(tc::smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(a) : "memory");
    return v;
}

template <int HD, int ROWS>
__global__ void __launch_bounds__(WARPS * 32, ROWS == 16 ? 2 : BLOCKS) decode_e4m3_kernel(
    const __nv_bfloat16* __restrict__ q, __nv_bfloat16* __restrict__ out, const uint8_t* __restrict__ kplane, const uint8_t* __restrict__ vplane,
    const uint8_t* __restrict__ kexp, const uint8_t* __restrict__ vexp, const int* __restrict__ positions, const int* __restrict__ row_req,
    const int* __restrict__ req_start, const int* __restrict__ req_prior, int n_requests, const int* __restrict__ table, int table_stride,
    int page_tokens, int page_shift, int n_pages, int n_heads, int n_kv, int head_batches, int window, float scale_log2, int splits,
    float* __restrict__ part_acc, float* __restrict__ part_ml) {
    constexpr int NB = ROWS / 8;           // column tiles of eight heads
    constexpr int QS = HD / 16;            // steps of 16 of the head's entries, and words of a key that are a lane's
    constexpr int VW = HD / 32;            // words of a value row that are a lane's
    constexpr int NT = HD / 16;            // row tiles of the output
    cj::after_predecessor();
    cj::release_successor();
    extern __shared__ __align__(128) uint8_t ring[];                   // [WARPS][STAGES][keys, values][STEP][HD], then the warps' results
    float (*red)[ROWS][HD + 4] = (float (*)[ROWS][HD + 4])ring;
    __shared__ float sm[WARPS][ROWS], sl[WARPS][ROWS], sn[WARPS][ROWS];
    float* together = (float*)(ring + sizeof(float) * WARPS * ROWS * (HD + 4));    // a cluster's block: its four warps' sums [ROWS][HD] ...
    __shared__ float2 together_ml[ROWS];                                          // ... and maximum and divisor
    __shared__ uint64_t bars[WARPS][STAGES];
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
    if (req < 0) p = -1;
    // keys [from, end): the window is the position's, also where the table ends before it
    const int from = window > 0 && p >= window ? p - window + 1 : 0, end = min(p, table_stride * page_tokens - 1) + 1;
    const int n_keys = max(0, end - from);
    // equal stretches of whole steps
    const int per = (((n_keys + splits - 1) / splits + STEP - 1) / STEP) * STEP;
    const int first = from + split * per, last = min(end, first + per);
    const int* tab = table + (size_t)max(req, 0) * table_stride;

    // Lane j looks up key j of a step: its page two steps before the products, from it the key's row in the planes (-1: none) and its exponents one
    // step before; the first lane of every run of keys that lie side by side in a page copies the run's codes.
    uint64_t* bar = bars[warp];
    if (lane < STAGES) mbar_init(&bar[lane], 1);
    tc::fence_barrier_init();
    __syncwarp();
    const uint32_t mine = tc::smem_u32(ring) + warp * STAGES * 2 * STEP * HD;
    int page = -1, at_page = 0, k_next = 0, v_next = 0;      // (exponents + 127; v_next below 0: no key)
    auto ask_page = [&](int k0) {
        const int key = k0 + lane, n = page_shift >= 0 ? key >> page_shift : key / page_tokens;
        at_page = key - n * page_tokens;
        page = key < last ? __ldg(tab + n) : -1;
    };
    auto ask = [&](int k0, int stage) {
        const bool there = page >= 0 && page < n_pages;
        const long long row = there ? ((long long)page * n_kv + kvh) * page_tokens + at_page : 0;
        const uint32_t have = __ballot_sync(0xffffffffu, there);
        if (lane == 0) mbar_expect_tx(&bar[stage], __popc(have) * 2 * HD);
        __syncwarp();
        if (there && (lane == 0 || at_page == 0)) {
            const uint32_t n = min(min(page_tokens - at_page, STEP - lane), last - (k0 + lane)) * HD;
            const uint32_t dst = mine + (stage * 2 * STEP + lane) * HD;
            bulk_load(dst, kplane + row * HD, n, &bar[stage]);
            bulk_load(dst + STEP * HD, vplane + row * HD, n, &bar[stage]);
        }
        k_next = there ? (int)kexp[row] : 0;
        v_next = there ? (int)vexp[row] : -1;
    };
    int k0 = first + warp * STEP;
    constexpr int STRIDE = WARPS * STEP;
    ask_page(k0);
    if (k0 < last) ask(k0, 0);
    ask_page(k0 + STRIDE);

    // the queries of heads g (and g + 8), entries t4 HD / 4 + 4 i + {0, 1} and {2, 3}; of heads 2 t4 and 2 t4 + 1 (and 8 more), what undoes
    // their power of two, with the scale in units of log 2
    uint32_t qb[NB][QS][2];
    float back[NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        uint32_t w[2 * QS];
        const int head = g + 8 * n;
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
        // (a query that is infinite somewhere has no finite score: all are NaN, as those of one that holds a NaN are by themselves)
        const float up = most < INFINITY ? power_of_two(e) : NAN, undo = scale_log2 * power_of_two(-e);
        back[n][0] = __shfl_sync(0xffffffffu, undo, 8 * t4);
        back[n][1] = __shfl_sync(0xffffffffu, undo, 8 * t4 + 4);
#pragma unroll
        for (int i = 0; i < QS; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) qb[n][i][j] = pack_f16(bf16_low(w[2 * i + j]) * up, bf16_high(w[2 * i + j]) * up);
    }

    float o[NB][NT][4];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][i][e] = 0.0f;
    float m[NB][2], l[NB][2], N[NB][2], h[NB][2];      // h: 2^(m - N)
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) m[n][e] = -INFINITY, l[n][e] = 0.0f, N[n][e] = -1e30f, h[n][e] = 0.0f;      // (N finite: m - N stays -infinity)

    uint32_t phase = 0;
    for (int stage = 0; k0 < last; k0 += STRIDE) {
        const int k_exp = k_next, v_exp = v_next;
        const bool more = k0 + STRIDE < last;
        if (more) {
            ask(k0 + STRIDE, stage ^ 1);
            ask_page(k0 + 2 * STRIDE);
        }
        if (!mbar_wait_warp(&bar[stage], phase, 21)) {
            if (more) mbar_wait_warp(&bar[stage ^ 1], phase ^ stage, 22);        // (the copies end before the block does)
            break;
        }
        const uint8_t* keys = ring + (warp * STAGES + stage) * 2 * STEP * HD;
        const uint8_t* values = keys + STEP * HD;
        const uint32_t there = __ballot_sync(0xffffffffu, v_exp >= 0);
        // ---- scores: s[n][u][2 k + e] of head 8 n + 2 t4 + e and key 16 u + 8 k + g
        float s[NB][2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][u][e] = 0.0f;
#pragma unroll
            for (int i = 0; i < QS / 4; ++i) {
                const uint4 a = *(const uint4*)(keys + (16 * u + g) * HD + t4 * (HD / 4) + i * 16);
                const uint4 b = *(const uint4*)(keys + (16 * u + 8 + g) * HD + t4 * (HD / 4) + i * 16);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t a0, a1, a2, a3;
                    e4m3x4_to_f16((&a.x)[j], a0, a2);
                    e4m3x4_to_f16((&b.x)[j], a1, a3);
#pragma unroll
                    for (int n = 0; n < NB; ++n) mma_f16(s[n][u], a0, a1, a2, a3, qb[n][4 * i + j][0], qb[n][4 * i + j][1]);
                }
            }
        }
        // scores in units of the queries' own until the exponential; m is the largest so far in units of log 2
        const float kf = __int_as_float(k_exp << 23);
        float mx[NB][2];
#pragma unroll
        for (int n = 0; n < NB; ++n) mx[n][0] = mx[n][1] = -INFINITY;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float f = __shfl_sync(0xffffffffu, kf, b * 8 + g);
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) s[n][b >> 1][2 * (b & 1) + e] *= f;
        }
        if (there != 0xffffffffu) {
#pragma unroll
            for (int b = 0; b < 4; ++b)
                if (!(there >> (b * 8 + g) & 1))
#pragma unroll
                    for (int n = 0; n < NB; ++n) s[n][b >> 1][2 * (b & 1)] = s[n][b >> 1][2 * (b & 1) + 1] = -INFINITY;
        }
        const float most = (float)(__reduce_max_sync(0xffffffffu, v_exp) - 127);
        bool moved = false;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = fmaxf(fmaxf(s[n][0][e], s[n][0][2 + e]), fmaxf(s[n][1][e], s[n][1][2 + e]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                mx[n][e] = fmaxf(m[n][e], x * back[n][e]);
                // (no key brings more than the largest score and the largest exponent together; whether one does is looked at below)
                moved = moved || mx[n][e] != m[n][e] || fmaf(x, back[n][e], most) > N[n][e] + 15.0f;
            }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                float old[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    old[e] = mx[n][e] == -INFINITY ? 1.0f : ex2(m[n][e] - mx[n][e]);
                    l[n][e] *= old[e];
                    m[n][e] = mx[n][e];
                    float y = -INFINITY;
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        y = fmaxf(y, fmaf(s[n][b >> 1][2 * (b & 1) + e], back[n][e], (float)(__shfl_sync(0xffffffffu, v_exp, b * 8 + g) - 127)));
                    y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4));
                    y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8));
                    y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
                    y = y > N[n][e] + 15.0f ? ceilf(y) - 12.0f : N[n][e];
                    old[e] = ex2(N[n][e] - y);
                    N[n][e] = y;
                    h[n][e] = ex2(m[n][e] - y);
                }
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][i][e] *= old[e & 1];
            }
        }
        // ---- weights: pb[n][b] of head 8 n + g and keys 8 b + 2 t4 + {0, 1}
        const float vf = power_of_two(max(v_exp - 127, -126));
        uint32_t pb[NB][4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float f = __shfl_sync(0xffffffffu, vf, b * 8 + g);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                float x[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float w = ex2(fmaf(s[n][b >> 1][2 * (b & 1) + e], back[n][e], m[n][e] == -INFINITY ? 0.0f : -m[n][e]));
                    l[n][e] += w;
                    x[e] = w * f * h[n][e];          // (in this order: f h alone could leave float32)
                }
                pb[n][b] = transposed(pack_f16(x[0], x[1]));
            }
        }
        // ---- values: row tile i holds entries g HD / 8 + 2 i (rows 0 .. 7) and + 2 i + 1 (8 .. 15) of the eight g
        uint32_t vw[2][4][VW];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = u * 16 + (i >> 1) * 8 + 2 * t4 + (i & 1);
                if (HD == 128) {
                    const uint4 x = *(const uint4*)(values + row * HD + g * 16);
                    vw[u][i][0] = x.x, vw[u][i][1] = x.y, vw[u][i][VW - 2] = x.z, vw[u][i][VW - 1] = x.w;
                } else {
                    const uint2 x = *(const uint2*)(values + row * HD + g * 8);
                    vw[u][i][0] = x.x, vw[u][i][1] = x.y;
                }
                if (there != 0xffffffffu && !(there >> row & 1))      // (a row of no key holds what was there before)
#pragma unroll
                    for (int w = 0; w < VW; ++w) vw[u][i][w] = 0;
            }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int w = 0; w < VW; ++w)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t a0, a1, a2, a3;
                    e4m3x4_to_f16(__byte_perm(vw[u][0][w], vw[u][1][w], j ? 0x7362 : 0x5140), a0, a1);
                    e4m3x4_to_f16(__byte_perm(vw[u][2][w], vw[u][3][w], j ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
                    for (int n = 0; n < NB; ++n) mma_f16(o[n][2 * w + j], a0, a1, a2, a3, pb[n][2 * u], pb[n][2 * u + 1]);
                }
        __syncwarp();                      // (every lane has read this step's stage)
        phase ^= stage;
        stage ^= 1;
    }
    __syncthreads();                       // the ring becomes the results' place

    // ---- the four warps' results, added in their order.  Here and below a stretch without keys is one whose sum of weights is 0 (any key leaves 1 or more):
    // its maximum does not tell, since scores that are NaN leave none and have to be in the result
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int head = 8 * n + 2 * t4 + e;
            l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
            l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
            l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
            if (g == 0) sm[warp][head] = m[n][e], sl[warp][head] = l[n][e], sn[warp][head] = N[n][e];
#pragma unroll
            for (int i = 0; i < NT; ++i) *(float2*)&red[warp][head][g * (HD / 8) + 2 * i] = make_float2(o[n][i][e], o[n][i][2 + e]);
        }
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
            if (sl[w][row] == 0.0f) continue;
            const float fr = exp2f(sn[w][row] - M);      // (weights that were kept beside N, as sums beside M)
            L += sl[w][row] * exp2f(sm[w][row] - M);
            a.x = fmaf(red[w][row][d], fr, a.x);
            a.y = fmaf(red[w][row][d + 1], fr, a.y);
        }
        const size_t head = (size_t)t * n_heads + h0 + row;
        if (splits == 1) {
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            *(__nv_bfloat162*)(out + head * HD + d) = __floats2bfloat162_rn(a.x * inv, a.y * inv);
        } else if (part_acc) {
            *(float2*)(part_acc + (head * splits + split) * HD + d) = a;
            if (d == 0) *(float2*)(part_ml + (head * splits + split) * 2) = make_float2(M, L);
        } else {
            *(float2*)(together + row * HD + d) = a;
            if (d == 0) together_ml[row] = make_float2(M, L);
        }
    }
    if (splits == 1 || part_acc) return;
    cluster_sync();
    for (int i = split * WARPS * 32 + tid; i < n_h * (HD / 2); i += splits * WARPS * 32) {
        const int row = i / (HD / 2), d = 2 * (i % (HD / 2));
        float2 ml[MOST_CLUSTER], v[MOST_CLUSTER];
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int b = 0; b < MOST_CLUSTER; ++b) {
            ml[b] = make_float2(-INFINITY, 0.0f);
            if (b < splits) ml[b] = ld_of_block((const float*)&together_ml[row], b), v[b] = ld_of_block(together + row * HD + d, b);
            M = fmaxf(M, ml[b].x);
        }
        float2 a = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int b = 0; b < MOST_CLUSTER; ++b) {
            if (ml[b].y == 0.0f) continue;
            const float f = exp2f(ml[b].x - M);
            L = fmaf(ml[b].y, f, L);
            a.x = fmaf(v[b].x, f, a.x);
            a.y = fmaf(v[b].y, f, a.y);
        }
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        *(__nv_bfloat162*)(out + ((size_t)t * n_heads + h0 + row) * HD + d) = __floats2bfloat162_rn(a.x * inv, a.y * inv);
    }
    cluster_sync();                        // (the others may still read this block's shared memory)
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
    for (int c = 0; c < splits; c += 32) {
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (c + lane < splits) ml = *(const float2*)(part_ml + (s0 + c + lane) * 2);
        const float mine = ml.y == 0.0f ? 0.0f : exp2f(ml.x - M);
        L = fmaf(ml.y, mine, L);
        const int n = min(32, splits - c);
#pragma unroll 8
        for (int s = 0; s < n; ++s) {
            const float f = __shfl_sync(0xffffffffu, mine, s);
#pragma unroll
            for (int j = 0; j < VEC; j += 2) {
                const float2 v = *(const float2*)(part_acc + (s0 + c + s) * HD + lane * VEC + j);
                a[j] = fmaf(v.x, f, a[j]);
                a[j + 1] = fmaf(v.y, f, a[j + 1]);
            }
        }
    }
    L = warp_sum(L);
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
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
// blocks, which are a cluster (up to eight) or, with scratch given, leave their results to a second kernel: part_acc float32 [T, n_heads, splits, hd] and part_ml [T, n_heads, splits, 2].  hd: 64 or 128.
// positions null: the rows are portions of requests, req_start int32 [n_requests + 1], req_prior [n_requests] (no scratch).
// table: int32 [n_requests, table_stride]; a row of no request sees no key, and a page of no number below n_pages holds none.
CJ_EXPORT int cj_decode_e4m3(const void* q, void* out, const void* kplane, const void* vplane, const void* kexp, const void* vexp,
                             int n_pages, const int* positions, const int* row_req, const int* req_start, const int* req_prior,
                             int n_requests, const int* table, int table_stride, int page_tokens, int T, int n_heads, int n_kv, int hd, int window, float scale, int splits, float* part_acc, float* part_ml,
                             cudaStream_t stream) {
    if (T <= 0) return 0;
    if (!q || !out || !kplane || !vplane || !kexp || !vexp || !table) return CJ_ERR_ARG;
    if (positions ? !row_req : (!req_start || !req_prior || part_acc)) return CJ_ERR_ARG;
    if (splits < 1 || (splits > MOST_CLUSTER && !part_acc) || (part_acc && !part_ml)) return CJ_ERR_ARG;
    if (n_heads <= 0 || n_kv <= 0 || n_heads % n_kv != 0 || page_tokens <= 0 || window < 0 || n_requests <= 0 || n_pages <= 0 || !(scale > 0.0f)) return CJ_ERR_SIZE;
    if (hd != 64 && hd != 128) return CJ_ERR_SIZE;
    if (((uintptr_t)q | (uintptr_t)kplane | (uintptr_t)vplane) & 15) return CJ_ERR_ALIGN;
    if ((uintptr_t)out & 3) return CJ_ERR_ALIGN;
    if ((long long)n_pages * n_kv * page_tokens > 0x7fffffffLL || (long long)table_stride * page_tokens > 0x7fffffffLL) return CJ_ERR_SIZE;
    const int group = n_heads / n_kv, rows = group > 8 ? 16 : 8, head_batches = (group + rows - 1) / rows;
    if ((long long)n_kv * head_batches > 65535 || splits > 65535) return CJ_ERR_SIZE;
    const dim3 grid(T, n_kv * head_batches, splits);
    auto kern = hd == 128 ? (rows == 8 ? decode_e4m3_kernel<128, 8> : decode_e4m3_kernel<128, 16>)
                          : (rows == 8 ? decode_e4m3_kernel<64, 8> : decode_e4m3_kernel<64, 16>);
    const int smem = max(WARPS * STAGES * 2 * STEP * hd, WARPS * rows * (hd + 4) * 4 + rows * hd * 4);
    if (splits == 1) part_acc = part_ml = nullptr;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = part_acc ? 1 : splits;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cj::overlap_launches() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kern, (const __nv_bfloat16*)q, (__nv_bfloat16*)out, (const uint8_t*)kplane, (const uint8_t*)vplane,
                       (const uint8_t*)kexp, (const uint8_t*)vexp, positions, row_req, req_start, req_prior, n_requests, table, table_stride,
                       page_tokens, (page_tokens & (page_tokens - 1)) == 0 ? __builtin_ctz(page_tokens) : -1, n_pages, n_heads, n_kv,
                       head_batches, window, scale * 1.4426950408889634f, splits, part_acc, part_ml);
    if (part_acc) {
        const int status = launch_status();
        if (status != 0) return status;
        const long long n = (long long)T * n_heads;
        auto merge = hd == 128 ? decode_e4m3_merge_kernel<128> : decode_e4m3_merge_kernel<64>;
        cj::launch(merge, dim3((unsigned)((n + 3) / 4)), dim3(128), 0, stream, (__nv_bfloat16*)out, (const float*)part_acc, (const float*)part_ml, n, splits);
    }
    return launch_status();
}

CJ_EXPORT int cj_cache_e4m3_error() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, tc::g_error_flag, sizeof(int)) != cudaSuccess) return -1;
    return v;
}
