// Products with 4-bit weights for many rows, on the 5th-generation tensor cores (tcgen05):
//
//     out[t, f] (+)= sum_k (s q)[f, k] x[t, k]   (+ bias[f]; or silu of it times a second product)
//
// with the weights and their layout of gemm_q4.cu.  A code times its scale is a bfloat16 number, so the weights are turned into
// bfloat16 on their way and the product is that of the unpacked weights to the bit.  They are the product's 128 rows and are read from
// tensor memory: eight warps take 128 features x 128 of K (a pair of blocks of 64), each two pieces of 16 features (a 16-byte load a lane
// each), and put them there by two 16x256b stores, whose lanes hold what the layout gave them; nothing is written back to shared
// memory, whose bandwidth the other operand needs.  The rows of x are the product's columns, up to 256 of them.
//
// Persistent blocks, one an SM: two warps load x by TMA, one the codes by bulk copies, 16 convert (two sets, a pair of blocks each in turn),
// one thread issues the products, eight warps drain an accumulator while the next fills where tensor memory has room for two (up to 192
// rows a tile).  The gated form puts 16 features of the gate and 16 of the other weight on each warp's 32 lanes, so that their sums meet by a
// shuffle.
//
// What bounds it: up to some 160 rows a tile the warps that share a scheduler.  Integer and bfloat16 instructions go out at one in two
// clocks each, a pair of blocks is 230 clocks of the integer pipe a scheduler, and the one thread that issues eight products, a wait and an arrival
// a pair does so between the others' instructions: 670 clocks a pair in all (64 rows x 6,144 x 6,144: 20 us; with waits, arrivals and ring
// sums for each block of 64, three instructions more a word of codes, and codes freed only after the product, 31 us).  Beyond, the tensor core
// (832 clocks a pair at 208 rows) and, with one accumulator, the time to drain it: 2,048 rows x 3,584 x 3,584 take 46 us, 1.14 PFLOP/s, in a
// burst and 55, 0.96, call after call (the power cap's clock).
#define CJ_LIB "gemm_q4_tc"
#include "common.cuh"
#include "q4.cuh"
#include "tc_common.cuh"

using namespace tc;

namespace {

constexpr int LOAD_X = 0, LOAD_CODES = 2, PRODUCT = 3, EPI0 = 4, EPI_WARPS = 8, CONV0 = EPI0 + EPI_WARPS, CONV_SETS = 2;      // warps
constexpr int THREADS = (CONV0 + 8 * CONV_SETS) * 32;
// (a converting set sees every other pair: an even number of stages of codes are its own, and no wait takes a round for another)
constexpr int MAX_STAGES = 4, CODE_STAGES = 6, MAX_GROUPS = 1024;
static_assert(CODE_STAGES % CONV_SETS == 0, "a set's stages of codes are its own");
constexpr int HALF_COLS = 32, SLOT_COLS = 2 * HALF_COLS;      // a pair of blocks of K: twice 128 rows x 64 bfloat16
constexpr int SMEM_LIMIT = 218 * 1024;        // (with the groups' tables, 8 KB, what a block can have)
constexpr int BAR_BYTES = 512;

struct Args {
    const uint8_t* w;
    const uint8_t* w_up;
    const float* bias;
    void* out;
    const int* offsets;
    long long ldo;
    int rows, features, K, groups, half_out, accumulate;
    int tok;                   // rows of x a tile takes
    int stages, accs;          // pairs of blocks of K that x and the weights in tensor memory have room for; accumulators
    int x_bytes;               // of a block of 64 of K; a stage has two
    // A float32 result's K goes in parts of so many pairs of blocks of 64, each summed from zero and added to what the parts before left: tcgen05 cuts its sums off
    // rather than rounding them, and an error that grows with their length stays that of 2,560 entries (2,048 x 3,584 x 3,584: 1.2e-6 of the result
    // in one part, 5e-7 in two).
    int part_pairs;
};

struct Tile {
    int group, f, tok0, tok_end;
};

// dense: features run fastest (neighbouring blocks share the rows of x); grouped: rows run fastest (they share weights)
__device__ __forceinline__ Tile tile_of(const Args& p, int tile, int feat_tiles, const int* before, const int* edge) {
    Tile t;
    if (!p.offsets) {
        t.group = 0;
        t.f = tile % feat_tiles;
        t.tok0 = tile / feat_tiles * p.tok;
        t.tok_end = min(p.rows, t.tok0 + p.tok);
        return t;
    }
    int lo = 0, hi = p.groups;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] * feat_tiles <= tile) lo = mid; else hi = mid;
    }
    const int n = before[lo + 1] - before[lo], local = tile - before[lo] * feat_tiles;
    t.group = lo;
    t.f = local / n;
    t.tok0 = edge[lo] + local % n * p.tok;
    t.tok_end = min(edge[lo + 1], t.tok0 + p.tok);
    return t;
}

// 16 lanes x 32 columns: lane (g, t) gives, for the eight columns of step j, columns 2 t, 2 t + 1 of row g and then of row g + 8
__device__ __forceinline__ void tmem_st_16x256b_x4(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
          "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

// A place in a ring and the parity of the round it is in, for what comes `by` places further each time (a division by a ring's length, which is not a
// constant, costs a converting warp as much as the conversion).
struct Ring {
    int at;
    uint32_t phase;
    __device__ __forceinline__ void move(int by, int length) {
        at += by;
        while (at >= length) at -= length, phase ^= 1;
    }
};

// Where a tile of features begins along K: each elsewhere, so that the blocks that share rows of x do not all read the same lines of L2 at the same
// time (2,048 rows, 3,584 x 3,584: 55 us where all begin at 0, 48 with this).
__device__ __forceinline__ int first_pair(int f, int feat_tiles, int n_pairs) { return (int)((long long)f * n_pairs / feat_tiles); }
__device__ __forceinline__ int turned(int pair, int turn, int n_pairs) { return pair + turn < n_pairs ? pair + turn : pair + turn - n_pairs; }

__device__ __forceinline__ void commit_at(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// A lane's 16 bytes of codes (features g and g + 8) times their scales, in the order of a 16x256b store.  A code + 8 in the upper four of a
// bfloat16's seven fraction bits, behind the exponent of 16, is the number 24 + code; one multiplication and addition brings
// (24 + code) s - 24 s, in which both products are exact (24 has two significant bits, s five) and so is the sum.
template <bool HALF>
__device__ __forceinline__ void unpack(uint32_t (&v)[16], const uint4& c, const uint32_t* sc) {
    const __nv_bfloat162 minus24(__ushort_as_bfloat16(0xc1c0), __ushort_as_bfloat16(0xc1c0));
    auto of = [](uint32_t w, uint32_t s, __nv_bfloat162 off) {
        const uint32_t n = (w & 0x00780078u) | 0x41804180u;
        const __nv_bfloat162 r = __hfma2(*(const __nv_bfloat162*)&n, *(const __nv_bfloat162*)&s, off);
        return *(const uint32_t*)&r;
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t s2 = sc[HALF ? h : 0], lo = __byte_perm(s2, 0, 0x1010), hi = __byte_perm(s2, 0, 0x3232);
        const __nv_bfloat162 lo24 = __hmul2(*(const __nv_bfloat162*)&lo, minus24), hi24 = __hmul2(*(const __nv_bfloat162*)&hi, minus24);
        const uint32_t a = h ? c.y : c.x, b = h ? c.w : c.z;
        v[8 * h] = of(a << 3, lo, lo24), v[8 * h + 1] = of(a >> 1, lo, lo24);
        v[8 * h + 2] = of(b << 3, hi, hi24), v[8 * h + 3] = of(b >> 1, hi, hi24);
        v[8 * h + 4] = of(a >> 5, lo, lo24), v[8 * h + 5] = of(a >> 9, lo, lo24);
        v[8 * h + 6] = of(b >> 5, hi, hi24), v[8 * h + 7] = of(b >> 9, hi, hi24);
    }
}

// each(j) for the 16 columns of a step of the epilogue, or for the first `left` of them: none of the whole ones asks for its place
template <typename F>
__device__ __forceinline__ void columns(int left, F&& each) {
    if (left >= 16) {
#pragma unroll
        for (int j = 0; j < 16; ++j) each(j);
    } else {
#pragma unroll
        for (int j = 0; j < 15; ++j)
            if (j < left) each(j);
    }
}

template <bool GATED, bool HALF>
__global__ void __launch_bounds__(THREADS, 1) gemm_q4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const Args p) {
    constexpr int FEAT = GATED ? 64 : 128;                         // features a tile takes
    constexpr int PIECE = q4::piece_bytes(HALF), TILE = q4::tile_bytes(HALF);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* code_ring = smem + (size_t)p.stages * 2 * p.x_bytes;
    uint64_t* full = (uint64_t*)(code_ring + CODE_STAGES * 2 * TILE);       // [stages] x has landed and the weights lie in tensor memory
    uint64_t* empty = full + MAX_STAGES;          // [stages] the products have read both
    uint64_t* code_full = empty + MAX_STAGES;     // [CODE_STAGES] codes have landed
    uint64_t* code_empty = code_full + CODE_STAGES;                         // [CODE_STAGES] a set has read them
    uint64_t* acc_full = code_empty + CODE_STAGES;     // [accs]
    uint64_t* acc_empty = acc_full + 2;
    uint2* told = (uint2*)(acc_empty + 2);        // [stages] the loading warp's word to the products: their shape, and whether the pair has two blocks
    uint32_t* tmem_slot = (uint32_t*)(told + MAX_STAGES);
    __shared__ int before[MAX_GROUPS + 1];        // tiles of rows of the groups before
    __shared__ int edge[MAX_GROUPS + 1];          // where the groups' rows begin
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) mbar_init(&full[s], 1 + 8), mbar_init(&empty[s], 1);
        for (int s = 0; s < CODE_STAGES; ++s) mbar_init(&code_full[s], 1), mbar_init(&code_empty[s], 8);
        for (int s = 0; s < p.accs; ++s) mbar_init(&acc_full[s], 1), mbar_init(&acc_empty[s], EPI_WARPS);
        fence_barrier_init();
    }
    if (warp == PRODUCT) tmem_alloc(tmem_slot, 512);
    if (p.offsets) {
        cj::after_predecessor();
        if (warp == EPI0) {
            int carry = 0;
            for (int g0 = 0; g0 < p.groups; g0 += 32) {
                const int g = g0 + lane;
                int n = 0;
                if (g < p.groups) {
                    const int begin = min(max(0, p.offsets[g]), p.rows), end = min(max(0, p.offsets[g + 1]), p.rows);
                    n = (max(0, end - begin) + p.tok - 1) / p.tok;
                    edge[g] = begin;
                    if (g + 1 == p.groups) edge[p.groups] = end;
                }
                int inc = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += v;
                }
                if (g < p.groups) before[g] = carry + inc - n;
                carry += __shfl_sync(0xffffffffu, inc, 31);
            }
            if (lane == 0) before[p.groups] = carry;
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    // (tensor memory is held: a following kernel's blocks may be set up beside this one)
    cj::release_successor();
    const uint32_t tmem = *tmem_slot;
    const int feat_tiles = (p.features + FEAT - 1) / FEAT, tiles_f = (p.features + 127) / 128, n_kb = (p.K + 63) / 64;
    const int n_pairs = (n_kb + 1) / 2;
    const int total = (p.offsets ? before[p.groups] : (p.rows + p.tok - 1) / p.tok) * feat_tiles;
    const int my_tiles = (int)blockIdx.x < total ? (total - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;
    const uint32_t acc0 = p.stages * SLOT_COLS;

    if (warp < LOAD_CODES) {
        // ---- x: one warp the even pairs of blocks of K, one the odd (what one thread has under way in bulk loads is bounded)
        if (elect_one()) {
            if (warp == LOAD_X) tma_prefetch_descriptor(&map_x);
            if (!p.offsets) cj::after_predecessor();
            int pair = warp - LOAD_X;
            Ring st{0, 0};
            st.move(pair, p.stages);
            bool ok = true;
            for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
                const Tile t = tile_of(p, tile, feat_tiles, before, edge);
                const int turn = first_pair(t.f, feat_tiles, n_pairs);
                const uint32_t idesc = umma_idesc_bf16(128, min(p.tok, (t.tok_end - t.tok0 + 15) & ~15));
                for (; pair < n_pairs; pair += 2, st.move(2, p.stages)) {
                    const int at = turned(pair, turn, n_pairs);
                    uint8_t* dst = smem + (size_t)st.at * 2 * p.x_bytes;
                    ok = mbar_wait(&empty[st.at], st.phase ^ 1, 1);
                    if (!ok) break;
                    const bool two = 2 * at + 1 < n_kb;
                    told[st.at] = make_uint2(idesc, two);
                    mbar_expect_tx(&full[st.at], two ? 2 * p.x_bytes : p.x_bytes);
                    tma_load_2d(dst, &map_x, &full[st.at], at * 128, t.tok0);
                    if (two) tma_load_2d(dst + p.x_bytes, &map_x, &full[st.at], at * 128 + 64, t.tok0);
                }
                pair -= n_pairs;
            }
        }
    } else if (warp == LOAD_CODES) {
        // ---- codes: weights are written by no kernel of a step, so that a dense product's leave before the wait for the kernel that makes x
        if (elect_one()) {
            Ring st{0, 0};
            bool ok = true, settled = p.offsets != nullptr;
            for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x) {
                const Tile t = tile_of(p, tile, feat_tiles, before, edge);
                const int turn = first_pair(t.f, feat_tiles, n_pairs);
                for (int pair = 0; pair < n_pairs; ++pair, st.move(1, CODE_STAGES)) {
                    if (!settled && st.phase) cj::after_predecessor(), settled = true;      // (from the second round on, places wait for products)
                    const int kb = 2 * turned(pair, turn, n_pairs), blocks = min(2, n_kb - kb);
                    uint8_t* dst = code_ring + st.at * 2 * TILE;
                    uint64_t* bar = &code_full[st.at];
                    ok = mbar_wait(&code_empty[st.at], st.phase ^ 1, 8);
                    if (!ok) break;
                    mbar_expect_tx(bar, blocks * TILE);
                    if (GATED) {
                        // of each block the gate's four pieces and the other weight's
                        const size_t at = (((size_t)t.group * tiles_f + (t.f >> 1)) * n_kb + kb) * TILE + (t.f & 1) * 4 * PIECE;
                        for (int b = 0; b < blocks; ++b) {
                            bulk_load(smem_u32(dst + b * TILE), p.w + at + b * TILE, 4 * PIECE, bar);
                            bulk_load(smem_u32(dst + b * TILE + 4 * PIECE), p.w_up + at + b * TILE, 4 * PIECE, bar);
                        }
                    } else
                        bulk_load(smem_u32(dst), p.w + (((size_t)t.group * tiles_f + t.f) * n_kb + kb) * TILE, blocks * TILE, bar);
                }
            }
        }
    } else if (warp == PRODUCT) {
        // ---- products (no wait with a limit begins before the kernel that makes x is done: how long that takes is not this kernel's to say)
        if (!p.offsets) cj::after_predecessor();
        if (elect_one()) {
            // One thread's instructions come one after the other, four clocks and more each, beside those of the warps that share its scheduler: waits, commits and
            // sums are for two blocks of K at a time, and the loop keeps addresses and descriptors instead of working them out of a place in a ring.
            const uint32_t full0 = smem_u32(full), full_end = full0 + 8 * p.stages;
            const uint64_t desc0 = umma_desc_sw128(smem);
            const uint32_t desc_half = (uint32_t)p.x_bytes >> 4, desc_step = 2 * desc_half;
            uint32_t bar = full0, phase = 0, at_tmem = tmem;
            uint64_t desc = desc0;
            Ring ac{0, 0};
            bool ok = true;
            for (int left = my_tiles; left > 0 && ok; --left) {
                for (int pair0 = 0; pair0 < n_pairs && ok; pair0 += p.part_pairs) {
                    ok = mbar_wait(&acc_empty[ac.at], ac.phase ^ 1, 2);
                    if (!ok) break;
                    const uint32_t acc = tmem + acc0 + ac.at * p.tok;
                    const int end = min(pair0 + p.part_pairs, n_pairs);
                    for (int pair = pair0; pair < end; ++pair) {
                        if (!mbar_try_wait_at(bar, phase)) ok = mbar_wait_slow(full + ((bar - full0) >> 3), phase, 3);
                        if (!ok) break;
                        tcgen05_fence_after();
                        const uint2 of = told[(bar - full0) >> 3];
                        const uint32_t idesc = of.x;
                        umma_bf16_a_tmem(acc, at_tmem, desc, idesc, pair > pair0 ? 1u : 0u);
                        umma_bf16_a_tmem(acc, at_tmem + 8, desc + 2, idesc, 1);
                        umma_bf16_a_tmem(acc, at_tmem + 16, desc + 4, idesc, 1);
                        umma_bf16_a_tmem(acc, at_tmem + 24, desc + 6, idesc, 1);
                        if (of.y) {
                            umma_bf16_a_tmem(acc, at_tmem + 32, desc + desc_half, idesc, 1);
                            umma_bf16_a_tmem(acc, at_tmem + 40, desc + desc_half + 2, idesc, 1);
                            umma_bf16_a_tmem(acc, at_tmem + 48, desc + desc_half + 4, idesc, 1);
                            umma_bf16_a_tmem(acc, at_tmem + 56, desc + desc_half + 6, idesc, 1);
                        }
                        commit_at(bar + 8 * MAX_STAGES);
                        bar += 8, desc += desc_step, at_tmem += SLOT_COLS;
                        if (bar == full_end) bar = full0, desc = desc0, at_tmem = tmem, phase ^= 1;
                    }
                    if (!ok) break;
                    umma_commit(&acc_full[ac.at]);
                    ac.move(1, p.accs);
                }
            }
        }
    } else if (warp >= CONV0) {
        // ---- codes to bfloat16: of a pair of blocks of K two pieces of 16 features a warp, into the 16 lanes of tensor memory that are the
        // pieces' rows (two sets of eight warps take the pairs in turn: one waits, loads and stores while the other computes)
        const int q = warp & 3, upper = (warp - CONV0) >> 2 & 1;   // the quarter of the lanes this warp may touch, and which half of it
        const int set = (warp - CONV0) >> 3;
        const uint32_t lanes = (uint32_t)(q * 32 + upper * 16) << 16;
        const uint8_t* mine = code_ring + (GATED ? upper * 4 + q : q * 2 + upper) * PIECE;
        Ring st{set, 0}, sl{0, 0};
        sl.move(set, p.stages);
        bool settled = p.offsets != nullptr;
        for (int left = my_tiles * n_pairs - set; left > 0; left -= CONV_SETS, st.move(CONV_SETS, CODE_STAGES), sl.move(CONV_SETS, p.stages)) {
            if (!settled && sl.phase) cj::after_predecessor(), settled = true;
            if (!mbar_wait_warp(&code_full[st.at], st.phase, 5)) break;
            // (where a pair has one block, what lies there is put down for the other and nobody reads it)
            const uint8_t* src = mine + st.at * 2 * TILE;
            const uint4 c0 = *(const uint4*)(src + lane * 16), c1 = *(const uint4*)(src + TILE + lane * 16);
            constexpr int SCALES = HALF ? 2 : 1;
            uint32_t sc[2 * SCALES];
#pragma unroll
            for (int h = 0; h < 2 * SCALES; ++h)
                sc[h] = *(const uint32_t*)(src + (h / SCALES) * TILE + 512 + (h % SCALES * 8 + (lane >> 2)) * 4);
            __syncwarp();
            if (lane == 0) mbar_arrive(&code_empty[st.at]);
            uint32_t v[16];
            unpack<HALF>(v, c0, sc);
            if (!mbar_wait_warp(&empty[sl.at], sl.phase ^ 1, 6)) break;
            tcgen05_fence_after();
            tmem_st_16x256b_x4(tmem + sl.at * SLOT_COLS + lanes, v);
            unpack<HALF>(v, c1, sc + SCALES);
            tmem_st_16x256b_x4(tmem + sl.at * SLOT_COLS + HALF_COLS + lanes, v);
            tmem_st_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[sl.at]);
        }
    } else {
        // ---- epilogue: two warps a quarter of the lanes, 16 columns in turn; a lane is a feature, columns are rows of x
        if (!p.offsets) cj::after_predecessor();
        const int q = warp & 3;
        Ring ac{0, 0};
        bool ok = true;
        for (int tile = blockIdx.x; tile < total && ok; tile += gridDim.x)
        for (int pair = 0; pair < n_pairs; pair += p.part_pairs, ac.move(1, p.accs)) {
            const Tile t = tile_of(p, tile, feat_tiles, before, edge);
            const int as = ac.at;
            const bool add = p.accumulate || pair > 0;
            ok = mbar_wait_warp(&acc_full[as], ac.phase, 7);
            if (!ok) break;
            tcgen05_fence_after();
            const uint32_t src = tmem + acc0 + as * p.tok + ((uint32_t)(q * 32) << 16);
            const int n = t.tok_end - t.tok0;
            const int feature = GATED ? t.f * 64 + q * 16 + (lane & 15) : t.f * 128 + q * 32 + lane;
            const bool in = feature < p.features;
            const float bias = !GATED && p.bias && in && pair == 0 ? p.bias[feature] : 0.0f;
#pragma unroll 1
            for (int c0 = ((warp - EPI0) >> 2) * 16; c0 < n; c0 += 4 * EPI_WARPS) {
                uint32_t v[16];
                tmem_ld16(src + c0, v);
                tmem_ld_wait();
                if (GATED) {
                    // lanes 0 .. 15 hold the gate's sums, 16 .. 31 the other weight's: the lower take the first eight rows, the upper the others
                    const bool low = lane < 16;
                    const int first = c0 + (low ? 0 : 8);
                    __nv_bfloat16* dst = (__nv_bfloat16*)p.out + (size_t)(t.tok0 + first) * p.ldo + feature;
                    float* dst32 = (float*)p.out + (size_t)(t.tok0 + first) * p.ldo + feature;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float mine = __uint_as_float(low ? v[j] : v[8 + j]);
                        const float other = __shfl_xor_sync(0xffffffffu, __uint_as_float(low ? v[8 + j] : v[j]), 16);
                        const float y = cj::gated_act_fast(low ? mine : other, low ? other : mine, 0.0f, 1.0f, 0.0f);
                        if (in && first + j < n) {
                            if (p.half_out) dst[(size_t)j * p.ldo] = __float2bfloat16_rn(y);
                            else dst32[(size_t)j * p.ldo] = y;
                        }
                    }
                } else if (in) {
                    // (adding by a reduction in L2: nobody else writes these entries, so the sums are those of a load, an addition and a store in
                    // their order, without the wait for the load)
                    const int left = n - c0;
                    if (p.half_out) {
                        __nv_bfloat16* dst = (__nv_bfloat16*)p.out + (size_t)(t.tok0 + c0) * p.ldo + feature;
                        columns(left, [&](int j) { dst[j * p.ldo] = __float2bfloat16_rn(__uint_as_float(v[j]) + bias); });
                    } else {
                        float* dst = (float*)p.out + (size_t)(t.tok0 + c0) * p.ldo + feature;
                        if (add) columns(left, [&](int j) {
                            asm volatile("red.global.add.f32 [%0], %1;" ::"l"(dst + j * p.ldo), "f"(__uint_as_float(v[j]) + bias) : "memory");
                        });
                        else columns(left, [&](int j) { dst[j * p.ldo] = __uint_as_float(v[j]) + bias; });
                    }
                }
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[as]);
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == PRODUCT) {
        tcgen05_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// The rows that a mixture's groups read, side by side: out[s] = x[index[s]], zeros where there is no such row.  A warp a row.
__global__ void __launch_bounds__(256) q4_gather_kernel(uint4* __restrict__ out, const __nv_bfloat16* __restrict__ x, long long ldx, int x_rows,
                                                        const int* __restrict__ index, int rows, int n16) {
    cj::after_predecessor();
    cj::release_successor();
    const int s = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (s >= rows) return;
    const int r = index[s];
    const uint4* src = r >= 0 && r < x_rows ? (const uint4*)(x + (size_t)r * ldx) : nullptr;
    for (int i = threadIdx.x & 31; i < n16; i += 32) out[(size_t)s * n16 + i] = src ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
}

}  // namespace

// x bf16 [x_rows, ldx] -> out bf16 [rows, K]; x, ldx, K and out of 16 bytes
CJ_EXPORT int cj_q4_gather(const void* x, long long ldx, int x_rows, const int* index, void* out, int rows, int K, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (!x || !index || !out || K <= 0 || x_rows <= 0) return CJ_ERR_ARG;
    if ((K & 7) || (ldx & 7) || (((uintptr_t)x | (uintptr_t)out) & 15)) return CJ_ERR_ALIGN;
    cj::launch(q4_gather_kernel, dim3((rows + 7) / 8), dim3(256), 0, stream, (uint4*)out, (const __nv_bfloat16*)x, ldx, x_rows, index, rows, K / 8);
    return cj::launch_status();
}

// As cj_gemm_q4, without gathered rows: row s of out comes from row s of x (x_rows of them; rows past the last are zeros).  x and ldx
// of 16 bytes; tok: rows of x a tile takes, a multiple of 16 from 16 to 256.
CJ_EXPORT int cj_gemm_q4_tc(const void* x, long long ldx, int x_rows, const void* w, const void* w_up, const float* bias, void* out, int out_dtype,
                            long long ldo, int rows, int features, int K, int groups, int half, const int* offsets, int accumulate, int tok,
                            int sms, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (!x || !w || !out || features <= 0 || K <= 0 || groups <= 0 || x_rows <= 0 || sms <= 0) return CJ_ERR_ARG;
    if (out_dtype != CJ_F32 && out_dtype != CJ_BF16) return CJ_ERR_DTYPE;
    if (accumulate && (out_dtype != CJ_F32 || w_up)) return CJ_ERR_DTYPE;
    if ((w_up && bias) || (!offsets && groups != 1)) return CJ_ERR_ARG;
    if ((ldx & 7) || ldx < K || ((uintptr_t)x & 15) || (((uintptr_t)w | (uintptr_t)w_up) & 15)) return CJ_ERR_ALIGN;
    if (groups > MAX_GROUPS || tok < 16 || tok > 256 || tok % 16 != 0) return CJ_ERR_SIZE;
    const int feat_tiles = (features + (w_up ? 63 : 127)) / (w_up ? 64 : 128);
    if ((long long)feat_tiles * ((rows + 15) / 16 + groups) > 0x7fffffffLL) return CJ_ERR_SIZE;
    CUtensorMap map;
    if (!make_map_bf16(&map, x, x_rows, K, ldx, tok)) return CJ_ERR_ARG;
    Args a{(const uint8_t*)w, (const uint8_t*)w_up, bias, out, offsets, ldo, rows, features, K, groups, out_dtype == CJ_BF16 ? 1 : 0, accumulate,
           tok, 0, 0, tok * 128, 0};
    const int n_pairs = (K + 127) / 128, parts = out_dtype == CJ_F32 && !w_up ? (n_pairs + 19) / 20 : 1;
    a.part_pairs = (n_pairs + parts - 1) / parts;
    const int code_ring = CODE_STAGES * 2 * q4::tile_bytes(half != 0);
    // two accumulators where the weights of two pairs fit beside them
    a.accs = 2 * tok + 2 * SLOT_COLS <= 512 ? 2 : 1;
    a.stages = min(min(MAX_STAGES, (512 - a.accs * tok) / SLOT_COLS), (SMEM_LIMIT - 1024 - BAR_BYTES - code_ring) / (2 * a.x_bytes));
    const int smem = a.stages * 2 * a.x_bytes + code_ring + BAR_BYTES + 1024;
    const long long most = offsets ? sms : (long long)feat_tiles * ((rows + tok - 1) / tok);
    auto kern = w_up ? (half ? gemm_q4_tc_kernel<true, true> : gemm_q4_tc_kernel<true, false>)
                     : (half ? gemm_q4_tc_kernel<false, true> : gemm_q4_tc_kernel<false, false>);
    // (the most that any call asks for: the attribute is the kernel's, and another thread may set it between here and the launch)
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT);
    if (e != cudaSuccess) return (int)e;
    cj::launch(kern, dim3((unsigned)(most < sms ? most : sms)), dim3(THREADS), smem, stream, map, a);
    return cj::launch_status();
}

CJ_EXPORT int cj_gemm_q4_tc_error() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, tc::g_error_flag, sizeof(int)) != cudaSuccess) return -1;
    return v;
}
