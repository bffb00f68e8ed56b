// Attention of portions of prompts over the 8-bit cache (cache_e4m3.cu) on the 5th-generation tensor cores (tcgen05), heads of 64 or 128.
//
// A block takes 256 query rows of one request and one query head, as two tiles of 128 rows that share every tile of 128 keys and values:
//     S = q . (code_k 2^e_k)^T        scores [128 x 128] in tensor memory
//     P = exp2(S scale - m)           four warps a query tile, a row a thread; P as bfloat16 over the columns of its scores
//     O += P . (code_v 2^e_v)         O in tensor memory
// A code times its power of two is a bfloat16 number exactly, whatever the exponents of the tokens beside it (f16 would keep more bits of P,
// but only values within 22 octaves of each other: a row's values could vanish beside larger ones that it does not even see).  So six warps
// turn codes into the bfloat16 tiles in shared memory that both products read, and the rest is attention over a bfloat16 cache: P, as there, is
// the one rounding.  The codes come by bulk copies of a page's run of rows, pages of any size, one warp's work: a tile's keys travel while its
// predecessor's values are converted (half the bytes of a bfloat16 cache: 16 KB a tile; plain loads into registers, tried first, held the
// conversions of the tile before up: 2,048 rows behind 4,096, 28 heads over 4 of 128: 290 us where this takes 240).  The two query tiles take turns between the exponential unit and the tensor
// core, each key tile is worked on as two halves of 64 keys, and the reference maximum moves only when it grows by more than 2^8.
// Where row blocks are few, two or four blocks - a cluster - take neighbouring stretches of the key tiles and join their outputs through each other's
// shared memory (512 rows behind 4,096, 16 heads: 109 us alone, 66 in two, 42 in four; 100 behind 8,000, 28 heads: 165, 94, 54).
// Bound, with blocks for all SMs, by what follows on one another in a key tile (3 us: exponentials 1.1, conversions, two products) and by the last
// round of blocks.  Every wait is bounded (tc_common.cuh).
#define CJ_LIB "attention_e4m3_tc"
#include "common.cuh"
#include "e4m3.cuh"
#include "tc_common.cuh"

using namespace tc;

namespace {

constexpr int BM = 128, QT = 2, BN = 128;         // query rows a tile, tiles a block, keys a tile
constexpr int STAGES = 2;
constexpr int CONV_WARPS = 6, LOADER = 6, PRODUCT = 7, SOFT0 = 8;
constexpr int THREADS = 16 * 32;
constexpr int HALF_BYTES = 128 * 64 * 2;          // [128 x 64] bfloat16, swizzled: 16 KB
constexpr float RESCALE_THRESHOLD = 8.0f;         // in log2 units
constexpr uint32_t TM_S = 0, TM_O = 256, TM_COLS = 512;

template <int HD>
struct Smem {
    static constexpr int TILE = HALF_BYTES * (HD / 64);
    static constexpr int Q = 0, K = QT * TILE, V = K + STAGES * TILE;
    static constexpr int CODES = V + STAGES * TILE, FACTORS = CODES + 2 * BN * HD, BAR = FACTORS + 2 * BN * 4;      // a tile's keys, and its values
    static constexpr int TOTAL = BAR + 256 + 1024;
};

struct Args {
    const __nv_bfloat16* q;
    __nv_bfloat16* out;
    const uint8_t *kplane, *vplane, *kexp, *vexp;
    const int *req_start, *req_prior, *table;
    int n_requests, table_stride, page_tokens, page_shift, n_pages, n_heads, n_kv, window;      // page_shift: -1 for a page of no power of two
    float scale_log2;
    int total_rows, block_rows, splits;      // splits: blocks of a cluster that share the keys of a row block, 1, 2 or 4
};

struct QueryTile {
    int rows, p0, begin, end;      // rows of the step (0: empty), position of the first, key tiles [begin, end] of the block's
};

__device__ __forceinline__ uint32_t of_block(const void* p, int rank) {      // what lies at p, in the cluster's block `rank`
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}

// The codes of a word that are NaN (0x7f and 0xff) made zeros; whether there were any
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ bool drop_nan(uint32_t& w) {
    const uint32_t hit = nan_codes(w);
    w &= ~((hit >> 7) * 0xffu);
    return hit != 0;
}

// the first position that a row at `pos` sees
__device__ __forceinline__ int from_of(int pos, int window) { return window > 0 && pos >= window ? pos - window + 1 : 0; }

// bits lo .. hi of a word, those of them that it has
__device__ __forceinline__ uint32_t within(int lo, int hi) {
    lo = max(lo, 0), hi = min(hi, 31);
    return lo <= hi ? 0xffffffffu >> (31 - (hi - lo)) << lo : 0u;
}

// four codes times a power of two, as bfloat16
__device__ __forceinline__ uint2 scaled_codes(uint32_t w, f32x2 f) {
    uint32_t lo, hi;
    cj::e4m3x4_to_f16(w, lo, hi);
    const float2 a = __half22float2(*(const __half2*)&lo), b = __half22float2(*(const __half2*)&hi);
    const float2 x = unpack2(mul2(pack2(a.x, a.y), f)), y = unpack2(mul2(pack2(b.x, b.y), f));
    const __nv_bfloat162 u = __floats2bfloat162_rn(x.x, x.y), v = __floats2bfloat162_rn(y.x, y.y);
    return make_uint2(*(const uint32_t*)&u, *(const uint32_t*)&v);
}

template <int HD>
__global__ void __launch_bounds__(THREADS, 1) prefill_e4m3_tc_kernel(const __grid_constant__ CUtensorMap map_q, const Args p) {
    using S = Smem<HD>;
    constexpr int TILE = S::TILE;
    // blocks beyond the portions' row blocks leave before anything else (a captured step's layout has room for more than it brings)
    cj::after_predecessor();
    {
        int tiles = 0;
        for (int r = threadIdx.x & 31; r < p.n_requests; r += 32)
            tiles += (__ldcg(p.req_start + r + 1) - __ldcg(p.req_start + r) + p.block_rows - 1) / p.block_rows;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
        if ((int)blockIdx.y >= tiles) return;
    }
    // the last row blocks of every request first: they see the most keys
    int req = -1, row0 = 0, rows = 0;
    {
        int b = (int)blockIdx.y;
        for (int level = 0; req < 0; ++level) {
            bool any = false;
            for (int r = 0; r < p.n_requests; ++r) {
                const int lo = p.req_start[r], n = p.req_start[r + 1] - lo;
                const int tiles = (n + p.block_rows - 1) / p.block_rows;
                if (tiles <= level) continue;
                any = true;
                if (b-- == 0) {
                    req = r;
                    row0 = lo + (tiles - 1 - level) * p.block_rows;
                    rows = min(p.block_rows, lo + n - row0);
                    break;
                }
            }
            if (!any) return;
        }
    }
    rows = min(rows, p.total_rows - row0);
    if (rows <= 0) return;
    const int h = blockIdx.x, kvh = h / (p.n_heads / p.n_kv);
    const int p0 = p.req_prior[req] + (row0 - p.req_start[req]);
    // (rows before the first position or behind the table's last page have a tile of the table too, in which they see no key)
    const int last_key = p.table_stride * p.page_tokens - 1, p_last = min(p0 + rows - 1, last_key);
    const int key_from = from_of(p0, p.window);
    auto tile_of = [&](int key) { return min(max(key, 0), last_key) / BN; };
    int kt_begin = tile_of(key_from);
    QueryTile qt[QT];
#pragma unroll
    for (int g = 0; g < QT; ++g) {
        qt[g].rows = max(0, min(BM, rows - g * BM));
        qt[g].p0 = p0 + g * BM;
        qt[g].begin = tile_of(from_of(qt[g].p0, p.window)) - kt_begin;
        qt[g].end = qt[g].rows > 0 ? tile_of(qt[g].p0 + qt[g].rows - 1) - kt_begin : qt[g].begin - 1;
    }
    int n_tiles = max(qt[0].end, qt[1].end) + 1;
    // a cluster's blocks take neighbouring stretches of the key tiles and join their results; where that would leave less than two tiles each the first
    // does it alone
    const int rank = blockIdx.z;
    const bool joined = p.splits > 1 && n_tiles >= 2 * p.splits;
    if (joined) {
        const int lo = rank * n_tiles / p.splits, hi = (rank + 1) * n_tiles / p.splits;
        kt_begin += lo;
        n_tiles = hi - lo;
#pragma unroll
        for (int g = 0; g < QT; ++g) qt[g].begin = max(qt[g].begin - lo, 0), qt[g].end = min(qt[g].end - lo, n_tiles - 1);
    } else if (rank > 0)
        return;
    const int* tab = p.table + (size_t)req * p.table_stride;

    __shared__ int place[7];               // first row, rows, whether the block joins others and more (for the end: registers are short between)
    // A weight of 0 times a value of NaN is NaN, for rows that do not see the key.  In key tiles that some rows see part of, NaN among the values are put
    // down as zeros, and written at the end to the rows that see them.
    __shared__ int dropped;
    // Which keys of a tile are there, a bit each.  Four tiles: the loader writes tile i's when the keys of i - 1 are converted, so when the scores
    // of i - 3 are done, which follow the products that read the weights of i - 4.
    __shared__ uint4 there[4];
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = (uint64_t*)(smem + S::BAR);
    uint64_t* q_full = bars;                      // the queries have landed
    uint64_t* k_full = bars + 1;                  // [STAGES]
    uint64_t* k_empty = k_full + STAGES;
    uint64_t* v_full = k_empty + STAGES;
    uint64_t* v_empty = v_full + STAGES;
    uint64_t* s_full = v_empty + STAGES;          // [QT] a query tile's scores are complete (and every product before them)
    uint64_t* p_full = s_full + QT;               // [QT][2] the weights of a tile's first / last 64 keys are written
    uint64_t* half_done = p_full + 2 * QT;        // [QT] the output product over a tile's first 64 keys is done
    uint64_t* o_done = half_done + QT;            // [QT] the last output product is done
    uint64_t* c_full = o_done + QT;               // [2] a tile's codes (of keys, of values) have landed, their powers of two are written
    uint64_t* c_empty = c_full + 2;               // [2] they are converted
    uint32_t* tmem_slot = (uint32_t*)(c_empty + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        place[0] = row0, place[1] = rows, place[2] = joined, place[3] = p0, place[4] = kt_begin, place[5] = n_tiles, place[6] = req;
        dropped = 0;
        for (int s = 0; s < 2; ++s) mbar_init(&c_full[s], 1), mbar_init(&c_empty[s], CONV_WARPS);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&k_full[s], CONV_WARPS * 32), mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], CONV_WARPS * 32), mbar_init(&v_empty[s], 1);
        }
        for (int g = 0; g < QT; ++g) {
            mbar_init(&s_full[g], 1), mbar_init(&half_done[g], 1), mbar_init(&o_done[g], 1);
            mbar_init(&p_full[2 * g], BM), mbar_init(&p_full[2 * g + 1], BM);
        }
        fence_barrier_init();
    }
    if (warp == PRODUCT) tmem_alloc(tmem_slot, TM_COLS);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    cj::release_successor();
    const uint32_t tmem_base = *tmem_slot;

    if (warp < CONV_WARPS) {
        // ---- codes -> bfloat16 tiles: 16 codes of a row a lane, in the order the products want the tiles: K0, V0, K1, V1, ...
        constexpr int PIECES = HD / 16, ROWS_WARP = 32 / PIECES, ROWS_PASS = CONV_WARPS * ROWS_WARP, PASSES = (BN + ROWS_PASS - 1) / ROWS_PASS;
        // (eight lanes that are served together take two rows and, of eight pieces, other halves of them: no two in one bank, coming or going)
        const int in_warp = PIECES == 8 ? lane >> 2 & 3 : lane >> 2;
        const int piece = PIECES == 8 ? ((lane & 3) | (lane >> 4 << 2)) ^ ((in_warp & 1) << 2) : lane & 3;
        const int chunk = (piece & 3) * 2, r0 = warp * ROWS_WARP + in_warp;
        const float* factors = (const float*)(smem + S::FACTORS);
        // key tiles [all_from, all_to) are seen whole by every row
        const int all_from = from_of(p0 + rows - 1, p.window), all_to = p0 + 1;
        bool ok = true;
        for (int i = 0; i < 2 * n_tiles && ok; ++i) {
            const int values = i & 1, t = i >> 1, s = t % STAGES;
            ok = mbar_wait_warp(&c_full[values], t & 1, 10) && mbar_wait_warp(values ? &v_empty[s] : &k_empty[s], ((t / STAGES) & 1) ^ 1, 11);
            if (!ok) break;
            const uint8_t* codes = smem + S::CODES + values * BN * HD + piece * 16;
            uint8_t* dst = smem + (values ? S::V : S::K) + s * TILE + (piece >> 2) * HALF_BYTES;
            // (where the codes lie, each lane its own: a branch among the conversions costs the tiles that need none 5 %)
            if (values && ((kt_begin + t) * BN < all_from || (kt_begin + t + 1) * BN > all_to)) {
#pragma unroll 1
                for (int r = r0; r < BN; r += ROWS_PASS) {
                    uint4* at = (uint4*)(smem + S::CODES + (BN + r) * HD + piece * 16);
                    uint4 c = *at;
                    const bool x = drop_nan(c.x), y = drop_nan(c.y), z = drop_nan(c.z), w = drop_nan(c.w);
                    if ((x || y || z || w) && factors[BN + r] != 0.0f) *at = c, dropped = 1;
                }
            }
            // (the passes' chains side by side: all loads first, and only the last pass may have no row)
            uint4 c[PASSES];
            float scale[PASSES];
#pragma unroll
            for (int j = 0; j < PASSES; ++j) {
                const int r = min(r0 + j * ROWS_PASS, BN - 1);
                c[j] = *(const uint4*)(codes + r * HD);
                scale[j] = factors[values * BN + r];
            }
#pragma unroll
            for (int j = 0; j < PASSES; ++j) {
                const int r = r0 + j * ROWS_PASS;
                if (scale[j] == 0.0f) c[j] = make_uint4(0u, 0u, 0u, 0u);    // (no key: the codes are what was there before)
                const f32x2 f = pack2(scale[j], scale[j]);
                const uint2 a = scaled_codes(c[j].x, f), b = scaled_codes(c[j].y, f), d = scaled_codes(c[j].z, f), e = scaled_codes(c[j].w, f);
                if (j < PASSES - 1 || r < BN) {
                    *(uint4*)(dst + r * 128 + ((chunk ^ (r & 7)) << 4)) = make_uint4(a.x, a.y, b.x, b.y);
                    *(uint4*)(dst + r * 128 + (((chunk + 1) ^ (r & 7)) << 4)) = make_uint4(d.x, d.y, e.x, e.y);
                }
            }
            fence_async_shared();
            mbar_arrive(values ? &v_full[s] : &k_full[s]);
            __syncwarp();
            if (lane == 0) mbar_arrive(&c_empty[values]);
        }
    } else if (warp == LOADER) {
        // ---- look-ups and copies: lane l has keys l, l + 32, ... of a tile; the first key of a page's run (within 32) copies it
        float* factors = (float*)(smem + S::FACTORS);
        int page[4], at_page[4];
        auto ask_pages = [&](int i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = (kt_begin + i) * BN + j * 32 + lane;
                const int n = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_tokens;
                at_page[j] = key - n * p.page_tokens;
                page[j] = key >= key_from && key <= p_last ? __ldg(tab + n) : -1;
            }
        };
        ask_pages(0);
        bool ok = true;
        for (int i = 0; i < n_tiles && ok; ++i) {
            int row[4], run[4], have = 0;
            uint32_t keys[4];
            uint32_t ek[4], ev[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = (kt_begin + i) * BN + j * 32 + lane;
                row[j] = page[j] >= 0 && page[j] < p.n_pages ? (page[j] * p.n_kv + kvh) * p.page_tokens + at_page[j] : -1;
                ek[j] = row[j] >= 0 ? p.kexp[row[j]] : 0;
                ev[j] = row[j] >= 0 ? p.vexp[row[j]] : 0;
                const bool first = row[j] >= 0 && (lane == 0 || at_page[j] == 0 || key == key_from);
                run[j] = first ? min(min(p.page_tokens - at_page[j], 32 - lane), p_last + 1 - key) : 0;
                keys[j] = __ballot_sync(0xffffffffu, row[j] >= 0);
                have += __popc(keys[j]);
            }
            if (i + 1 < n_tiles) ask_pages(i + 1);
#pragma unroll
            for (int values = 0; values < 2; ++values) {
                if (ok) ok = mbar_wait_warp(&c_empty[values], (i & 1) ^ 1, 12);
                if (!ok) break;
#pragma unroll
                for (int j = 0; j < 4; ++j) factors[values * BN + j * 32 + lane] = __uint_as_float((values ? ev[j] : ek[j]) << 23);
                if (values == 0 && lane == 0) there[i & 3] = make_uint4(keys[0], keys[1], keys[2], keys[3]);
                __syncwarp();
                if (lane == 0) mbar_expect_tx(&c_full[values], have * HD);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (run[j] > 0)
                        bulk_load(smem_u32(smem + S::CODES + (values * BN + j * 32 + lane) * HD), (values ? p.vplane : p.kplane) + (size_t)row[j] * HD,
                                  run[j] * HD, &c_full[values]);
            }
        }
        // (the copies under way end before the block does: the converting warps wait for each, unless a wait ran out)
        if (!ok)
            for (int values = 0; values < 2; ++values) mbar_wait_warp(&c_full[values], 0, 14), mbar_wait_warp(&c_full[values], 1, 14);
    } else if (warp == PRODUCT) {
        // ---- products, in the order S_a(0) S_b(0), then per key tile i: PV_a(i) S_a(i + 1) PV_b(i) S_b(i + 1), each PV in two halves of
        // 64 keys.  S_g(i + 1) overwrites the columns PV_g(i) reads P from; one thread's products run in the order they were issued
        if (elect_one()) {
            // rows [row0, row0 + 256) of the [rows, heads x HD] view, columns of this head (rows past the step's end read as zero)
            const int q_tiles = qt[1].rows > 0 ? 2 : 1;
            mbar_expect_tx(q_full, q_tiles * TILE);
            for (int g = 0; g < q_tiles; ++g)
                for (int half = 0; half < HD / 64; ++half)
                    tma_load_2d(smem + S::Q + g * TILE + half * HALF_BYTES, &map_q, q_full, h * HD + half * 64, row0 + g * BM);
            bool ok = mbar_wait(q_full, 0, 12);
            int p_seen[QT] = {0, 0};
            auto uses = [&](int g, int i) { return i >= qt[g].begin && i <= qt[g].end; };
            auto scores = [&](int g, int i) {
                const int s = i % STAGES;
                const uint32_t acc = tmem_base + TM_S + g * BN;
#pragma unroll
                for (int half = 0; half < HD / 64; ++half) {
                    const uint64_t dq = umma_desc_sw128(smem + S::Q + g * TILE + half * HALF_BYTES);
                    const uint64_t dk = umma_desc_sw128(smem + S::K + s * TILE + half * HALF_BYTES);
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_bf16(acc, dq + 2 * k, dk + 2 * k, umma_idesc_bf16(128, BN), (half | k) ? 1u : 0u);
                }
                umma_commit(&s_full[g]);
            };
            if (ok) ok = mbar_wait(&k_full[0], 0, 13);
            if (ok) {
                tcgen05_fence_after();
#pragma unroll
                for (int g = 0; g < QT; ++g)
                    if (uses(g, 0)) scores(g, 0);
                umma_commit(&k_empty[0]);
            }
            for (int i = 0; i < n_tiles && ok; ++i) {
                const int s = i % STAGES;
                const bool next = i + 1 < n_tiles;
                ok = mbar_wait(&v_full[s], (i / STAGES) & 1, 19);
                if (!ok) break;
                const uint64_t dv = umma_desc_mn_sw128(smem + S::V + s * TILE, HALF_BYTES);
                bool k_there = false;
#pragma unroll
                for (int g = 0; g < QT; ++g) {
                    if (!ok) break;
                    if (uses(g, i)) {
                        const uint32_t acc = tmem_base + TM_O + g * HD, pa = tmem_base + TM_S + g * BN;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            ok = mbar_wait(&p_full[2 * g + half], p_seen[g] & 1, 15);
                            if (!ok) break;
                            tcgen05_fence_after();
                            // 16 keys are 8 columns of P and two 8-row groups of V (2048 bytes); B is MN-major (bit 16)
#pragma unroll
                            for (int k = 4 * half; k < 4 * half + 4; ++k)
                                umma_bf16_a_tmem(acc, pa + 8 * k, dv + (uint64_t)(k * 2048 >> 4), umma_idesc_bf16(128, HD) | (1u << 16),
                                                 (i > qt[g].begin || k > 0) ? 1u : 0u);
                            if (half == 0) umma_commit(&half_done[g]);
                        }
                        if (!ok) break;
                        ++p_seen[g];
                        if (i == qt[g].end) umma_commit(&o_done[g]);
                    }
                    if (g == QT - 1) umma_commit(&v_empty[s]);
                    if (next && (uses(g, i + 1) || g == QT - 1)) {
                        if (!k_there) {
                            ok = mbar_wait(&k_full[(i + 1) % STAGES], ((i + 1) / STAGES) & 1, 13);
                            if (!ok) break;
                            tcgen05_fence_after();
                            k_there = true;
                        }
                        if (uses(g, i + 1)) scores(g, i + 1);
                        if (g == QT - 1) umma_commit(&k_empty[(i + 1) % STAGES]);
                    }
                }
            }
        }
    } else {
        // ---- softmax of one query tile, a row a thread ------------------------------------------------------------
        const int g = (warp - SOFT0) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const QueryTile mine = g == 0 ? qt[0] : qt[1];
        const int pos = mine.p0 + r, from = from_of(pos, p.window);
        const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
        const uint32_t s_addr = tmem_base + TM_S + g * BN + lane_off, o_addr = tmem_base + TM_O + g * HD + lane_off;
        float m_ref = -INFINITY, l = 0.0f;
        bool ok = true, seen = false;
        const int n_mine = mine.end - mine.begin + 1;
        for (int j = 0; j < n_mine && ok; ++j) {
            ok = mbar_wait_warp(&s_full[g], j & 1, 16);
            if (!ok) break;
            tcgen05_fence_after();
            const int kbase = (kt_begin + mine.begin + j) * BN;
            const uint32_t* present = (const uint32_t*)&there[(mine.begin + j) & 3];
            const bool whole = from <= kbase && pos >= kbase + BN - 1 && (present[0] & present[1] & present[2] & present[3]) == 0xffffffffu;
            seen = seen || whole;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                constexpr int HC = BN / 2;
                uint32_t v[HC];
                tmem_ld32<0>(s_addr + half * HC, v);
                tmem_ld32<32>(s_addr + half * HC + 32, v);
                tmem_ld_wait();
                if (!whole) {
                    // a bit for each key this row sees: one of its range that is there
                    const uint32_t see0 = within(from - kbase - half * HC, pos - kbase - half * HC) & present[2 * half];
                    const uint32_t see1 = within(from - kbase - half * HC - 32, pos - kbase - half * HC - 32) & present[2 * half + 1];
                    seen = seen || (see0 | see1) != 0;
#pragma unroll
                    for (int c = 0; c < HC; ++c)
                        if (!((c < 32 ? see0 : see1) >> (c & 31) & 1)) v[c] = 0xff800000u;       // -inf
                }
                // The largest score first, in four chains of three-way maxima, then one pass of exponentials.  (One pass with the reference
                // maximum so far, which finds the largest on its way and is repeated where that moves the reference, is shorter by the wait for
                // the maximum, but a warp repeats it for any of its 32 rows: keys of uneven lengths, 2,048 rows behind 4,096, took 300 us.)
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < HC; c += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], __uint_as_float(v[c + 2 * k]), __uint_as_float(v[c + 2 * k + 1]));
                const float largest = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * p.scale_log2;
                const bool rescale = largest > m_ref + RESCALE_THRESHOLD && m_ref != -INFINITY;
                const float m_use = rescale || m_ref == -INFINITY ? fmaxf(m_ref, largest) : m_ref;
                const float factor = rescale ? exp2f(m_ref - m_use) : 1.0f;
                const float neg_sub = m_use == -INFINITY ? 0.0f : -m_use;
                const f32x2 scale2 = pack2(p.scale_log2, p.scale_log2), sub2 = pack2(neg_sub, neg_sub);
                f32x2 sum2a = pack2(0.0f, 0.0f), sum2b = sum2a;
                uint32_t packed[HC / 2];
#pragma unroll
                for (int c = 0; c < HC; c += 4) {
                    const float2 t0 = unpack2(fma2(pack2(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), scale2, sub2));
                    const float2 t1 = unpack2(fma2(pack2(__uint_as_float(v[c + 2]), __uint_as_float(v[c + 3])), scale2, sub2));
                    const float e0 = ex2(t0.x), e1 = ex2(t0.y), e2 = ex2(t1.x), e3 = ex2(t1.y);
                    sum2a = add2(sum2a, pack2(e0, e1));
                    sum2b = add2(sum2b, pack2(e2, e3));
                    const __nv_bfloat162 b0 = __floats2bfloat162_rn(e0, e1), b1 = __floats2bfloat162_rn(e2, e3);
                    packed[c >> 1] = *(const uint32_t*)&b0;
                    packed[(c >> 1) + 1] = *(const uint32_t*)&b1;
                }
                const float2 sa = unpack2(sum2a), sb = unpack2(sum2b);
                const float sum = (sa.x + sa.y) + (sb.x + sb.y);
                tmem_st32<0>(s_addr + half * (HC / 2), packed);
                l = l * factor + sum;
                m_ref = m_use;
                // O may be rescaled once the product before is done (that over the last tile's second half was before this tile's scores were)
                if (half == 1) {
                    ok = mbar_wait_warp(&half_done[g], j & 1, 17);
                    if (!ok) break;
                    tcgen05_fence_after();
                }
                if (__any_sync(0xffffffffu, rescale)) {        // rare
#pragma unroll 1
                    for (int c0 = 0; c0 < HD; c0 += 16) {
                        uint32_t o[16];
                        tmem_ld16(o_addr + c0, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int q = 0; q < 16; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * factor);
                        tmem_st16(o_addr + c0, o);
                    }
                }
                tmem_st_wait();
                tcgen05_fence_before();
                mbar_arrive(&p_full[2 * g + half]);
            }
        }
        // ---- the rows' results ----------------------------------------------------------------------------------
        if (ok && n_mine > 0) ok = mbar_wait_warp(&o_done[g], 0, 18);
        tcgen05_fence_after();
        // a row whose keys leave no weight at all has scores of -infinity alone (an infinite query's): a softmax of NaN, not the zeros of a row without keys
        if (seen && l == 0.0f) l = NAN;
        if (place[2]) {
            // for the cluster: O as it is, over the tiles of keys and values (both query tiles are done with them), 16-byte chunks turned by the row so
            // that a warp's rows lie in different banks; the rows' reference maxima and sums over the codes
            asm volatile("bar.sync 1, %0;" ::"n"(QT * BM) : "memory");
            float* dst = (float*)(smem + S::K) + (g * BM + r) * HD;
            const int turn = r & (HD / 4 - 1);
            ((float2*)(smem + S::CODES))[g * BM + r] = make_float2(m_ref, ok ? l : 0.0f);
#pragma unroll 1
            for (int c0 = 0; c0 < HD && n_mine > 0; c0 += 16) {
                uint32_t o[16];
                tmem_ld16(o_addr + c0, o);
                tmem_ld_wait();
#pragma unroll
                for (int q = 0; q < 4; ++q) *(uint4*)(dst + (((c0 >> 2) + q) ^ turn) * 4) = make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
            }
        } else if (ok && n_mine > 0) {
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
            __nv_bfloat16* dst = p.out + ((size_t)(place[0] + g * BM + r) * p.n_heads + blockIdx.x) * HD;
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += 16) {
                uint32_t o[16];
                tmem_ld16(o_addr + c0, o);
                tmem_ld_wait();
                if (g * BM + r < place[1]) {
                    uint4 u[2];
                    __nv_bfloat162* b = (__nv_bfloat162*)u;
#pragma unroll
                    for (int q = 0; q < 8; ++q) b[q] = __floats2bfloat162_rn(__uint_as_float(o[2 * q]) * inv, __uint_as_float(o[2 * q + 1]) * inv);
                    *(uint4*)(dst + c0) = u[0];
                    *(uint4*)(dst + c0 + 8) = u[1];
                }
            }
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (place[2]) {
        cluster_sync();
        const int first_row = place[0], n_rows = place[1];
        // the rows dealt to the cluster's blocks: a warp a row, four entries a lane, the blocks' results in their order
        const int share = QT * BM / p.splits;
        for (int i = warp; i < share; i += THREADS / 32) {
            const int row = (int)blockIdx.z * share + i;
            if (row >= n_rows) break;
            float2 ml[4];
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                ml[b] = make_float2(-INFINITY, 0.0f);
                if (b < p.splits)
                    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml[b].x), "=f"(ml[b].y)
                                 : "r"(of_block((float2*)(smem + S::CODES) + row, b)) : "memory");
                M = fmaxf(M, ml[b].x);
            }
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (lane < HD / 4) {
                const float* src = (const float*)(smem + S::K) + row * HD + (lane ^ (row & (HD / 4 - 1))) * 4;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    if (ml[b].y == 0.0f) continue;      // (no key of this block's; NaN scores leave a maximum of -infinity and a sum of NaN)
                    float4 v;
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(of_block(src, b)) : "memory");
                    const float f = exp2f(ml[b].x - M);
                    L = fmaf(ml[b].y, f, L);
                    a.x = fmaf(v.x, f, a.x), a.y = fmaf(v.y, f, a.y), a.z = fmaf(v.z, f, a.z), a.w = fmaf(v.w, f, a.w);
                }
                const float inv = L > 0.0f || L != L ? 1.0f / L : 0.0f;
                const __nv_bfloat162 x = __floats2bfloat162_rn(a.x * inv, a.y * inv), y = __floats2bfloat162_rn(a.z * inv, a.w * inv);
                *(uint2*)(p.out + ((size_t)(first_row + row) * p.n_heads + blockIdx.x) * HD + lane * 4) = make_uint2(*(const uint32_t*)&x, *(const uint32_t*)&y);
            }
        }
        cluster_sync();                    // (the others may still read this block's shared memory)
    }
    if (dropped) {                         // rare: a warp a key, the rows that see it
        const int first_row = place[0], n_rows = place[1], pos0 = place[3], key0 = place[4] * BN, end = min(pos0 + n_rows, p.table_stride * p.page_tokens);
        for (int key = key0 + warp; key < min(key0 + place[5] * BN, end); key += THREADS / 32) {
            if (key < from_of(pos0, p.window)) continue;
            const int tile0 = key / BN * BN, page = p.table[(size_t)place[6] * p.table_stride + key / p.page_tokens];
            if ((tile0 >= from_of(pos0 + n_rows - 1, p.window) && tile0 + BN <= pos0 + 1) || page < 0 || page >= p.n_pages) continue;
            const size_t at = ((size_t)(page * p.n_kv + blockIdx.x / (p.n_heads / p.n_kv)) * p.page_tokens + key % p.page_tokens) * HD;
            const int to = p.window > 0 && key - pos0 < n_rows - p.window ? key - pos0 + p.window : n_rows;
            for (int d = lane; d < HD; d += 32)
                if (nan_codes(p.vplane[at + d]) & 0x80)
                    for (int r = max(0, key - pos0); r < to; ++r) p.out[((size_t)(first_row + r) * p.n_heads + blockIdx.x) * HD + d] = __float2bfloat16_rn(NAN);
        }
    }
    if (warp == PRODUCT) {
        tcgen05_fence_after();
        tmem_dealloc(tmem_base, TM_COLS);
    }
}

}  // namespace

// q, out: bf16 [total_rows, n_heads, hd]; the cache as cj_append_e4m3 writes it; rows req_start[r] .. req_start[r + 1] are request r's
// from position req_prior[r] on.  hd: 64 or 128; scale > 0.
CJ_EXPORT int cj_prefill_e4m3_tc(const void* q, void* out, const void* kplane, const void* vplane, const void* kexp, const void* vexp, int n_pages,
                                 const int* req_start, const int* req_prior, int n_requests, int total_rows, const int* table, int table_stride,
                                 int page_tokens, int n_heads, int n_kv, int hd, int window, float scale, int sms,
                                 cudaStream_t stream) {
    if (total_rows <= 0 || n_requests <= 0) return 0;
    if (!q || !out || !kplane || !vplane || !kexp || !vexp || !req_start || !req_prior || !table) return CJ_ERR_ARG;
    if (n_heads <= 0 || n_kv <= 0 || n_heads % n_kv != 0 || page_tokens <= 0 || n_pages <= 0 || window < 0 || !(scale > 0.0f)) return CJ_ERR_SIZE;
    if (hd != 64 && hd != 128) return CJ_ERR_SIZE;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)kplane | (uintptr_t)vplane) & 15) return CJ_ERR_ALIGN;
    if ((long long)n_pages * n_kv * page_tokens > 0x7fffffffLL || (long long)table_stride * page_tokens > 0x7fffffffLL - 256) return CJ_ERR_SIZE;
    // 256 rows a block; where that leaves SMs without one two or four blocks share a row block's keys (a cluster), and where they still do 128 rows
    // (us, 256 rows alone, in four, 128 alone, in four: 64 rows behind 2,000, 16 heads, 52, 24, 52, 24; 200 behind 300, heads of 64, 18, 18, 15, 16; 256 behind
    // 1,024, 28 heads, 40, 23, 35, 38: more blocks than SMs)
    const long long blocks = ((long long)(total_rows + 255) / 256 + n_requests - 1) * n_heads;
    const int splits = 4 * blocks <= sms ? 4 : 2 * blocks <= sms ? 2 : 1, block_rows = 2 * splits * blocks <= sms ? 128 : 256;
    const long long row_blocks = ((long long)total_rows + block_rows - 1) / block_rows + n_requests;
    if (row_blocks > 65535) return CJ_ERR_SIZE;
    CUtensorMap map_q;
    if (!make_map_bf16(&map_q, q, total_rows, (long long)n_heads * hd, (long long)n_heads * hd, BM)) return CJ_ERR_ARG;
    const Args a{(const __nv_bfloat16*)q, (__nv_bfloat16*)out, (const uint8_t*)kplane, (const uint8_t*)vplane, (const uint8_t*)kexp,
                 (const uint8_t*)vexp, req_start, req_prior, table, n_requests, table_stride, page_tokens,
                 (page_tokens & (page_tokens - 1)) == 0 ? __builtin_ctz(page_tokens) : -1, n_pages, n_heads, n_kv, window,
                 scale * 1.4426950408889634f, total_rows, block_rows, splits};
    auto kern = hd == 128 ? prefill_e4m3_tc_kernel<128> : prefill_e4m3_tc_kernel<64>;
    const int smem = hd == 128 ? Smem<128>::TOTAL : Smem<64>::TOTAL;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n_heads, (unsigned)row_blocks, splits);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = splits;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cj::overlap_launches() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kern, map_q, a);
    return cj::launch_status();
}

CJ_EXPORT int cj_prefill_e4m3_tc_error() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, tc::g_error_flag, sizeof(int)) != cudaSuccess) return -1;
    return v;
}
