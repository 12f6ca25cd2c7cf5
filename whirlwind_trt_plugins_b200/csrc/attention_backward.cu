// attention_backward.cu -- ww_cross_attention_backward on the 5th-generation
// tensor cores.
//
//   P  = 2^(x - lse2)                x, lse2 the scores and their log sum in log2 units
//   dP = dO V^T,  dS = P (dP - delta),  delta = rowsum(dO * O)
//   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K,  dtable[b] = sum of dS over bucket b
//
// Two kernels of one form, each forming S and dP for itself, so that every sum
// is owned by one CTA and none needs atomics (the same call gives the same
// bits):
//   keys:     128 keys on the rows (S^T, dP^T), streaming 64 queries at a time
//             over all query heads of the key head; dV and dK in TMEM
//   queries:  128 queries on the rows, streaming 64 keys at a time; dQ in TMEM
// The row operands are A operands in TMEM (in shared memory where the accumulators
// leave no room: keys at D = 128), which keeps their re-reading for
// every tile off the shared memory; each streamed tile is the K-major B operand
// of the two score products and, unchanged, the MN-major B operand of the
// accumulating ones; P and dS return to TMEM over S and dP as A operands.  Two
// tiles are under way on an SM, each with two warpgroups of elementwise work (32 of
// its 64 columns each): of two CTAs, whose starts and ends overlap as well, or of
// one where the accumulators take half of TMEM.
//
// 16-bit ranges: P is kept as 2^6 P, dS in fp16 as 2^(6 + e) dS.  delta is a mean of
// dP, so |dP - delta| <= M = 2 |dO row| max |v row| over the valid keys; e is chosen
// with 2^8 <= 2^e M < 2^9, which keeps 2^(6 + e) |dS| below 2^15 whatever the values
// are (P <= 1 up to its rounding) and leaves half of fp16's smallest step at 2^-39 M:
// neither large values nor gradients as small as a mean over a batch leaves them fall
// out of its range.  Over queries a row has its own M, over keys M is the batch item's.
// The row norms come from the kernel that forms delta.  Powers of two, taken out again
// at the end.
//
// Bound: per 128 x 64 tile 512 clocks of exponentials (16 per clock and SM) in
// each kernel against 8 D (dK, dV) and 6 D (dQ) clocks of products.
// Measured: a map of 4800, 8 heads of 128, bf16 with a bias: 340 us for the
// gradients, 690 TFLOP/s of the five products (seven are formed; 311 us in short
// runs); 1200 to 1777 tokens, 4 x 16 heads of 64 on 4: 100 us; 1080 heads of 32 in
// rows of 320, fp16, masked, with a bias: 296 us, of them 20 for deltas and norms; a
// CTA of five tiles spends 4000 of its 17000 clocks (5800 of 21600 over queries) before
// its first tile.
// The two kernels do not need each other: `queries` is launched behind `keys` and
// takes the SMs that its last round leaves (rows of 320, forward and gradients:
// 16 us less than one after the other; the order that it then needs by hand, see `seen`,
// takes 4 of them), then one join for both.
//
// dtable: a tile whose positions all lie in one bucket adds its plain sum.
// Otherwise dS goes through shared memory in fp32, 32 columns at a time (rounded as
// for its product, the errors of dtable are half as large again and rows of 320 take
// 353 us in place of 367); a thread sums one diagonal j - i (one read and one add per
// value, no conflicts), diagonals are collected per CTA and joined to buckets, CTAs
// and warpgroups in order.
#include "attention.cuh"
#include "tensor_map.cuh"
#include "umma.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

namespace ww {
namespace {

constexpr int kRows = 128;
constexpr int kCols = 64;
constexpr int kShift = 6;         // P is kept times 2^kShift
constexpr int kPitch = 33;        // words of a row of 32 dS in shared memory

struct BwdParams {
    CUtensorMap q, k, v, dout;  // boxes of 64 tokens
    const void* r1;             // row operands: keys: k, v; queries: q, dout
    const void* r2;
    const int32_t* k_lens;
    const uint8_t* key_mask;
    const void* table;
    const float* nlse2;   // [B * Hq][Lq_pad] kShift - log2 units; -inf: no gradient
    const float* ndelta;  // [B * Hq][Lq_pad]
    const float* norm2;   // fp16: [B * Hq][Lq_pad] |dO row|^2
    const uint32_t* tops; // fp16: [B] bits of max |dO row|^2, max |v row|^2
    uint32_t* seen;       // set by `keys` once it has seen the three above; null where `queries` runs alone
    void* d1;             // keys: dk; queries: dq
    void* d2;             // keys: dv
    float* part;          // split items: [item][split][d1, d2][128][D] fp32
    float* table_part;    // queries: [CTA][buckets]
    RelBuckets rel;
    int64_t r1_strides[3], r2_strides[3];
    int32_t B, Lq, Lk, Hq, Hk, D, Lq_pad;
    int32_t blocks, whole_items, splits, q_tiles;
    Divisor by_block, by_head;
    int32_t q_b, q_h, k_b, k_h, v_b, v_h, g_b, g_h;
    int32_t max_entries;  // relative positions a CTA keeps
    float scale, scale2;
    int* err;
};

template <int DP, bool KEYS>
struct Layout {
    // tiles under way: two in one CTA of an SM, or one in each of two.  Two CTAs need
    // TMEM for their accumulators and, to be fast, for their row operands twice:
    // keys at D = 64, 1200 x 1777 tokens, 4 x 16 heads: one CTA 61 us, two with the row
    // operands in shared memory 112 us; rows of 320, 3 heads of 32: 195 and 143 us.
    static constexpr int kTiles = DP >= (KEYS ? 64 : 128) ? 2 : 1;
    static constexpr int kCtas = 2 / kTiles;
    static constexpr int kGroups = 2 * kTiles;         // warpgroups: two per tile
    static constexpr int kThreads = kGroups * 128 + 64;
    static constexpr int kMmaWarp = kGroups * 4, kLoadWarp = kMmaWarp + 1;
    static constexpr bool kRowsInTmem = !(KEYS && DP == 128);
    static constexpr int kRow = DP == 32 ? 64 : 128;   // bytes of an operand row
    static constexpr int kVals = kRow / 2;
    static constexpr int kChunks = DP * 2 / kRow;
    static constexpr int kRowChunk = kRows * kRow;     // row operand
    static constexpr int kRowBytes = kRows * DP * 2;
    static constexpr int kColChunk = kCols * kRow;     // streamed operand
    static constexpr int kColBytes = kCols * DP * 2;
    // a place is free only when its tile's products are done: one more than tiles under way
    static constexpr int kStages = KEYS && DP == 64 ? 4 : 3;
    static constexpr int kC = kRowsInTmem ? 0 : 2 * kRowBytes;     // stages of C1, C2
    static constexpr int kVec = kC + kStages * 2 * kColBytes;      // KEYS: nlse2, ndelta of 64 queries per stage
    // queries: limits of 64 keys per stage, then flags
    static constexpr int kBar = kVec + (KEYS ? kStages * 2 * kCols * 4 : kStages * (kCols + 4) * 4);
    static constexpr int kBias = kBar + 256;                       // bias tables, see below
    // TMEM columns: S of the tiles, dP of the tiles, accumulators, row operands
    static constexpr int kDp = kTiles * kCols, kAcc1 = 2 * kDp, kAcc2 = kAcc1 + DP, kR1 = kAcc1 + (KEYS ? 2 : 1) * DP,
                         kR2 = kR1 + DP / 2, kColumns = 512 / kCtas;
    static_assert(kR1 + (kRowsInTmem ? DP : 0) <= kColumns, "TMEM");
};

template <int DP, bool KEYS>
struct Bars {
    static constexpr int kStages = Layout<DP, KEYS>::kStages;
    uint64_t r_full, c_full[kStages], c_ready[kStages], c_empty[kStages], s_full[Layout<DP, KEYS>::kTiles],
        p_ready[Layout<DP, KEYS>::kTiles], done;
    uint32_t tmem;
};

// Shared memory after the barriers, with a bias (E = entries, W warpgroups):
//   buckets  [E] bytes
//   KEYS:    values [W][E] floats, rebuilt when the head changes
//   queries: values [E], with the gradient's diagonals [W][E], plain sums
//            [4 W warps][buckets] and dS [W][128][33] floats
__host__ __device__ constexpr int bias_bytes(bool keys, int groups, int entries, int buckets)
{
    const int e = (entries + 15) / 16 * 16;
    return keys ? e + groups * e * 4 : e + (1 + groups) * e * 4 + groups * 4 * buckets * 4 + groups * kRows * kPitch * 4;
}

// Exponent e with 2^8 <= 2^e M < 2^9 for M = 2 sqrt(g2 v2), from the squared norms of a
// row of dO and of the largest row of V; 0 where M is 0 (dS is) or not finite.
__device__ __forceinline__ int ds_exponent(float g2, float v2)
{
    const int m = static_cast<int>(__float_as_uint(2.0f * sqrtf(g2 * v2)) >> 23);  // 127 + that of M
    return m > 0 && m < 255 ? 127 + 8 - m : 0;
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }

template <typename T, int DP, bool KEYS, bool BIAS>
__global__ void __launch_bounds__(Layout<DP, KEYS>::kThreads, Layout<DP, KEYS>::kCtas)
    attention_backward_kernel(const __grid_constant__ BwdParams p)
{
    using L = Layout<DP, KEYS>;
    using Bar = Bars<DP, KEYS>;
    constexpr int S = L::kStages, NT = L::kTiles, kGroups = L::kGroups, kThreads = L::kThreads, kMmaWarp = L::kMmaWarp,
                  kLoadWarp = L::kLoadWarp;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    extern __shared__ uint8_t raw[];
    uint8_t* base = raw + ((1024 - (umma::smem_addr(raw) & 1023)) & 1023);
    const uint32_t sm = umma::smem_addr(base);
    Bar* bar = reinterpret_cast<Bar*>(base + L::kBar);
    const auto at = [](const uint64_t& b) { return umma::smem_addr(&b); };

    // `keys` waits for the grid of the deltas.  `queries` starts while the last CTAs of `keys`
    // run and is not ordered behind that grid by its launch: `keys` passes the order on, by a
    // word that it releases after its wait and `queries` acquires before it reads them
    if (KEYS) wait_for_launches_before();

    // items (row block, head, batch item); the last ones are split over their streamed tiles
    const int blk = blockIdx.x;
    const bool in_parts = blk >= p.whole_items;
    const int split = in_parts ? (blk - p.whole_items) % p.splits : 0, splits = in_parts ? p.splits : 1;
    const int item = in_parts ? p.whole_items + (blk - p.whole_items) / p.splits : blk;
    const int heads = KEYS ? p.Hk : p.Hq, group = p.Hq / p.Hk;
    const int bh = p.by_block.div(item), block = item - bh * p.blocks, b = p.by_head.div(bh), h = bh - b * heads;
    const int row0 = block * kRows;
    const int len = p.k_lens == nullptr ? p.Lk : min(max(__ldg(p.k_lens + b), 0), p.Lk);
    // streamed tiles of this CTA
    const int n_all = KEYS ? (row0 < len ? group * p.q_tiles : 0) : (len + kCols - 1) / kCols;
    int first, n;
    part_of(n_all, split, splits, first, n);

    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;  // warp-uniform: roles branch as warps
    const int wg = warp / 4;
    // the streamed tiles' next load: head (KEYS) and place along the streamed axis
    int load_h = KEYS ? h * group + first / max(p.q_tiles, 1) : h / group, load_at = KEYS ? first % max(p.q_tiles, 1) : first;
    const auto load = [&](int i) {  // one thread of the load warp
        const int s = i % S;
        umma::mbar_arrive_expect_tx(at(bar->c_full[s]), 2 * L::kColBytes + (KEYS ? 2 * kCols * 4 : 0));
        const uint32_t to = sm + L::kC + s * 2 * L::kColBytes;
        const int l = load_at * kCols;
#pragma unroll
        for (int c = 0; c < L::kChunks; ++c) {
            umma::tma_load_4d(to + c * L::kColChunk, KEYS ? &p.q : &p.k, c * L::kVals, load_h * (KEYS ? p.q_h : p.k_h), l,
                              b * (KEYS ? p.q_b : p.k_b), at(bar->c_full[s]));
            umma::tma_load_4d(to + L::kColBytes + c * L::kColChunk, KEYS ? &p.dout : &p.v, c * L::kVals,
                              load_h * (KEYS ? p.g_h : p.v_h), l, b * (KEYS ? p.g_b : p.v_b), at(bar->c_full[s]));
        }
        if (KEYS) {
            const int64_t row = (static_cast<int64_t>(b) * p.Hq + load_h) * p.Lq_pad + l;
            const uint32_t vec = sm + L::kVec + s * 2 * kCols * 4;
            umma::bulk_g2s(vec, p.nlse2 + row, kCols * 4, at(bar->c_full[s]));
            umma::bulk_g2s(vec + kCols * 4, p.ndelta + row, kCols * 4, at(bar->c_full[s]));
        }
        ++load_at;
        if (KEYS && load_at == p.q_tiles) {
            load_at = 0;
            ++load_h;
        }
    };
    if (warp == kLoadWarp && lane == 0) {
        umma::mbar_init(at(bar->r_full), L::kRowsInTmem ? 8 : 1);
        for (int s = 0; s < S; ++s) {
            umma::mbar_init(at(bar->c_full[s]), 1);
            umma::mbar_init(at(bar->c_ready[s]), 1);
            umma::mbar_init(at(bar->c_empty[s]), 1);
        }
        for (int s = 0; s < NT; ++s) {
            umma::mbar_init(at(bar->s_full[s]), 1);
            umma::mbar_init(at(bar->p_ready[s]), 8);  // one arrival per warp
        }
        umma::mbar_init(at(bar->done), 1);
        umma::mbar_fence_init();
        umma::fence_proxy_async_smem();
        if (n > 0) {
            if (!L::kRowsInTmem) {
                // a half of the row tile that lies beyond the tensor reads as zeros like any other place outside
                umma::mbar_arrive_expect_tx(at(bar->r_full), 2 * L::kRowBytes);
                for (int half = 0; half < 2; ++half)
                    for (int c = 0; c < L::kChunks; ++c) {
                        const uint32_t off = c * L::kRowChunk + half * L::kColChunk;
                        const int l = min(row0 + half * kCols, p.Lk);
                        umma::tma_load_4d(sm + off, &p.k, c * L::kVals, h * p.k_h, l, b * p.k_b, at(bar->r_full));
                        umma::tma_load_4d(sm + L::kRowBytes + off, &p.v, c * L::kVals, h * p.v_h, l, b * p.v_b, at(bar->r_full));
                    }
            }
            for (int i = 0; i < S && i < n; ++i) load(i);
        }
    }
    // row operands: warpgroup 0 takes the first, 1 the second, a row per thread; on their way
    // while the rest is set up
    uint32_t rows[L::kRowsInTmem ? DP / 2 : 1];
    if (L::kRowsInTmem && wg < 2 && n > 0) {
        const int row = row0 + threadIdx.x % 128;
        const int64_t* stride = wg == 0 ? p.r1_strides : p.r2_strides;
        const T* from = static_cast<const T*>(wg == 0 ? p.r1 : p.r2) + b * stride[0] + row * stride[1] + h * stride[2];
        const bool live = row < (KEYS ? p.Lk : p.Lq);
#pragma unroll
        for (int c = 0; c < DP; c += 8) {
            uint4 u = make_uint4(0, 0, 0, 0);
            if (live && c < p.D) u = __ldg(reinterpret_cast<const uint4*>(from + c));
            if (L::kRowsInTmem) {
                rows[c / 2] = u.x;
                rows[c / 2 + 1] = u.y;
                rows[c / 2 + 2] = u.z;
                rows[c / 2 + 3] = u.w;
            }
        }
    }
    RelRange range;
    uint8_t* buckets = base + L::kBias;
    float* values = nullptr;  // bias of [range]; KEYS: of this warpgroup's current head
    const int entries = (p.max_entries + 15) / 16 * 16;
    if (BIAS) {
        // positions j - i - offset of the CTA's tiles, padded rows and columns included
        range = KEYS ? rel_range(p.rel, row0 - (p.q_tiles * kCols - 1) - p.rel.q_offset, row0 + kRows - 1 - p.rel.q_offset)
                     : rel_range(p.rel, first * kCols - (row0 + kRows - 1) - p.rel.q_offset,
                                 (first + n) * kCols - 1 - row0 - p.rel.q_offset);
        values = reinterpret_cast<float*>(base + L::kBias + entries) + (KEYS ? min(wg, kGroups - 1) * entries : 0);
        if (n > 0) {
            TableRow<T> table;
            if (!KEYS) table.load(p.rel, p.table, h, lane);
            for (int e0 = warp * 32; warp < kGroups * 4 && e0 < range.count(); e0 += kGroups * 128) {  // the others have their own starts
                const int e = min(e0 + lane, range.count() - 1), bu = rel_bucket(p.rel, range.lo + e);
                buckets[e] = static_cast<uint8_t>(bu);
                if (!KEYS) values[e] = table.get(p.rel, bu);
            }
        }
        if (!KEYS)  // diagonals, then plain sums
            for (int e = threadIdx.x; wg < kGroups && e < kGroups * entries + kGroups * 4 * p.rel.total; e += kGroups * 128)
                values[entries + e] = 0.0f;
    }
    if (KEYS && blk == 0 && threadIdx.x == 0 && p.seen != nullptr) store_release(p.seen, 1);
    if (warp == kMmaWarp) {
        // set before `queries` can start, so the first look finds it
        if (!KEYS && p.seen != nullptr && !wait_acquire(p.seen, 1) && lane == 0) record_device_error(p.err, kErrMbarTimeout | 0x33);
        __syncwarp();
        umma::tmem_alloc(umma::smem_addr(&bar->tmem), L::kColumns);
    }
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = bar->tmem;
    if (KEYS) start_launch_behind();  // this CTA has its TMEM columns
    // queries with masked keys: the load warp clears their rows of K and V before a
    // tile is used (its products then see zeros, whatever the places held) and
    // leaves limits (0 or -inf) that join the scores
    const bool masks = !KEYS && (p.key_mask != nullptr || len % kCols != 0);
    float* limits = reinterpret_cast<float*>(base + L::kVec);
    uint32_t* wholes = reinterpret_cast<uint32_t*>(limits + S * kCols);
    const auto tile_bar = [&](int s) { return masks ? at(bar->c_ready[s]) : at(bar->c_full[s]); };

    if (warp == kLoadWarp) {
        if (n > 0) {
            bool ok = true;
            // tile i's place is free once its products are done, which wait for the tiles
            // up to i + NT - 1: all of them loaded (and cleared) before this waits for it
            const auto next = [&](int i) {
                if (lane != 0 || i < 0 || i + S >= n || !ok) return;
                ok = umma::mbar_poll(at(bar->c_empty[i % S]), (i / S) & 1);
                if (ok) load(i + S);
            };
            for (int i = 0; i < n; ++i) {
                if (!masks) next(i - 1);
                if (!masks) continue;
                const int s = i % S, k0 = (first + i) * kCols;
                uint32_t in_mask = 0;
#pragma unroll
                for (int c = 0; c < kCols; c += 32) {
                    const int key = k0 + c + lane;
                    if (key < len && (p.key_mask == nullptr || __ldg(p.key_mask + static_cast<int64_t>(b) * p.Lk + key) != 0))
                        in_mask |= 1u << (c / 32);
                }
                ok = __shfl_sync(~0u, ok, 0) && umma::mbar_poll(at(bar->c_full[s]), (i / S) & 1);
                bool all = true;
#pragma unroll
                for (int c = 0; c < kCols; c += 32) {
                    const bool in = (in_mask >> (c / 32)) & 1;
                    all = all && in;
                    limits[s * kCols + c + lane] = in ? 0.0f : -INFINITY;
                    if (!in) {
                        const uint32_t to = sm + L::kC + s * 2 * L::kColBytes + (c + lane) * L::kRow;
                        for (int x = 0; x < 2 * L::kChunks; ++x)
#pragma unroll
                            for (int j = 0; j < L::kRow; j += 16) umma::st_shared_v4(to + x * L::kColChunk + j, 0, 0, 0, 0);
                    }
                }
                all = __all_sync(~0u, all);
                if (lane == 0) wholes[s] = all;
                umma::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) umma::mbar_arrive(at(bar->c_ready[s]));
                next(i - 1);
                __syncwarp();
            }
            if (lane == 0 && !ok) record_device_error(p.err, kErrMbarTimeout | 0x30);
        }
    } else if (warp == kMmaWarp) {
        if (n > 0) {
            // the warp runs as a whole, one elected lane issues, everything in uniform
            // registers (see attention_forward.cu)
            constexpr bool bf = !kHalf;
            constexpr uint32_t id_s = umma::idesc_16bit(bf, kRows, kCols, false), id_a = umma::idesc_16bit(bf, kRows, DP, true);
            const uint32_t tm = __reduce_or_sync(~0u, tmem);
            const uint64_t r_desc = umma::smem_desc_swizzled<L::kRow>(sm, 16);
            const uint64_t c_desc = umma::smem_desc_swizzled<L::kRow>(sm + L::kC, 16);
            const uint64_t a_desc = umma::smem_desc_swizzled<L::kRow>(sm + L::kC, L::kColChunk);
            const auto scores = [&](int i) {
                const uint64_t cd = umma::desc_advance(c_desc, i % S * 2 * L::kColBytes);
                const uint32_t to = tm + i % NT * kCols;
                if (umma::elect_one()) {
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int j = 0; j < DP / 16; ++j) {
                            const uint64_t bd = umma::desc_advance(cd, x * L::kColBytes + j * 16 / L::kVals * L::kColChunk +
                                                                           j * 16 % L::kVals * 2);
                            if (L::kRowsInTmem)
                                umma::mma_f16_ts(to + x * L::kDp, tm + (x ? L::kR2 : L::kR1) + j * 8, bd, id_s, j > 0);
                            else
                                umma::mma_f16_ss(to + x * L::kDp,
                                                 umma::desc_advance(r_desc, x * L::kRowBytes + j * 16 / L::kVals * L::kRowChunk +
                                                                                j * 16 % L::kVals * 2),
                                                 bd, id_s, j > 0);
                        }
                    umma::mma_commit(at(bar->s_full[i % NT]));
                }
                __syncwarp();
            };
            bool ok = umma::mbar_poll(at(bar->r_full), 0);
            umma::fence_after_sync();
            for (int i = 0; i < NT && i < n && ok; ++i) {
                ok = umma::mbar_poll(tile_bar(i), 0);
                if (ok) scores(i);
            }
            for (int i = 0; i < n && ok; ++i) {
                ok = umma::mbar_poll(at(bar->p_ready[i % NT]), (i / NT) & 1);
                if (!ok) break;
                umma::fence_after_sync();
                const uint64_t ad = umma::desc_advance(a_desc, i % S * 2 * L::kColBytes);
                const uint32_t from = tm + i % NT * kCols;
                if (umma::elect_one()) {
#pragma unroll
                    for (int j = 0; j < kCols / 16; ++j) {
                        const uint32_t a = from + j / 2 * 32 + j % 2 * 8;  // each warpgroup's 32 values over its own 32 scores
                        umma::mma_f16_ts(tm + L::kAcc1, a + L::kDp, umma::desc_advance(ad, j * 16 * L::kRow), id_a,
                                         i > 0 || j > 0);
                        if (KEYS)
                            umma::mma_f16_ts(tm + L::kAcc2, a,
                                             umma::desc_advance(ad, L::kColBytes + j * 16 * L::kRow), id_a, i > 0 || j > 0);
                    }
                    umma::mma_commit(at(bar->c_empty[i % S]));
                    if (i == n - 1) umma::mma_commit(at(bar->done));
                }
                __syncwarp();
                if (i + NT < n) {
                    ok = umma::mbar_poll(tile_bar((i + NT) % S), ((i + NT) / S) & 1);
                    if (ok) scores(i + NT);
                }
            }
            if (!ok && lane == 0) record_device_error(p.err, kErrMbarTimeout | 0x31);
        }
    } else {
        const int st = wg >> 1, half = wg & 1;  // tile of those under way, columns of it
        const int r = threadIdx.x % 128, row = row0 + r;
        const uint32_t lanes = static_cast<uint32_t>(warp % 4) << 21;
        const uint32_t s_col = tmem + lanes + st * kCols, dp_col = s_col + L::kDp;
        bool ok = true;  // once a wait has run out: no more waits, but every barrier is kept
        if (L::kRowsInTmem && wg < 2 && n > 0) {
#pragma unroll
            for (int c = 0; c < (L::kRowsInTmem ? DP / 2 : 0); c += 16)
                umma::tmem_st16(tmem + lanes + (wg == 0 ? L::kR1 : L::kR2) + c, rows + c);  // two values a column
            umma::tmem_wait_st();
            umma::fence_before_sync();
            __syncwarp();
            if (lane == 0) umma::mbar_arrive(at(bar->r_full));
        }
        // fp16: dS is kept times 2^e too; without tiles nobody may have written the norms, and every
        // sum is 0
        int e = 0;
        bool row_ok = row < (KEYS ? len : p.Lq);
        float my_nlse = -INFINITY, my_ndelta = 0.0f;
        if (KEYS) {
            if (row_ok && p.key_mask != nullptr) row_ok = __ldg(p.key_mask + static_cast<int64_t>(b) * p.Lk + row) != 0;
            if (kHalf && n > 0) e = ds_exponent(f32(__ldcg(p.tops + 2 * b)), f32(__ldcg(p.tops + 2 * b + 1)));
        } else if (row_ok) {
            const int64_t i = (static_cast<int64_t>(b) * p.Hq + h) * p.Lq_pad + row;
            if (kHalf && n > 0) e = ds_exponent(__ldcg(p.norm2 + i), f32(__ldcg(p.tops + 2 * b + 1)));
            my_nlse = __ldcg(p.nlse2 + i) + e;  // P is not needed without its 2^e here
            my_ndelta = __ldcg(p.ndelta + i);
        }
        const float f = power_of_two(e), inv_f = power_of_two(-e);
        const bool any_row = row0 + warp % 4 * 32 < (KEYS ? len : p.Lq);  // else this warp keeps the barriers only
        const Pair scale_2 = pair(p.scale2, p.scale2), f_2 = KEYS ? pair(f, f) : pair(inv_f, inv_f), ndelta_2 = pair(my_ndelta, my_ndelta);
        int built = -1;  // KEYS: head of `values`
        float* diag = values + (1 + wg) * entries;
        float* plain = values + (1 + kGroups) * entries + warp * p.rel.total;
        float* tile = values + (1 + kGroups) * entries + kGroups * 4 * p.rel.total + wg * kRows * kPitch;
        if (BIAS && !KEYS && !any_row)
            for (int j = 0; j < 32; ++j) tile[r * kPitch + j] = 0.0f;
        int ch = h, qt = first + st;  // tile i's head (KEYS) and its place along the streamed axis
        if (KEYS && n > 0) {
            ch = h * group + (first + st) / p.q_tiles;
            qt = (first + st) % p.q_tiles;
        }
        for (int i = st; i < n; i += NT) {
            const int s = i % S, col0 = qt * kCols + half * 32;
            float flat = 0.0f;
            const float* mine = nullptr;  // bias of this row's first column
            int flat_bucket = 0;
            if (BIAS) {
                if (KEYS && built != ch) {
                    warpgroup_sync(wg);
                    TableRow<T> table;
                    table.load(p.rel, p.table, ch, lane);
                    for (int e0 = warp % 4 * 32; e0 < range.count(); e0 += 128) {
                        const int e = min(e0 + lane, range.count() - 1);
                        values[e] = table.get(p.rel, buckets[e]);
                    }
                    warpgroup_sync(wg);
                    built = ch;
                }
                // j - i - offset over these 128 x 32
                const int lo = KEYS ? row0 - (col0 + 31) - p.rel.q_offset : col0 - (row0 + kRows - 1) - p.rel.q_offset;
                flat_bucket = bucket_at(range, buckets, lo);
                if (flat_bucket == bucket_at(range, buckets, lo + kRows + 30))
                    flat = values[min(max(lo, range.lo), range.hi) - range.lo];
                else
                    mine = values + (KEYS ? row - col0 : col0 - row) - p.rel.q_offset - range.lo;
            }
            if (KEYS || masks) ok = ok && umma::mbar_poll(tile_bar(s), (i / S) & 1);  // its vectors or limits
            const bool limited = masks && wholes[s] == 0;
            const float4* lim = reinterpret_cast<const float4*>(limits + s * kCols) + half * 8;
            ok = ok && umma::mbar_poll(at(bar->s_full[st]), (i / NT) & 1);
            umma::fence_after_sync();
            const float4* nlse = reinterpret_cast<const float4*>(base + L::kVec + s * 2 * kCols * 4) + half * 8;
            const float row_add = flat + (KEYS ? 0.0f : my_nlse);
            Pair total = pair(0.0f, 0.0f);
            const bool sums = BIAS && !KEYS;
            if (sums && mine != nullptr) warpgroup_sync(wg);  // the diagonals before have been read
            // W: bias by position, M: limits; resolved outside the unrolled columns
            const auto columns = [&](auto w, auto l) {
                constexpr bool W = decltype(w)::value, M = decltype(l)::value;
                const Pair add_2 = pair(row_add, row_add);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t x[16], d[16], pk[8], dk[8];
                    umma::tmem_ld16(s_col + half * 32 + c * 16, x);
                    umma::tmem_ld16(dp_col + half * 32 + c * 16, d);
                    umma::tmem_wait_ld16(x);
                    umma::tmem_wait_ld16(d);
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        Pair arg = fma2(pair(f32(x[j]), f32(x[j + 1])), scale_2, add_2);
                        Pair nd = ndelta_2;
                        if (KEYS) {
                            const float4 a = nlse[c * 4 + j / 4], e = nlse[kCols / 4 + c * 4 + j / 4];
                            arg = add2(arg, j % 4 == 0 ? pair(a.x, a.y) : pair(a.z, a.w));
                            nd = j % 4 == 0 ? pair(e.x, e.y) : pair(e.z, e.w);
                        }
                        if (M) {
                            const float4 a = lim[c * 4 + j / 4];
                            arg = add2(arg, j % 4 == 0 ? pair(a.x, a.y) : pair(a.z, a.w));
                        }
                        if (W) {
                            const int k = c * 16 + j;
                            arg = add2(arg, KEYS ? pair(mine[-k], mine[-k - 1]) : pair(mine[k], mine[k + 1]));
                        }
                        float p0, p1;
                        if (!BIAS && j % 8 == 6) {  // a quarter on the FMA pipe
                            unpair(exp2_poly<true>(arg), p0, p1);
                        } else {
                            unpair(arg, p0, p1);
                            p0 = exp2_approx(p0);
                            p1 = exp2_approx(p1);
                        }
                        const Pair dp = pair(f32(d[j]), f32(d[j + 1]));
                        Pair ds;
                        if (kHalf && KEYS) ds = mul2(pair(p0, p1), mul2(add2(dp, nd), f_2));
                        else ds = mul2(pair(p0, p1), add2(dp, nd));
                        if (BIAS && !KEYS && !W) total = add2(total, ds);
                        float d0, d1;
                        unpair(ds, d0, d1);
                        if (KEYS) pk[j / 2] = pack2<T>(p0, p1);
                        dk[j / 2] = pack2<T>(d0, d1);
                        if (W && !KEYS) {
                            if (kHalf) unpair(mul2(ds, f_2), d0, d1);  // rows meet in the table's sums: without 2^e
                            tile[r * kPitch + c * 16 + j] = d0;
                            tile[r * kPitch + c * 16 + j + 1] = d1;
                        }
                    }
                    // over columns of this half of the tile only: the other half may not have been read
                    if (KEYS) umma::tmem_st8(s_col + half * 32 + c * 8, pk);
                    umma::tmem_st8(dp_col + half * 32 + c * 8, dk);
                }
            };
            if (any_row) {
                using No = std::false_type;
                if (!KEYS && limited) {
                    if (BIAS && mine != nullptr) columns(std::integral_constant<bool, BIAS>{}, std::integral_constant<bool, !KEYS>{});
                    else columns(No{}, std::integral_constant<bool, !KEYS>{});
                } else {
                    if (BIAS && mine != nullptr) columns(std::integral_constant<bool, BIAS>{}, No{});
                    else columns(No{}, No{});
                }
            }
            umma::tmem_wait_st();
            umma::fence_before_sync();
            __syncwarp();
            if (lane == 0) umma::mbar_arrive(at(bar->p_ready[st]));
            if (sums) {
                if (mine == nullptr) {
                    float t0, t1;
                    unpair(total, t0, t1);
                    t0 = (t0 + t1) * inv_f;
                    for (int o = 16; o > 0; o >>= 1) t0 += __shfl_xor_sync(~0u, t0, o);
                    if (lane == 0) plain[flat_bucket] += t0;
                } else {
                    // sums along j - i: each thread a diagonal, column j of row j + 127 - r;
                    // past the last row, warp 0's threads go on from row 0: diagonal
                    // r - 127 ends, r + 1 begins (r < 31)
                    warpgroup_sync(wg);
                    const float* at0 = tile + (127 - r) * kPitch;
                    float* to = diag + col0 - row0 - p.rel.q_offset - range.lo;
                    if (warp % 4 != 0) {
                        float run[2] = {0.0f, 0.0f};
#pragma unroll
                        for (int j = 0; j < 32; ++j) run[j & 1] += at0[j * (kPitch + 1)];
                        to[r - 127] += run[0] + run[1];
                    } else {
                        float before = 0.0f, after = 0.0f;
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float v = at0[j * (kPitch + 1) - (j <= r ? 0 : kRows * kPitch)];
                            before += j <= r ? v : 0.0f;
                            after += j <= r ? 0.0f : v;
                        }
                        to[r - 127] += before;
                        if (r < 31) to[r + 1] += after;
                    }
                }
            }
            qt += NT;
            if (KEYS)
                while (qt >= p.q_tiles) {
                    qt -= p.q_tiles;
                    ++ch;
                }
        }
        if (n > 0) ok = ok && umma::mbar_poll(at(bar->done), 0);
        umma::fence_after_sync();
        if (!ok) record_device_error(p.err, kErrMbarTimeout | 0x32);
        // the warpgroups share the accumulators' columns (keys: dk, then dv)
        const int rows_of = KEYS ? p.Lk : p.Lq;
        constexpr int kSpan = (KEYS ? 2 : 1) * DP / kGroups;
        const bool second = KEYS && wg >= kGroups / 2;
        const float mul = second ? 1.0f / (1 << kShift) : p.scale / (1 << kShift) * inv_f;
        const int begin = (KEYS ? wg % (kGroups / 2) : wg) * kSpan;
        const uint32_t acc = tmem + lanes + (second ? L::kAcc2 : L::kAcc1) + begin;
        T* to = static_cast<T*>(second ? p.d2 : p.d1) + ((static_cast<int64_t>(b) * rows_of + row) * heads + h) * p.D;
        float* part = p.part + (((static_cast<int64_t>(item - p.whole_items) * p.splits + split) * (KEYS ? 2 : 1) + second) * kRows + r) * p.D;
#pragma unroll
        for (int c = 0; c < kSpan; c += 8) {
            uint32_t o[8];
            const int d0 = begin + c;
            if (n > 0) {
                umma::tmem_ld8(acc + c, o);
                umma::tmem_wait_ld8(o);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = 0;
            }
            if (row >= rows_of || d0 >= p.D) continue;
            if (KEYS && !row_ok) {  // a masked key: 0, whatever its rows held (rows do not mix)
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = 0;
            }
            if (in_parts) {
                *reinterpret_cast<float4*>(part + d0) =
                    make_float4(f32(o[0]) * mul, f32(o[1]) * mul, f32(o[2]) * mul, f32(o[3]) * mul);
                *reinterpret_cast<float4*>(part + d0 + 4) =
                    make_float4(f32(o[4]) * mul, f32(o[5]) * mul, f32(o[6]) * mul, f32(o[7]) * mul);
            } else {
                *reinterpret_cast<uint4*>(to + d0) =
                    make_uint4(pack2<T>(f32(o[0]) * mul, f32(o[1]) * mul), pack2<T>(f32(o[2]) * mul, f32(o[3]) * mul),
                               pack2<T>(f32(o[4]) * mul, f32(o[5]) * mul), pack2<T>(f32(o[6]) * mul, f32(o[7]) * mul));
            }
        }
        umma::fence_before_sync();
    }
    __syncthreads();
    if (warp == kMmaWarp) {
        umma::fence_after_sync();
        umma::tmem_dealloc(tmem, L::kColumns);
    }
    if (BIAS && !KEYS) {
        // buckets of this CTA: 8 lanes run over a bucket's positions
        const float* diag = values + entries;
        const float* plain = values + (1 + kGroups) * entries;
        constexpr float back = 1.0f / (1 << kShift);
        const int sub = lane % 8;
        for (int t0 = warp * 4; t0 < p.rel.total; t0 += kThreads / 8) {
            const int t = min(t0 + lane / 8, p.rel.total - 1);
            float sum = 0.0f;
            if (n > 0) {
                const RelRange x = bucket_positions(p.rel, t);
                const int lo = max(x.lo, range.lo) - range.lo, hi = min(x.hi, range.hi) - range.lo;
                for (int e = lo + sub; e <= hi; e += 8)
#pragma unroll
                    for (int w = 0; w < kGroups; ++w) sum += diag[w * entries + e];
            }
#pragma unroll
            for (int w = 0; w < kGroups * 4; w += 8) sum += plain[(w + sub) * p.rel.total + t];
            for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            if (sub == 0 && t0 + lane / 8 < p.rel.total) p.table_part[static_cast<int64_t>(blk) * p.rel.total + t] = sum * back;
        }
    }
    if (!KEYS) wait_for_launches_before();  // what follows this grid may read what `keys` wrote
}

// -delta = -rowsum(dO * O) and kShift - lse in log2 units, both laid out
// [B * Hq][Lq_pad] with rows of no gradient (lse -inf, padding) at nlse2 = -inf; for fp16
// also |dO row|^2, laid out the same, and each batch item's largest of them and of the
// valid rows of V, which the blocks from first_v on read (an integer maximum of
// non-negative floats: no order; a NaN is above all).  kLanes >= D / 8 lanes per row,
// 8 values each (of V 16).
struct DeltaParams {
    float *nlse2, *ndelta, *norm2;
    uint32_t *tops, *seen;
    int32_t Lq_pad, first_v;
    Divisor by_q, by_v, by_hq, by_hk;  // blocks of a batch item, heads
};

// 8 values as pairs of fp32.
template <typename T>
__device__ __forceinline__ void to_pairs(const uint4& u, Pair (&f)[4])
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const T* e = reinterpret_cast<const T*>(&w[j]);
        f[j] = pair(to_float(e[0]), to_float(e[1]));
    }
}

template <typename T, int kLanes>
__global__ void __launch_bounds__(256) attention_delta_kernel(const __grid_constant__ ww_attention_t a,
                                                              const __grid_constant__ DeltaParams p)
{
    constexpr bool kHalf = std::is_same<T, __half>::value;
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.seen = 0;  // what an earlier call left
    // token of row `row` of a batch item (64-bit divisions would be most of the kernel)
    const auto token_of = [](int64_t row, int64_t rows, const Divisor& heads) {
        return rows <= INT32_MAX - 512 ? heads.div(static_cast<int>(row)) : static_cast<int>(row / heads.d);
    };
    const bool of_v = kHalf && static_cast<int>(blockIdx.x) >= p.first_v;
    float square;
    int b;
    if (!of_v) {
        b = p.by_q.div(blockIdx.x);
        const int lane = threadIdx.x % kLanes;
        const int64_t rows = static_cast<int64_t>(p.Lq_pad) * a.Hq;
        const int64_t row = static_cast<int64_t>(blockIdx.x - b * p.by_q.d) * (256 / kLanes) + threadIdx.x / kLanes;
        const int i = token_of(row, rows, p.by_hq), h = static_cast<int>(row - static_cast<int64_t>(i) * a.Hq);
        const bool live = row < rows && i < a.Lq;
        Pair sums = pair(0.0f, 0.0f), squares = sums;
        if (live && lane * 8 < a.D) {
            const T* g = static_cast<const T*>(a.dout) + b * a.dout_strides[0] + i * a.dout_strides[1] + h * a.dout_strides[2];
            const T* o = static_cast<const T*>(a.out) + (static_cast<int64_t>(b) * a.Lq * a.Hq + row) * a.D;
            Pair gp[4], op[4];
            to_pairs<T>(*reinterpret_cast<const uint4*>(g + lane * 8), gp);
            to_pairs<T>(*reinterpret_cast<const uint4*>(o + lane * 8), op);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sums = fma2(gp[j], op[j], sums);
                if (kHalf) squares = fma2(gp[j], gp[j], squares);
            }
        }
        float sum, other;
        unpair(sums, sum, other);
        sum += other;
        unpair(squares, square, other);
        square += other;
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(~0u, sum, o);
            if (kHalf) square += __shfl_xor_sync(~0u, square, o);
        }
        if (row < rows && lane == 0) {
            const int64_t bh = static_cast<int64_t>(b) * a.Hq + h, to = bh * p.Lq_pad + i;
            const float l = live ? a.lse[bh * a.Lq + i] : -INFINITY;
            p.nlse2[to] = l == -INFINITY ? -INFINITY : kShift - l * kLog2eF;
            p.ndelta[to] = -sum;
            if (kHalf) p.norm2[to] = square;
        }
    } else {
        constexpr int kPer = kLanes / 2;  // lanes of a row: 16 values each
        const int x = blockIdx.x - p.first_v, lane = threadIdx.x % kPer;
        b = p.by_v.div(x);
        const int64_t rows = static_cast<int64_t>(a.Lk) * a.Hk;
        const int64_t row = static_cast<int64_t>(x - b * p.by_v.d) * (256 / kPer) + threadIdx.x / kPer;
        const int j = token_of(row, rows, p.by_hk), h = static_cast<int>(row - static_cast<int64_t>(j) * a.Hk);
        Pair squares = pair(0.0f, 0.0f);
        if (row < rows && j < (a.k_lens == nullptr ? a.Lk : a.k_lens[b]) &&
            (a.key_mask == nullptr || a.key_mask[static_cast<int64_t>(b) * a.Lk + j] != 0)) {
            const T* v = static_cast<const T*>(a.v) + b * a.v_strides[0] + j * a.v_strides[1] + h * a.v_strides[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int d = lane * 16 + c * 8;
                if (d >= a.D) break;
                Pair vp[4];
                to_pairs<T>(*reinterpret_cast<const uint4*>(v + d), vp);
#pragma unroll
                for (int k = 0; k < 4; ++k) squares = fma2(vp[k], vp[k], squares);
            }
        }
        float other;
        unpair(squares, square, other);
        square += other;
#pragma unroll
        for (int o = kPer / 2; o > 0; o >>= 1) square += __shfl_xor_sync(~0u, square, o);
    }
    if (kHalf) {
        __shared__ uint32_t block_top;
        if (threadIdx.x == 0) block_top = 0;
        __syncthreads();
        const uint32_t m = __reduce_max_sync(~0u, __float_as_uint(square) & 0x7fffffffu);
        if (threadIdx.x % 32 == 0) atomicMax(&block_top, m);
        __syncthreads();
        if (threadIdx.x == 0 && block_top > 0) atomicMax(p.tops + 2 * b + of_v, block_top);
    }
}

// Joins the parts of both kernels' split items in order: kSumRows rows of an item
// and output per CTA, 4 values per thread and step.
constexpr int kSumRows = 8;
struct SumParams {
    const float* part;
    void *d1, *d2;
    int32_t count, whole_items, splits, outputs;  // CTAs along x (outputs of split items) and what they join
    int32_t blocks, heads, L;
};

template <typename T>
__global__ void __launch_bounds__(256) attention_sum_kernel(const SumParams keys, const SumParams queries, int D)
{
    wait_for_launches_before();
    const bool second = static_cast<int>(blockIdx.x) >= keys.count;
    const SumParams& p = second ? queries : keys;
    const int x = blockIdx.x - (second ? keys.count : 0);
    const int k = x / p.outputs, which = x % p.outputs, item = p.whole_items + k;
    const int row0 = item % p.blocks * kRows, h = item / p.blocks % p.heads;
    const int64_t b = item / p.blocks / p.heads;
    T* out = static_cast<T*>(which == 0 ? p.d1 : p.d2);
    const int begin = blockIdx.y * kSumRows * D;
    for (int e = begin + threadIdx.x * 4; e < begin + kSumRows * D; e += 256 * 4) {
        const int r = e / D, d = e - r * D;
        if (row0 + r >= p.L) break;
        float4 s = make_float4(0, 0, 0, 0);
#pragma unroll 8
        for (int n = 0; n < p.splits; ++n) {
            const float4 v = *reinterpret_cast<const float4*>(
                p.part + ((static_cast<int64_t>(k) * p.splits + n) * p.outputs + which) * kRows * D + e);
            s.x += v.x;
            s.y += v.y;
            s.z += v.z;
            s.w += v.w;
        }
        *reinterpret_cast<uint2*>(out + ((b * p.L + row0 + r) * p.heads + h) * D + d) =
            make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
    }
}

// Table gradient of one head: the CTAs' buckets in order.  Items are numbered
// (batch item, head, block); those from whole_items on have `splits` CTAs each.
// Each of the 256 warps of a cluster takes every 256th item of the head (item
// numbers grow with n), 32 buckets at a time; then the warps' sums in order, and
// the CTAs'.  1080 items of 3 heads: 12.6 us with one CTA per head.
constexpr int kTableCtas = 8;
template <typename T>
__global__ void __cluster_dims__(kTableCtas, 1, 1) __launch_bounds__(1024)
    attention_table_kernel(const float* part, T* out, int B, int Hq, int blocks, int whole_items, int splits, int total)
{
    __shared__ float sums[32][33], mine[32];
    wait_for_launches_before();
    const auto cluster = cooperative_groups::this_cluster();
    const int rank = blockIdx.x % kTableCtas, h = blockIdx.x / kTableCtas, lane = threadIdx.x % 32,
              t = blockIdx.y * 32 + lane, w = threadIdx.x / 32;
    constexpr int kWarps = 32 * kTableCtas;
    float s = 0.0f;
    if (t < total) {
        const auto item_of = [&](int n) { return (static_cast<int64_t>(n / blocks) * Hq + h) * blocks + n % blocks; };
        int n = w * kTableCtas + rank;
        for (; n + 3 * kWarps < B * blocks && item_of(n + 3 * kWarps) < whole_items; n += 4 * kWarps) {  // loads in flight
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = part[item_of(n + k * kWarps) * total + t];
#pragma unroll
            for (int k = 0; k < 4; ++k) s += v[k];
        }
        for (; n < B * blocks; n += kWarps) {
            const int64_t item = item_of(n);
            const bool one = item < whole_items;
            const int64_t at = one ? item : whole_items + (item - whole_items) * splits;
            const int parts = one ? 1 : splits;
#pragma unroll 8
            for (int k = 0; k < parts; ++k) s += part[(at + k) * total + t];
        }
    }
    sums[w][lane] = s;
    __syncthreads();
    if (w == 0) {
        s = 0.0f;
        for (int n = 0; n < 32; ++n) s += sums[n][lane];
        mine[lane] = s;
    }
    cluster.sync();
    if (rank == 0 && w == 0 && t < total) {
        s = 0.0f;
        for (int n = 0; n < kTableCtas; ++n) s += *cluster.map_shared_rank(mine + lane, n);
        out[h * total + t] = from_float<T>(s);
    }
    cluster.sync();  // until the sums have been read
}

// How one of the two kernels runs: the items that do not fill a round of the
// GPU's CTAs (slots) are split over their streamed tiles.
struct Half {
    int blocks, whole, rest, splits;
    int64_t ctas() const { return i64(whole) + i64(rest) * splits; }
};

Half make_half(int blocks, int64_t items, int64_t tiles, int slots) noexcept
{
    Half r;
    r.blocks = blocks;
    r.rest = static_cast<int>(items % slots);
    r.splits = tail_splits(r.rest, slots, tiles);
    if (r.splits == 1) r.rest = 0;
    r.whole = static_cast<int>(items - r.rest);
    return r;
}

// Both, and where the workspace's parts are.
struct Plan {
    Half q, k;
    int Lq_pad;
    int64_t seen, nlse2, ndelta, norm2, q_part, k_part, table, bytes;  // byte offsets; fp16's largest norms stand first
};

bool make_plan(const ww_attention_t& p, int sms, Plan* plan) noexcept
{
    Plan& r = *plan;
    const int q_blocks = (p.Lq + kRows - 1) / kRows, k_blocks = (p.Lk + kRows - 1) / kRows;
    r.Lq_pad = (p.Lq + kCols - 1) / kCols * kCols;
    const int64_t q_items = i64(q_blocks) * p.B * p.Hq, k_items = i64(k_blocks) * p.B * p.Hk;
    if (q_items > (1 << 30) || k_items > (1 << 30)) return false;
    const int q_slots = sms * (p.D > 64 ? 1 : 2), k_slots = sms * (p.D > 32 ? 1 : 2);  // Layout::kCtas
    r.q = make_half(q_blocks, q_items, (p.Lk + kCols - 1) / kCols, q_slots);
    // `queries` fills what a last round of `keys` leaves free.  Splitting that round is
    // worth its join only where it is under half full (8 heads of a map of 4800, 8 of 148
    // CTAs: split 446 us, else 479; 4 x 4 heads of 1777 keys, 76 CTAs: 151 and 144).
    const bool full = q_items > 0 && k_items % k_slots * 2 >= k_slots;
    r.k = make_half(k_blocks, k_items, full ? 1 : i64(r.Lq_pad / kCols) * (p.Hq / p.Hk), k_slots);
    const int64_t rows = i64(p.B) * p.Hq * r.Lq_pad;
    const int64_t q_part = i64(r.q.rest) * r.q.splits * kRows * p.D * 4, k_part = i64(r.k.rest) * r.k.splits * 2 * kRows * p.D * 4;
    r.seen = i64(p.B) * 8;
    r.nlse2 = (r.seen + 4 + 255) / 256 * 256;
    r.ndelta = r.nlse2 + rows * 4;
    r.norm2 = r.ndelta + rows * 4;
    r.q_part = r.norm2 + (p.dtype == WW_DTYPE_HALF ? rows * 4 : 0);
    r.k_part = r.q_part + q_part;
    r.table = r.k_part + k_part;
    r.bytes = r.table + (p.bias_table != nullptr ? r.q.ctas() * p.num_buckets * 4 : 0);
    return true;
}

template <typename T, int DP, bool KEYS, bool BIAS>
int launch_one(const BwdParams& f, int64_t ctas, bool behind, cudaStream_t stream) noexcept
{
    using L = Layout<DP, KEYS>;
    const auto kernel = attention_backward_kernel<T, DP, KEYS, BIAS>;
    static_assert(!BIAS || 1024 + L::kBias + bias_bytes(KEYS, L::kGroups, kMaxPositions, kMaxBuckets) <= kMaxShared, "shared memory");
    const int bytes = 1024 + L::kBias + (BIAS ? bias_bytes(KEYS, L::kGroups, f.max_entries, f.rel.total) : 0);
    static std::atomic<uint64_t> raised{0};
    if (!allow_shared_memory(reinterpret_cast<const void*>(kernel), raised)) return launch_status("cross_attention_backward");
    if (behind) launch_behind(kernel, dim3(static_cast<unsigned>(ctas)), dim3(L::kThreads), bytes, stream, f);
    else kernel<<<static_cast<unsigned>(ctas), L::kThreads, bytes, stream>>>(f);
    return launch_status("cross_attention_backward");
}

template <typename T, bool KEYS>
int launch(const BwdParams& f, int64_t ctas, bool behind, cudaStream_t stream) noexcept
{
    if (ctas == 0) return WW_SUCCESS;
    const int dp = f.D <= 32 ? 32 : f.D <= 64 ? 64 : 128;
    if (f.table != nullptr)
        return dp == 32 ? launch_one<T, 32, KEYS, true>(f, ctas, behind, stream)
             : dp == 64 ? launch_one<T, 64, KEYS, true>(f, ctas, behind, stream) : launch_one<T, 128, KEYS, true>(f, ctas, behind, stream);
    return dp == 32 ? launch_one<T, 32, KEYS, false>(f, ctas, behind, stream)
         : dp == 64 ? launch_one<T, 64, KEYS, false>(f, ctas, behind, stream) : launch_one<T, 128, KEYS, false>(f, ctas, behind, stream);
}

template <typename T, bool KEYS>
int run_half(BwdParams& f, const Half& half, bool behind, cudaStream_t stream) noexcept
{
    f.blocks = half.blocks;
    f.by_block = make_divisor(half.blocks > 0 ? half.blocks : 1);
    f.by_head = make_divisor(KEYS ? f.Hk : f.Hq);
    f.whole_items = half.whole;
    f.splits = half.splits;
    return launch<T, KEYS>(f, half.ctas(), behind, stream);
}

SumParams sum_params(const Half& half, bool keys, const float* part, void* d1, void* d2, int heads, int L) noexcept
{
    const int outputs = keys ? 2 : 1;
    return {part, d1, d2, half.rest * outputs, half.whole, half.splits, outputs, half.blocks, heads, L};
}

template <typename T>
int backward(const ww_attention_t& p, const Plan& plan, cudaStream_t stream) noexcept
{
    constexpr bool bf = !std::is_same<T, __half>::value;
    const bool has_q = p.B > 0 && p.Lq > 0, has_k = p.B > 0 && p.Lk > 0;
    uint8_t* ws = static_cast<uint8_t*>(p.workspace);
    BwdParams f;
    const int cols = p.D <= 32 ? 32 : 64;
    const int nq[3] = {p.B, p.Lq, p.Hq}, nk[3] = {p.B, p.Lk, p.Hk};
    if (has_q && (!encode_vectors_map(&f.q, bf, p.q, p.D, nq, p.q_strides, cols, kCols) ||
                  !encode_vectors_map(&f.dout, bf, p.dout, p.D, nq, p.dout_strides, cols, kCols)))
        return WW_ERR_UNSUPPORTED;
    if (has_k && (!encode_vectors_map(&f.k, bf, p.k, p.D, nk, p.k_strides, cols, kCols) ||
                  !encode_vectors_map(&f.v, bf, p.v, p.D, nk, p.v_strides, cols, kCols)))
        return WW_ERR_UNSUPPORTED;
    f.k_lens = p.k_lens;
    f.key_mask = p.key_mask;
    f.table = p.bias_table;
    f.tops = reinterpret_cast<uint32_t*>(ws);
    f.norm2 = reinterpret_cast<float*>(ws + plan.norm2);
    f.seen = has_q && has_k ? reinterpret_cast<uint32_t*>(ws + plan.seen) : nullptr;
    f.nlse2 = reinterpret_cast<float*>(ws + plan.nlse2);
    f.ndelta = reinterpret_cast<float*>(ws + plan.ndelta);
    f.table_part = reinterpret_cast<float*>(ws + plan.table);
    if (p.bias_table != nullptr)
        make_buckets(p.num_buckets, p.max_distance, p.bidirectional, p.q_offset, &f.rel);
    f.B = p.B;
    f.Lq = p.Lq;
    f.Lk = p.Lk;
    f.Hq = p.Hq;
    f.Hk = p.Hk;
    f.D = p.D;
    f.Lq_pad = plan.Lq_pad;
    f.q_tiles = plan.Lq_pad / kCols;
    f.q_b = p.q_strides[0] != 0;
    f.q_h = p.q_strides[2] != 0;
    f.k_b = p.k_strides[0] != 0;
    f.k_h = p.k_strides[2] != 0;
    f.v_b = p.v_strides[0] != 0;
    f.v_h = p.v_strides[2] != 0;
    f.g_b = p.dout_strides[0] != 0;
    f.g_h = p.dout_strides[2] != 0;
    f.scale = p.scale;
    f.scale2 = p.scale * kLog2eF;
    f.err = device_error_slot();
    if (f.err == nullptr) return WW_ERR_DEVICE;

    int st = WW_SUCCESS;
    if (has_q) {
        if (!bf && cudaMemsetAsync(ws, 0, static_cast<size_t>(p.B) * 8, stream) != cudaSuccess)
            return launch_status("cross_attention_backward");
        const int per = p.D <= 32 ? 64 : p.D <= 64 ? 32 : 16;  // rows of a block
        const int64_t of_q = (i64(plan.Lq_pad) * p.Hq + per - 1) / per, of_v = bf ? 0 : (i64(p.Lk) * p.Hk + 2 * per - 1) / (2 * per);
        if ((of_q + of_v) * p.B > 0x7fffffff) return WW_ERR_UNSUPPORTED;
        const DeltaParams delta = {const_cast<float*>(f.nlse2), const_cast<float*>(f.ndelta), const_cast<float*>(f.norm2),
                                   reinterpret_cast<uint32_t*>(ws), reinterpret_cast<uint32_t*>(ws + plan.seen),
                                   plan.Lq_pad, static_cast<int>(of_q * p.B),
                                   make_divisor(static_cast<int>(of_q)), make_divisor(of_v > 0 ? static_cast<int>(of_v) : 1),
                                   make_divisor(p.Hq), make_divisor(p.Hk)};
        const auto kernel = per == 64 ? attention_delta_kernel<T, 4> : per == 32 ? attention_delta_kernel<T, 8>
                                                                                 : attention_delta_kernel<T, 16>;
        kernel<<<static_cast<unsigned>((of_q + of_v) * p.B), 256, 0, stream>>>(p, delta);
        st = launch_status("cross_attention_backward");
    }
    const int far = rel_positions(p.max_distance);
    if (st == WW_SUCCESS && has_k) {
        f.part = reinterpret_cast<float*>(ws + plan.k_part);
        f.d1 = p.dk;
        f.d2 = p.dv;
        f.r1 = p.k;
        f.r2 = p.v;
        std::copy(p.k_strides, p.k_strides + 3, f.r1_strides);
        std::copy(p.v_strides, p.v_strides + 3, f.r2_strides);
        f.max_entries = std::min(far, plan.Lq_pad + kRows);
        st = run_half<T, true>(f, plan.k, has_q, stream);
    }
    if (st == WW_SUCCESS && has_q) {
        f.part = reinterpret_cast<float*>(ws + plan.q_part);
        f.d1 = p.dq;
        f.d2 = nullptr;
        f.r1 = p.q;
        f.r2 = p.dout;
        std::copy(p.q_strides, p.q_strides + 3, f.r1_strides);
        std::copy(p.dout_strides, p.dout_strides + 3, f.r2_strides);
        f.max_entries = std::min(far, (p.Lk + kCols - 1) / kCols * kCols + kRows);
        st = run_half<T, false>(f, plan.q, has_k, stream);
    }
    const SumParams keys = sum_params(plan.k, true, reinterpret_cast<const float*>(ws + plan.k_part), p.dk, p.dv, p.Hk, p.Lk);
    const SumParams queries = sum_params(plan.q, false, reinterpret_cast<const float*>(ws + plan.q_part), p.dq, nullptr, p.Hq, p.Lq);
    if (st == WW_SUCCESS && keys.count + queries.count > 0) {
        launch_behind(attention_sum_kernel<T>, dim3(keys.count + queries.count, kRows / kSumRows), dim3(256), 0, stream, keys,
                      queries, p.D);
        st = launch_status("cross_attention_backward");
    }
    if (st == WW_SUCCESS && p.bias_table != nullptr) {
        launch_behind(attention_table_kernel<T>, dim3(p.Hq * kTableCtas, (p.num_buckets + 31) / 32), dim3(1024), 0, stream,
                      f.table_part, static_cast<T*>(p.dbias_table), has_q ? p.B : 0, p.Hq, plan.q.blocks, plan.q.whole,
                      plan.q.splits, p.num_buckets);
        st = launch_status("cross_attention_backward");
    }
    return st;
}

int sm_count() noexcept
{
    DeviceInfo d;
    return current_device_info(&d) == WW_SUCCESS ? d.sm_count : 148;
}

}  // namespace
}  // namespace ww

extern "C" {

int64_t ww_cross_attention_backward_workspace(const ww_attention_t* p)
{
    ww::Plan plan;
    if (p == nullptr || ww::check_attention(*p) != WW_SUCCESS || !ww::make_plan(*p, ww::sm_count(), &plan)) return 0;
    return plan.bytes;
}

int ww_cross_attention_backward(const ww_attention_t* p, void* stream)
{
    if (p == nullptr) return WW_ERR_NULL_POINTER;
    ww::Plan plan;
    int st = ww::check_attention(*p);
    if (st == WW_SUCCESS && !ww::make_plan(*p, ww::sm_count(), &plan)) st = WW_ERR_UNSUPPORTED;
    if (st == WW_SUCCESS) st = ww::check_attention_backward(*p, plan.bytes);
    if (st != WW_SUCCESS) return st;
    ww::DeviceInfo d;
    if ((st = ww::current_device_info(&d)) != WW_SUCCESS) return st;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return p->dtype == WW_DTYPE_HALF ? ww::backward<__half>(*p, plan, s) : ww::backward<__nv_bfloat16>(*p, plan, s);
}

}  // extern "C"
