// attention_forward.cu -- ww_cross_attention: softmax(scale Q K^T + bias) V on
// the 5th-generation tensor cores, one pass over the keys.
//
// For a tile of 128 query rows and KT keys at a time, with x = scale log2(e) s
// + bias log2(e) the scores in log2 units:
//
//   S = Q K^T                       tcgen05.mma, operands staged by TMA, S in TMEM
//   m' = max(m, max_j x_j)          one thread per row: its KT scores from TMEM
//   P_j = 2^(x_j - m'), l = l 2^(m - m') + sum_j P_j
//   O = O 2^(m - m') + P V          P goes back to TMEM as the A operand
//   out = O / l, lse = ln 2 (m + log2 l)
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since the
// last time (P then stays below 2^8, exact in 16 bits' range): after the first
// tiles that hardly happens, and no tile needs the read-multiply-write of O.
//
// Roles: per query tile 4 warps that turn scores into P and one that issues its
// MMAs; one warp for every TMA load and the limits of masked keys.
//
// Bound: the exponential, 16 per clock and SM: 1024 clocks for 128 x 128
// scores, against 16 D clocks for their products (8192 fp16 FMA per clock):
// 512 at D = 32, equal at D = 64.  A round trip (scores, maximum, P, product) is
// a chain of latencies several times its exponentials, so what counts is how
// many tiles of an SM are under way: 64 keys at a time keep a tile's TMEM at
// 64 + D columns (P overwrites its scores, the next S is issued behind the
// product that reads them: MMAs of one thread run in issue order), and scores
// are read 32 columns at a time in a loop that fits 80 registers -- four tiles on
// an SM, 16 warps of elementwise work (two tiles at D = 128, where S, P and O of
// a tile take 192 columns).
//   NT = 1  four CTAs of one query tile: starts and ends overlap as well; of short
//           rows one CTA takes several query blocks of a head, of several batch items
//   NT = 2  two CTAs of two query tiles against the same keys: half the reads of
//           K and V from L2, for long rows (make_plan has both sides)
//
// Measured, fp16: 19200 queries to 19200 keys, 5 heads of 64: 665 us in long runs, where
// the power cap lowers the clock, 710 TFLOP/s, 2.8e12 exponentials a second (16 per
// clock: 4.5e12), 605 us in short ones; 8192 to 8192, 8 heads of 128: 320 us, 860
// TFLOP/s, 305 in short runs; 12032 heads of 32 in rows of 312, 5 % of the keys
// masked, with a bias: 753 us, a third of the exponentials' rate -- a tile's four
// warps take 1000 to 1500 clocks for each of the two passes over its scores, and
// five tiles to a row leave the start (tables, first loads) in sight.
//
// Masked keys: the load warp clears their rows of K and V before a tile is used
// (its products then see zeros, whatever the places held: 0 times a NaN would not
// be 0) and leaves limits, 0 or -inf, that join the scores; tiles without a masked
// key skip the limits, calls without one the clearing.
// The relative bias of a head depends on j - i alone: a CTA puts its values by
// position into shared memory once, a row reads a tile's at fixed offsets from
// its own start (neighbouring rows one apart: no bank conflicts); tiles beyond
// max_distance add a constant.
//
// Few rows against many keys: the keys are split over CTAs, each writes its
// normalised fp32 rows and log sums, a second kernel joins them in order.
#include "attention.cuh"
#include "attention_token.cuh"
#include "tensor_map.cuh"
#include "umma.cuh"

#include <algorithm>
#include <type_traits>

namespace ww {
namespace {

constexpr int kTile = 128;       // query rows of a tile
constexpr int kBox = 64;         // tokens of a TMA box
constexpr int kPolyOf = 4;       // one pair of exponentials in so many on the FMA pipe
constexpr float kRescale = 8.0f; // log2 growth of the maximum that is left in P

struct FwdParams {
    CUtensorMap q, k, v;
    void* out;
    float* lse;
    const int32_t* k_lens;
    const uint8_t* key_mask;
    const void* table;
    float* part_o;    // split items: [item][split][NT * 128][D], normalised
    float* part_lse;  // [item][split][NT * 128], log2
    RelBuckets rel;
    int32_t B, Lq, Lk, Hq, group, D;
    int32_t q_blocks, per_cta, groups;  // query blocks, those of one CTA, groups of them
    int32_t wide, row_blocks;           // groups run over all batch items of a head; the blocks they share out
    int32_t whole_items, splits;
    Divisor by_block, by_head, by_group, by_q;
    int32_t q_b, q_h, k_b, k_h, v_b, v_h;  // 0 where the tensor is broadcast
    int32_t max_entries;                   // relative positions a CTA keeps
    float scale2;                          // scale * log2(e)
    int* err;
    const float2* powers;                  // of keys and values, [batch item][key head]
    int32_t Hk;
};

template <int DP, int NT>
struct Layout {
    static constexpr int kKeys = 64;                       // keys of a tile
    static constexpr int kRow = DP == 32 ? 64 : 128;       // bytes of an operand row
    static constexpr int kCols = kRow / 2;                 // values in it
    static constexpr int kChunks = DP * 2 / kRow;          // rows of one token
    static constexpr int kQChunk = kTile * kRow;
    static constexpr int kQBytes = kTile * DP * 2;
    static constexpr int kChunk = kKeys * kRow;            // of a tile of K or V
    static constexpr int kBytes = kKeys * DP * 2;
    static constexpr int kStages = NT == 2 ? 3 : 2;
    static constexpr int kK = NT * kQBytes;
    static constexpr int kV = kK + kStages * kBytes;
    static constexpr int kLim = kV + kStages * kBytes;     // [stages][keys] limits, [stages] flags
    static constexpr int kBar = kLim + kStages * (kKeys + 4) * 4;
    static constexpr int kBias = kBar + 256;               // [entries] values
    static constexpr int kTotal = kBias + 1024;            // + alignment of the base, + the bias
    static constexpr int kNeed = NT * (kKeys + DP);
    static constexpr int kColumns = kNeed <= 128 ? 128 : kNeed <= 256 ? 256 : 512;
    static constexpr int kThreads = NT * 160 + 32;         // softmax warps, MMA warps, TMA warp
    static constexpr int kCtas = 512 / kColumns;
};

template <int DP, int NT>
struct Bars {
    static constexpr int kStages = Layout<DP, NT>::kStages;
    uint64_t q_full, q_empty, k_full[kStages], k_ready[kStages], k_empty[kStages], v_full[kStages], v_ready[kStages],
        v_empty[kStages], s_full[NT], p_ready[NT],
        o_full[NT], o_free[NT];
    uint32_t tmem;
};

// N scores in log2 units with bias and limits, and their maximum.
template <bool BIAS, bool LIMIT, int N>
__device__ __forceinline__ float score_pass(uint32_t (&x)[N], float scale2, float flat, const float* bias,
                                            const float* limit)
{
    float top[2] = {-INFINITY, -INFINITY};
    const Pair scale_2 = pair(scale2, scale2), flat_2 = pair(flat, flat);
#pragma unroll
    for (int j = 0; j < N; j += 4) {
        Pair y0 = fma2(pair(f32(x[j]), f32(x[j + 1])), scale_2, BIAS ? pair(bias[j], bias[j + 1]) : flat_2);
        Pair y1 = fma2(pair(f32(x[j + 2]), f32(x[j + 3])), scale_2, BIAS ? pair(bias[j + 2], bias[j + 3]) : flat_2);
        if (LIMIT) {
            const float4 lim = *reinterpret_cast<const float4*>(limit + j);
            y0 = add2(y0, pair(lim.x, lim.y));
            y1 = add2(y1, pair(lim.z, lim.w));
        }
        float y[4];
        unpair(y0, y[0], y[1]);
        unpair(y1, y[2], y[3]);
        top[0] = max3(top[0], y[0], y[1]);
        top[1] = max3(top[1], y[2], y[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[j + i] = __float_as_uint(y[i]);
    }
    return fmaxf(top[0], top[1]);
}

// P = 2^(mul x + add) of N columns: summed, rounded and put into N / 2 columns of
// TMEM.  POLY: one pair in kPolyOf on the FMA pipe (whole tiles without a bias
// of their own; a NaN or +inf among their scores has made `add` NaN, and -inf gives
// 2^-126 in place of 0).
template <typename T, bool POLY, int N>
__device__ __forceinline__ void exp_pass(const uint32_t (&x)[N], float mul, float add, Pair& sum, uint32_t to)
{
    uint32_t pk[N / 2];
    const Pair mul_2 = pair(mul, mul), add_2 = pair(add, add);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
        const Pair arg = fma2(pair(f32(x[2 * j]), f32(x[2 * j + 1])), mul_2, add_2);
        float a, b;
        if (POLY && j % kPolyOf == kPolyOf - 1) {
            unpair(exp2_poly<false>(arg), a, b);
        } else {
            unpair(arg, a, b);
            a = exp2_approx(a);
            b = exp2_approx(b);
        }
        sum = add2(sum, pair(a, b));
        pk[j] = pack2<T>(a, b);
    }
    if constexpr (N == 32) umma::tmem_st16(to, pk);
    else umma::tmem_st8(to, pk);
}

// POWERS: keys and values come divided by powers of two, which scores and results take back.
template <typename T, int DP, int NT, bool POWERS>
__global__ void __launch_bounds__(Layout<DP, NT>::kThreads, Layout<DP, NT>::kCtas)
    attention_forward_kernel(const __grid_constant__ FwdParams p)
{
    using L = Layout<DP, NT>;
    using Bar = Bars<DP, NT>;
    constexpr int S = L::kStages, KT = L::kKeys;
    extern __shared__ uint8_t raw[];
    uint8_t* base = raw + ((1024 - (umma::smem_addr(raw) & 1023)) & 1023);
    const uint32_t sm = umma::smem_addr(base);
    Bar* bar = reinterpret_cast<Bar*>(base + L::kBar);
    const auto at = [](const uint64_t& b) { return umma::smem_addr(&b); };

    // items (group of query blocks, head, batch item); the last ones are split over their keys
    const int blk = blockIdx.x;
    const bool in_parts = blk >= p.whole_items;
    const int split = in_parts ? (blk - p.whole_items) % p.splits : 0, splits = in_parts ? p.splits : 1;
    const int item = in_parts ? p.whole_items + (blk - p.whole_items) / p.splits : blk;
    // (wide: every batch item has the same number of key tiles, and one group may run over several)
    const bool wide = NT == 1 && p.wide != 0;
    const int outer = p.by_block.div(item), u0 = (item - outer * p.groups) * p.per_cta;
    const int b0 = wide ? 0 : p.by_head.div(outer), h = wide ? outer : outer - b0 * p.Hq, g = p.by_group.div(h);
    const int nq = min(p.per_cta, p.row_blocks - u0);  // query blocks of this CTA, one after the other
    const auto batch_of = [&](int qi) { return wide ? p.by_q.div(u0 + qi) : b0; };
    const auto q_of = [&](int qi) { return (u0 + qi - (wide ? batch_of(qi) * p.q_blocks : 0)) * (NT * kTile); };
    const auto tiles_of = [&](int qi) { return NT == 1 || q_of(qi) + kTile >= p.Lq ? 1 : 2; };  // query tiles with rows
    const int len = p.k_lens == nullptr ? p.Lk : min(max(__ldg(p.k_lens + b0), 0), p.Lk);
    const int n_all = (len + KT - 1) / KT;
    int first, n;
    part_of(n_all, split, splits, first, n);
    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;  // warp-uniform: roles branch as warps
    // keys of a tile
    const auto cols_of = [&](int kt) { return min(KT, len - (first + kt) * KT); };
    float* limits = reinterpret_cast<float*>(base + L::kLim);
    uint32_t* wholes = reinterpret_cast<uint32_t*>(limits + S * KT);  // tile without a masked key

    const bool masks = p.key_mask != nullptr || len % KT != 0;
    const auto k_bar = [&](int s) { return masks ? at(bar->k_ready[s]) : at(bar->k_full[s]); };
    const auto v_bar = [&](int s) { return masks ? at(bar->v_ready[s]) : at(bar->v_full[s]); };

    // tiles are numbered over all query blocks: number i is key tile i % n of block i / n
    const auto load_k = [&](int i, int kt, int b) {
        const int s = i % S;
        umma::mbar_arrive_expect_tx(at(bar->k_full[s]), L::kBytes);
        for (int c = 0; c < L::kChunks; ++c)
            for (int x = 0; x < KT; x += kBox)
                umma::tma_load_4d(sm + L::kK + s * L::kBytes + c * L::kChunk + x * L::kRow, &p.k, c * L::kCols, g * p.k_h,
                                  (first + kt) * KT + x, b * p.k_b, at(bar->k_full[s]));
    };
    const auto load_v = [&](int i, int kt, int b) {
        const int s = i % S;
        umma::mbar_arrive_expect_tx(at(bar->v_full[s]), L::kBytes);
        for (int c = 0; c < L::kChunks; ++c)
            for (int x = 0; x < KT; x += kBox)
                umma::tma_load_4d(sm + L::kV + s * L::kBytes + c * L::kChunk + x * L::kRow, &p.v, c * L::kCols, g * p.v_h,
                                  (first + kt) * KT + x, b * p.v_b, at(bar->v_full[s]));
    };
    const auto load_q = [&](int qi) {
        const int tiles = tiles_of(qi), b = batch_of(qi);
        umma::mbar_arrive_expect_tx(at(bar->q_full), tiles * L::kQBytes);
        for (int t = 0; t < tiles; ++t)
            for (int c = 0; c < L::kChunks; ++c)
                for (int x = 0; x < kTile; x += kBox)  // a box beyond the last row reads zeros
                    umma::tma_load_4d(sm + t * L::kQBytes + c * L::kQChunk + x * L::kRow, &p.q, c * L::kCols, h * p.q_h,
                                      min(q_of(qi) + t * kTile + x, p.Lq), b * p.q_b, at(bar->q_full));
    };
    if (warp == NT * 5 && lane == 0) {
        // this thread alone uses the barriers until the block's first barrier below
        umma::mbar_init(at(bar->q_full), 1);
        umma::mbar_init(at(bar->q_empty), NT);  // one MMA warp per tile
        for (int s = 0; s < S; ++s) {
            umma::mbar_init(at(bar->k_full[s]), 1);
            umma::mbar_init(at(bar->k_ready[s]), 1);
            umma::mbar_init(at(bar->v_ready[s]), 1);
            umma::mbar_init(at(bar->k_empty[s]), NT);
            umma::mbar_init(at(bar->v_full[s]), 1);
            umma::mbar_init(at(bar->v_empty[s]), NT);
        }
        for (int t = 0; t < NT; ++t) {
            umma::mbar_init(at(bar->s_full[t]), 1);
            umma::mbar_init(at(bar->p_ready[t]), 4);  // one arrival per warp
            umma::mbar_init(at(bar->o_full[t]), 1);
            umma::mbar_init(at(bar->o_free[t]), 4);
        }
        umma::mbar_fence_init();
        umma::fence_proxy_async_smem();
        if (n > 0) {
            load_q(0);
            load_k(0, 0, batch_of(0));
            load_v(0, 0, batch_of(0));
        }
    }
    RelRange range;  // positions j - i - q_offset of the tiles, padded rows and columns included
    float* values = reinterpret_cast<float*>(base + L::kBias);
    if (p.rel.per_side != 0 && n > 0) {
        const int q_lo = wide ? 0 : q_of(0), q_end = wide ? p.q_blocks * kTile : q_of(nq);
        range = rel_range(p.rel, first * KT - (q_end - 1) - p.rel.q_offset, (first + n) * KT - 1 - q_lo - p.rel.q_offset);
        TableRow<T> table;
        table.load(p.rel, p.table, h, lane);
        for (int e0 = warp * 32; warp < NT * 4 && e0 < range.count(); e0 += NT * 128) {  // the other warps have their own starts
            const int e = min(e0 + lane, range.count() - 1), bu = rel_bucket(p.rel, range.lo + e);
            values[e] = table.get(p.rel, bu);
        }
    }
    if (warp == NT * 4) umma::tmem_alloc(umma::smem_addr(&bar->tmem), L::kColumns);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = bar->tmem;

    if (warp == NT * 5) {
        bool ok = true;
        int load_kt = 0, load_qi = 0;  // of the next tile to load
        const auto load = [&](int i) {  // lane 0; tile 0 is on its way already
            if (i > 0) {
                const int s = i % S;
                const uint32_t ph = (i / S + 1) & 1;
                if (load_kt == 0) {
                    ok = ok && umma::mbar_poll(at(bar->q_empty), (load_qi - 1) & 1);
                    if (ok) load_q(load_qi);
                }
                ok = ok && umma::mbar_poll(at(bar->k_empty[s]), ph);
                if (ok) load_k(i, load_kt, batch_of(load_qi));
                ok = ok && umma::mbar_poll(at(bar->v_empty[s]), ph);
                if (ok) load_v(i, load_kt, batch_of(load_qi));
            }
            if (++load_kt == n) {
                load_kt = 0;
                ++load_qi;
            }
        };
        const int total = nq * n;
        if (!masks) {
            if (lane == 0)
                for (int i = 0; i < total && ok; ++i) load(i);
        } else if (n > 0) {
            // Tile i - 1 + S is asked for when tile i has been cleared: it waits for the products
            // of tile i - 1, and, where a query block ends between (one tile of queries, S = 2),
            // for the scores of tile i.
            static_assert(NT == 2 || S == 2, "query blocks follow one another");
            if (lane == 0) load(0);
            if (lane == 0 && n > 1)
                for (int i = 1; i < S && i < n; ++i) load(i);
            int loaded = min(S, n), kt = 0, qi = 0;
            for (int i = 0; i < total; ++i) {
                const int s = i % S, k0 = (first + kt) * KT;
                const uint8_t* mask = p.key_mask + static_cast<int64_t>(batch_of(qi)) * p.Lk;
                uint32_t in_mask = 0;
#pragma unroll
                for (int c = 0; c < KT; c += 32) {
                    const int key = k0 + c + lane;
                    if (key < len && (p.key_mask == nullptr || __ldg(mask + key) != 0))
                        in_mask |= 1u << (c / 32);
                }
                ok = __shfl_sync(~0u, ok, 0);
                bool all = true;
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    ok = ok && umma::mbar_poll(kv == 0 ? at(bar->k_full[s]) : at(bar->v_full[s]), (i / S) & 1);
#pragma unroll
                    for (int c = 0; c < KT; c += 32) {
                        const bool in = (in_mask >> (c / 32)) & 1;
                        all = all && in;
                        if (kv == 0) limits[s * KT + c + lane] = in ? 0.0f : -INFINITY;
                        if (!in) {
                            const uint32_t to = sm + (kv == 0 ? L::kK : L::kV) + s * L::kBytes + (c + lane) * L::kRow;
                            for (int x = 0; x < L::kChunks; ++x)
#pragma unroll
                                for (int j = 0; j < L::kRow; j += 16) umma::st_shared_v4(to + x * L::kChunk + j, 0, 0, 0, 0);
                        }
                    }
                    if (kv == 0) {
                        all = __all_sync(~0u, all);
                        if (lane == 0) wholes[s] = all;
                    }
                    umma::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) umma::mbar_arrive(kv == 0 ? at(bar->k_ready[s]) : at(bar->v_ready[s]));
                }
                // tiles of the next block follow their block's last one (S = 2: tile i + 1)
                while (loaded < total && loaded <= max(i - 1 + S, i + 1)) {
                    if (lane == 0) load(loaded);
                    ++loaded;
                }
                __syncwarp();
                if (++kt == n) {
                    kt = 0;
                    ++qi;
                }
            }
        }
        if (lane == 0 && !ok) record_device_error(p.err, kErrMbarTimeout | 0x20);
    } else if (warp >= NT * 4) {
        const int t = warp - NT * 4;
        if (n > 0) {
            // The warp runs the loop as a whole, one elected lane issues; descriptors are
            // formed once and advanced by constants and loops are unrolled, so that all a
            // product needs is in uniform registers (formed per product in one thread
            // they took 100 clocks each, more than the products).
            constexpr bool bf = !std::is_same<T, __half>::value;
            // all columns of a tile: those beyond its keys are products with zeros, not what TMEM held
            constexpr uint32_t id_s = umma::idesc_16bit(bf, kTile, KT, false), id_o = umma::idesc_16bit(bf, kTile, DP, true);
            const uint32_t s_col = __reduce_or_sync(~0u, tmem) + t * KT, o_col = s_col + (NT - t) * KT + t * DP;
            const uint64_t q_desc = umma::smem_desc_swizzled<L::kRow>(sm + t * L::kQBytes, 16);
            const uint64_t k_desc = umma::smem_desc_swizzled<L::kRow>(sm + L::kK, 16);
            const uint64_t v_desc = umma::smem_desc_swizzled<L::kRow>(sm + L::kV, L::kChunk);
            const auto qk = [&](int i, int kt) {
                const int s = i % S;
                const uint64_t kd = umma::desc_advance(k_desc, s * L::kBytes);
                if (umma::elect_one()) {
#pragma unroll
                    for (int j = 0; j < DP / 16; ++j)
                        umma::mma_f16_ss(s_col, umma::desc_advance(q_desc, j * 16 / L::kCols * L::kQChunk + j * 16 % L::kCols * 2),
                                         umma::desc_advance(kd, j * 16 / L::kCols * L::kChunk + j * 16 % L::kCols * 2), id_s, j > 0);
                    umma::mma_commit(at(bar->s_full[t]));
                    umma::mma_commit(at(bar->k_empty[s]));
                    if (kt == n - 1) umma::mma_commit(at(bar->q_empty));
                }
                __syncwarp();
            };
            bool ok = true;
            int i = 0;
            for (int qi = 0; qi < nq && ok; ++qi) {
                ok = umma::mbar_poll(at(bar->q_full), qi & 1);
                if (t >= tiles_of(qi)) {
                    // a tile without rows: its share of the places is given back as they are filled
                    if (ok && lane == 0) umma::mbar_arrive(at(bar->q_empty));
                    for (int kt = 0; kt < n && ok; ++kt, ++i) {
                        const int s = i % S;
                        ok = umma::mbar_poll(k_bar(s), (i / S) & 1);
                        if (ok && lane == 0) umma::mbar_arrive(at(bar->k_empty[s]));
                        ok = ok && umma::mbar_poll(v_bar(s), (i / S) & 1);
                        if (ok && lane == 0) umma::mbar_arrive(at(bar->v_empty[s]));
                    }
                    continue;
                }
                ok = ok && umma::mbar_poll(k_bar(i % S), (i / S) & 1);
                if (ok) qk(i, 0);
                for (int kt = 0; kt < n && ok; ++kt, ++i) {
                    const int s = i % S, cols = cols_of(kt);
                    ok = umma::mbar_poll(v_bar(s), (i / S) & 1) && umma::mbar_poll(at(bar->p_ready[t]), i & 1);
                    // the O before has been read
                    if (kt == 0 && qi > 0) ok = ok && umma::mbar_poll(at(bar->o_free[t]), (qi - 1) & 1);
                    if (!ok) break;
                    umma::fence_after_sync();
                    const uint64_t vd = umma::desc_advance(v_desc, s * L::kBytes);
                    if (umma::elect_one()) {
#pragma unroll
                        for (int j = 0; j < KT / 16; ++j)
                            if (j * 16 < cols)
                                umma::mma_f16_ts(o_col, s_col + j * 8, umma::desc_advance(vd, j * 16 * L::kRow), id_o, kt > 0 || j > 0);
                        umma::mma_commit(at(bar->v_empty[s]));
                        if (kt == n - 1) umma::mma_commit(at(bar->o_full[t]));
                    }
                    __syncwarp();
                    if (kt + 1 < n) {
                        ok = umma::mbar_poll(k_bar((i + 1) % S), ((i + 1) / S) & 1);
                        if (ok) qk(i + 1, kt + 1);
                    }
                }
            }
            if (!ok && lane == 0) record_device_error(p.err, kErrMbarTimeout | 0x21);
        }
    } else {
        const int t = warp / 4, r = threadIdx.x % 128;
        const uint32_t lanes = static_cast<uint32_t>(warp % 4) << 21;  // TMEM lane of this warp's first row
        const uint32_t s_col = tmem + lanes + t * KT, o_col = tmem + lanes + NT * KT + t * DP;
        constexpr bool kAhead = NT == 2 || DP == 128;
        bool ok = true;  // once a wait has run out: no more waits, everything else goes on
        int number = 0;
        for (int qi = 0; qi < nq && t < tiles_of(qi); ++qi) {
            const int q0 = q_of(qi), i = q0 + t * kTile + r;
            const auto power = [&] { return p.powers + static_cast<int64_t>(batch_of(qi)) * p.Hk + p.by_group.div(h); };
            const float scale2 = POWERS ? p.scale2 * __ldg(&power()->x) : p.scale2;
            float m = -INFINITY;
            Pair l2 = pair(0.0f, 0.0f);  // sums of the even and of the odd columns
            const bool any_row = q0 + t * kTile + warp % 4 * 32 < p.Lq;  // else this warp keeps the barriers only
            for (int kt = 0; kt < n; ++kt, ++number) {
                const int s = number % S, k0 = (first + kt) * KT, cols = cols_of(kt);
                // the bias: one value for the tile, or by j - i from this row's start
                float flat = 0.0f;
                const float* mine = nullptr;
                if (p.rel.per_side != 0) {
                    const int lo = k0 - (q0 + t * kTile + kTile - 1) - p.rel.q_offset, hi = lo + kTile + KT - 2;
                    if (hi <= -p.rel.max_distance || lo >= p.rel.max_distance || (!p.rel.bidirectional && lo >= 0))
                        flat = values[min(max(lo, range.lo), range.hi) - range.lo];
                    else
                        mine = values + k0 - i - p.rel.q_offset - range.lo;
                }
                if (masks) ok = ok && umma::mbar_poll(at(bar->k_ready[s]), (number / S) & 1);  // its limits
                const bool whole = !masks || wholes[s] != 0;
                ok = ok && umma::mbar_poll(at(bar->s_full[t]), number & 1);
                umma::fence_after_sync();
                const int chunks = any_row ? (cols + 31) / 32 : 0;
                // raw scores: scale and constant join the exponential's argument
                const bool plain = whole && mine == nullptr && scale2 >= 0.0f && flat > -INFINITY;
                float top = -INFINITY, add;
                const float* lim = limits + s * KT;
                const auto largest = [&](auto raw_scores, int c, auto& x) {  // of the N columns from c on
                    constexpr int N = sizeof(x) / 4;
                    if (raw_scores) {
                        float top1 = -INFINITY;
#pragma unroll
                        for (int j = 0; j < N; j += 4) {
                            top = max3_nan(top, f32(x[j]), f32(x[j + 1]));
                            top1 = max3_nan(top1, f32(x[j + 2]), f32(x[j + 3]));
                        }
                        top = max_nan(top, top1);
                    } else {
                        float tc;
                        if (mine == nullptr)
                            tc = whole ? score_pass<false, false>(x, scale2, flat, nullptr, nullptr)
                                       : score_pass<false, true>(x, scale2, flat, nullptr, lim + c);
                        else
                            tc = whole ? score_pass<true, false>(x, scale2, 0.0f, mine + c, nullptr)
                                       : score_pass<true, true>(x, scale2, 0.0f, mine + c, lim + c);
                        top = fmaxf(top, tc);
                        if constexpr (N == 32) umma::tmem_st32(s_col + c, x);
                        else umma::tmem_st16(s_col + c, x);
                    }
                };
                const auto exps = [&](auto raw_scores, int c, const auto& x) {  // P of N columns, over scores that have been read
                    if (raw_scores) exp_pass<T, true>(x, scale2, add, l2, s_col + c / 2);
                    else exp_pass<T, false>(x, 1.0f, add, l2, s_col + c / 2);
                };
                const auto columns = [&](const auto& use, auto raw_scores) {
                    // Raw scores, with no other work to hide behind, where registers allow (long
                    // queries, wide heads): 16 at a time, the next ones on their way meanwhile.
                    // 19200 to 19200, 5 heads of 64: 638 -> 600 us; 8192, 8 of 128: 334 -> 297.
                    // Elsewhere it spills (rows of 160: 35 us, so 39).
                    if constexpr (kAhead && std::is_same<decltype(raw_scores), std::true_type>::value) {
                        if (!any_row) return;
                        uint32_t x[2][16];
                        umma::tmem_ld16(s_col, x[0]);
#pragma unroll
                        for (int c = 0; c < KT; c += 16) {
                            umma::tmem_wait_ld16(x[c / 16 & 1]);
                            if (c + 16 < KT) umma::tmem_ld16(s_col + c + 16, x[c / 16 + 1 & 1]);
                            use(raw_scores, c, x[c / 16 & 1]);
                        }
                    } else {
#pragma unroll 1
                        for (int c = 0; c < chunks; ++c) {
                            uint32_t x[32];
                            umma::tmem_ld32(s_col + c * 32, x);
                            umma::tmem_wait_ld32(x);
                            use(raw_scores, c * 32, x);
                        }
                    }
                };
                const auto pass = [&](const auto& use) {
                    if constexpr (kAhead) {  // the choice outside the loop, which is unrolled
                        if (plain) columns(use, std::true_type{});
                        else columns(use, std::false_type{});
                    } else {
                        columns(use, plain);
                    }
                };
                pass(largest);
                if (!plain) umma::tmem_wait_st();
                if (plain) top = fmaf(top, scale2, flat);
                // grow the maximum: always on the first tile, then only past kRescale.  A NaN score (of
                // raw ones; others keep it to the sum) or one of +inf makes it NaN, and with it the row.
                if (__any_sync(~0u, kt == 0 || !(top <= m + kRescale))) {
                    float mn = max_nan(m, top);
                    if (mn == INFINITY) mn = NAN;
                    if (kt > 0) {  // the product before is done: its commit came before that of these scores
                        const float f = exp2_approx(m == -INFINITY ? -INFINITY : m - mn);
                        l2 = mul2(l2, pair(f, f));
#pragma unroll 1
                        for (int c = 0; c < DP; c += 16) {
                            uint32_t o[16];
                            umma::tmem_ld16(o_col + c, o);
                            umma::tmem_wait_ld16(o);
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(f32(o[j]) * f);
                            umma::tmem_st16(o_col + c, o);
                        }
                    }
                    m = mn;
                }
                add = (plain ? flat : 0.0f) - (m == -INFINITY ? 0.0f : m);
                pass(exps);
                umma::tmem_wait_st();
                umma::fence_before_sync();
                __syncwarp();
                if (lane == 0) umma::mbar_arrive(at(bar->p_ready[t]));
            }
            if (n > 0) ok = ok && umma::mbar_poll(at(bar->o_full[t]), qi & 1);
            umma::fence_after_sync();
            float l_even, l_odd;
            unpair(l2, l_even, l_odd);
            float sum = l_even + l_odd;
            if (m == -INFINITY && sum < 1.0f) sum = 0.0f;  // scores of -inf alone: an empty row
            const float inv = (sum == 0.0f ? 0.0f : 1.0f / sum) * (POWERS ? __ldg(&power()->y) : 1.0f);
            const int64_t b = batch_of(qi), row = (b * p.Lq + i) * p.Hq + h;
            const int64_t part = (static_cast<int64_t>(item - p.whole_items) * p.splits + split) * (NT * kTile) + t * kTile + r;
#pragma unroll
            for (int c = 0; c < DP; c += 32) {
                uint32_t o[32];
                if (n > 0) {
                    umma::tmem_ld32(o_col + c, o);
                    umma::tmem_wait_ld32(o);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = 0;
                }
                if (i >= p.Lq) continue;
                if (in_parts) {
                    float* to = p.part_o + part * p.D + c;
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        if (c + j < p.D)
                            *reinterpret_cast<float4*>(to + j) =
                                make_float4(f32(o[j]) * inv, f32(o[j + 1]) * inv, f32(o[j + 2]) * inv, f32(o[j + 3]) * inv);
                } else {
                    T* to = static_cast<T*>(p.out) + row * p.D + c;
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
                        if (c + j < p.D)
                            *reinterpret_cast<uint4*>(to + j) = make_uint4(
                                pack2<T>(f32(o[j]) * inv, f32(o[j + 1]) * inv), pack2<T>(f32(o[j + 2]) * inv, f32(o[j + 3]) * inv),
                                pack2<T>(f32(o[j + 4]) * inv, f32(o[j + 5]) * inv),
                                pack2<T>(f32(o[j + 6]) * inv, f32(o[j + 7]) * inv));
                }
            }
            if (i < p.Lq) {
                const float lse2 = sum == 0.0f ? -INFINITY : m + log2f(sum);
                if (in_parts) p.part_lse[part] = lse2;
                else if (p.lse != nullptr) p.lse[(b * p.Hq + h) * p.Lq + i] = lse2 * kLn2F;
            }
            umma::fence_before_sync();
            __syncwarp();
            if (lane == 0) umma::mbar_arrive(at(bar->o_free[t]));
        }
        if (!ok) record_device_error(p.err, kErrMbarTimeout | 0x22);
    }
    __syncthreads();
    if (warp == NT * 4) {
        umma::fence_after_sync();
        umma::tmem_dealloc(tmem, L::kColumns);
    }
}

// Joins the parts of a row: out = sum_s 2^(lse_s - top) out_s / sum_s 2^(lse_s - top),
// in order.  One warp per row, 4 values per lane; items as numbered by the kernel
// that wrote the parts: (query block, head, batch item) with `rows` query rows, or
// for the token form (key head, batch item) with rows (shared head, token).
template <typename T>
__global__ void __launch_bounds__(128) attention_join_kernel(const float* part_o, const float* part_lse, void* out,
                                                             float* lse, int whole_items, int splits, int rows, int q_blocks,
                                                             int Lq, int Hq, int Hk, int D)
{
    const int k = blockIdx.x, r = blockIdx.y * 4 + threadIdx.x / 32, lane = threadIdx.x % 32;
    const int item = whole_items + k;
    int64_t b;
    int h, i;
    if (q_blocks == 0) {
        b = item / Hk;
        h = item % Hk * (Hq / Hk) + r / Lq;
        i = r % Lq;
    } else {
        b = item / q_blocks / Hq;
        h = item / q_blocks % Hq;
        i = item % q_blocks * rows + r;
    }
    if (r >= rows || i >= Lq) return;
    wait_for_launches_before();
    const int64_t first = static_cast<int64_t>(k) * splits * rows + r;  // + s * rows
    float top = -INFINITY;
    for (int s = lane; s < splits; s += 32) top = fmaxf(top, part_lse[first + static_cast<int64_t>(s) * rows]);
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
        const int64_t at = first + static_cast<int64_t>(s) * rows;
        const float w = exp2_approx(part_lse[at] - base);
        sum += w;
        if (lane * 4 < D) {  // a part without keys is written as zeros
            const float4 v = *reinterpret_cast<const float4*>(part_o + at * D + lane * 4);
            acc.x += w * v.x;
            acc.y += w * v.y;
            acc.z += w * v.z;
            acc.w += w * v.w;
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (lane * 4 < D)
        *reinterpret_cast<uint2*>(static_cast<T*>(out) + ((b * Lq + i) * Hq + h) * D + lane * 4) =
            make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
    if (lse != nullptr && lane == 0) lse[(b * Hq + h) * Lq + i] = sum == 0.0f ? -INFINITY : (base + log2f(sum)) * kLn2F;
}

// How a call runs: few rows per key (attention_token.cu) or tiles of query rows,
// and which items are split over their keys: those that do not fill a round of
// the GPU's CTAs (all of them, where there are few).
struct Plan {
    bool token;
    bool wide;
    int nt, q_blocks, per_cta, row_blocks, outer, groups, whole, rest, splits, rows;
    int64_t part_rows() const { return i64(rest) * splits * rows; }
    int64_t part_bytes(int D) const { return part_rows() * (D + 1) * 4; }
    void without_parts()
    {
        splits = 1;
        rest = 0;
        whole = groups * outer;
    }
};

// Tiles one after the other in `items` CTAs of `tiles` each and a start that costs
// as much as `start` tiles, the last round split where that is sooner (tail_splits).
double tail_time(int64_t items, int slots, int64_t tiles, double start) noexcept
{
    const int rest = static_cast<int>(items % slots), splits = tail_splits(rest, slots, tiles);
    const double one = tiles + start, last = splits == 1 ? one : static_cast<double>(tiles) * rest / slots + 14.0;
    return static_cast<double>(items / slots) * one + (rest == 0 ? 0.0 : last);
}

bool make_plan(const ww_attention_t& p, int sms, Plan* plan) noexcept
{
    Plan& r = *plan;
    r.token = token_form(p, sms);
    if (r.token) {
        r.wide = false;
        r.q_blocks = r.groups = r.per_cta = r.row_blocks = r.outer = 0;
        r.nt = 0;
        r.rows = p.Hq / p.Hk * p.Lq;
        r.splits = token_splits(p, sms);
        if (i64(p.B) * p.Hk * r.splits > (1 << 30)) return false;
        r.whole = 0;
        r.rest = r.splits > 1 ? p.B * p.Hk : 0;
        return true;
    }
    // Two query tiles per CTA for long queries.  fp16, two tiles and one: 8192 to 8192, 8 heads
    // of 64 209 us and 223, 4096, 16 of 32 108 and 112; 2048, 40 of 64 76 and 75; 4 x 1200 to
    // 1777 57 and 53; rows of 312 with a bias 1144 and 797; 8192, 8 heads of 128, where both
    // take all of TMEM, 375 and 334.
    r.nt = p.Lq > 2048 && p.D <= 64 ? 2 : 1;
    r.rows = r.nt * kTile;
    r.q_blocks = (p.Lq + r.rows - 1) / r.rows;
    const int64_t heads = i64(p.B) * p.Hq, tiles = (p.Lk + 63) / 64;
    if (heads * r.q_blocks > (1 << 30)) return false;
    const int slots = sms * (p.D > 64 ? 2 : 4) / r.nt;
    // Query blocks of one CTA, of one (batch item, head) or, where all items have the same
    // length, of a head over several items: the count whose rounds end soonest, several
    // items only where that is clearly sooner (they share no keys).  fp16, one block per
    // CTA or those of one item, and several items:
    //   4908 x 6 heads of 80, 51 to 43 tokens, with a bias: 558 us and 364
    //   2000 x 4 heads of 32, 60 to 60: 68 and 43; 1504 x 8 of 32, 312 to 312: 574 and
    //   590, masked and with a bias 796 and 753; 360 x 3 of 32, 320 to 320: 83 and 86
    constexpr double kClearly = 1.15;
    const double start = p.bias_table != nullptr ? 2.5 : 1.25;
    r.per_cta = 1;
    r.wide = false;
    double least = tail_time(heads * r.q_blocks, slots, tiles, start);
    for (int wide = 0; wide < 2; ++wide) {
        if (r.nt == 2 || heads == 0 || (wide && p.k_lens != nullptr)) break;
        const int64_t outer = wide ? p.Hq : heads, blocks = wide ? i64(p.B) * r.q_blocks : r.q_blocks;
        const int64_t rounds = (outer + slots - 1) / slots;
        for (int64_t k = rounds; k < rounds + 4; ++k) {  // CTAs for k rounds
            const int64_t per_outer = k * slots / outer, n = (blocks + per_outer - 1) / per_outer;
            const double time = static_cast<double>(k) * (static_cast<double>(n) * tiles + start) * (wide ? kClearly : 1.0);
            if (n > 1 && time < least) {
                least = time;
                r.per_cta = static_cast<int>(n);
                r.wide = wide != 0;
            }
        }
    }
    r.outer = static_cast<int>(r.wide ? p.Hq : heads);
    r.row_blocks = r.wide ? p.B * r.q_blocks : r.q_blocks;
    r.groups = (r.row_blocks + r.per_cta - 1) / r.per_cta;
    const int64_t items = i64(r.outer) * r.groups;
    r.rest = static_cast<int>(items % slots);
    r.splits = r.per_cta == 1 ? tail_splits(r.rest, slots, tiles) : 1;  // the join counts blocks
    if (r.splits == 1) r.rest = 0;
    r.whole = static_cast<int>(items - r.rest);
    return true;
}

template <typename T, int DP, int NT>
int launch(const FwdParams& f, int64_t ctas, cudaStream_t stream) noexcept
{
    using L = Layout<DP, NT>;
    // only fp16's range is too narrow for some keys and values
    auto kernel = attention_forward_kernel<T, DP, NT, false>;
    if constexpr (std::is_same<T, __half>::value)
        if (f.powers != nullptr) kernel = attention_forward_kernel<T, DP, NT, true>;
    static_assert(L::kTotal + 4 * ((kMaxPositions + 15) / 16 * 16) <= kMaxShared, "shared memory");
    const int bytes = L::kTotal + 4 * f.max_entries;
    static std::atomic<uint64_t> raised[2];
    if (!allow_shared_memory(reinterpret_cast<const void*>(kernel), raised[f.powers != nullptr])) return launch_status("cross_attention");
    kernel<<<static_cast<unsigned>(ctas), L::kThreads, bytes, stream>>>(f);
    return launch_status("cross_attention");
}

template <typename T>
int tiles(const ww_attention_t& p, const Plan& plan, float* part_o, float* part_lse, const float2* powers, cudaStream_t stream) noexcept
{
    FwdParams f;
    f.powers = powers;
    const int dp = p.D <= 32 ? 32 : p.D <= 64 ? 64 : 128;
    constexpr bool bf = !std::is_same<T, __half>::value;
    const int nq[3] = {p.B, p.Lq, p.Hq}, nk[3] = {p.B, p.Lk, p.Hk};
    const int cols = dp == 32 ? 32 : 64;
    if (!encode_vectors_map(&f.q, bf, p.q, p.D, nq, p.q_strides, cols, kBox)) return WW_ERR_UNSUPPORTED;
    if (p.Lk > 0) {
        if (!encode_vectors_map(&f.k, bf, p.k, p.D, nk, p.k_strides, cols, kBox) ||
            !encode_vectors_map(&f.v, bf, p.v, p.D, nk, p.v_strides, cols, kBox))
            return WW_ERR_UNSUPPORTED;
    }
    f.out = p.out;
    f.lse = p.lse;
    f.k_lens = p.k_lens;
    f.key_mask = p.key_mask;
    f.table = p.bias_table;
    f.max_entries = 0;
    if (p.bias_table != nullptr) {
        make_buckets(p.num_buckets, p.max_distance, p.bidirectional, p.q_offset, &f.rel);
        const int all = (p.Lk + 127) / 128 * 128 + (plan.wide ? plan.q_blocks : plan.per_cta) * plan.nt * kTile;
        f.max_entries = (std::min(rel_positions(p.max_distance), all) + 15) / 16 * 16;
    }
    f.part_o = part_o;
    f.part_lse = part_lse;
    f.B = p.B;
    f.Lq = p.Lq;
    f.Lk = p.Lk;
    f.Hq = p.Hq;
    f.Hk = p.Hk;
    f.group = p.Hq / p.Hk;
    f.D = p.D;
    f.q_blocks = plan.q_blocks;
    f.per_cta = plan.per_cta;
    f.groups = plan.groups;
    f.wide = plan.wide;
    f.row_blocks = plan.row_blocks;
    f.by_block = make_divisor(plan.groups);
    f.by_head = make_divisor(p.Hq);
    f.by_q = make_divisor(plan.q_blocks);
    f.by_group = make_divisor(p.Hq / p.Hk);
    f.whole_items = plan.whole;
    f.splits = plan.splits;
    f.q_b = p.q_strides[0] != 0;
    f.q_h = p.q_strides[2] != 0;
    f.k_b = p.k_strides[0] != 0;
    f.k_h = p.k_strides[2] != 0;
    f.v_b = p.v_strides[0] != 0;
    f.v_h = p.v_strides[2] != 0;
    f.scale2 = p.scale * kLog2eF;
    f.err = device_error_slot();
    const int64_t ctas = plan.whole + i64(plan.rest) * plan.splits;
    if (f.err == nullptr) return WW_ERR_DEVICE;
    if (plan.nt == 1)
        return dp == 32 ? launch<T, 32, 1>(f, ctas, stream)
             : dp == 64 ? launch<T, 64, 1>(f, ctas, stream) : launch<T, 128, 1>(f, ctas, stream);
    return dp == 32 ? launch<T, 32, 2>(f, ctas, stream) : launch<T, 64, 2>(f, ctas, stream);
}

template <typename T>
int forward(const ww_attention_t& p, const Plan& plan, const float2* powers, cudaStream_t stream) noexcept
{
    float* part_o = static_cast<float*>(p.workspace);
    float* part_lse = part_o + plan.part_rows() * p.D;
    const int st = plan.token ? attention_token_launch(p, plan.splits, part_o, part_lse, stream)
                              : tiles<T>(p, plan, part_o, part_lse, powers, stream);
    if (st != WW_SUCCESS || plan.rest == 0) return st;
    launch_behind(attention_join_kernel<T>, dim3(plan.rest, (plan.rows + 3) / 4), dim3(128), 0, stream, part_o, part_lse, p.out,
                  p.lse, plan.whole, plan.splits, plan.rows, plan.q_blocks, p.Lq, p.Hq, p.Hk, p.D);
    return launch_status("cross_attention");
}

int sm_count() noexcept
{
    DeviceInfo d;
    return current_device_info(&d) == WW_SUCCESS ? d.sm_count : 148;
}

}  // namespace

int attention_join_launch(const ww_attention_t& p, int items, int splits, int rows, const float* part_o, const float* part_lse,
                          const char* name, cudaStream_t stream) noexcept
{
    const auto go = [&](auto kernel) {
        launch_behind(kernel, dim3(items, (rows + 3) / 4), dim3(128), 0, stream, part_o, part_lse, p.out, p.lse, 0, splits, rows, 0,
                      p.Lq, p.Hq, p.Hk, p.D);
    };
    if (p.dtype == WW_DTYPE_HALF) go(attention_join_kernel<__half>);
    else go(attention_join_kernel<__nv_bfloat16>);
    return launch_status(name);
}

int cross_attention(const ww_attention_t& p, const float2* powers, void* stream) noexcept
{
    int st = check_attention(p);
    if (st != WW_SUCCESS || p.B == 0 || p.Lq == 0) return st;
    DeviceInfo d;
    if ((st = current_device_info(&d)) != WW_SUCCESS) return st;
    Plan plan;
    if (!make_plan(p, d.sm_count, &plan)) return WW_ERR_UNSUPPORTED;
    if (p.workspace == nullptr) plan.without_parts();
    else if (plan.part_bytes(p.D) > p.workspace_bytes) return WW_ERR_UNSUPPORTED;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return p.dtype == WW_DTYPE_HALF ? forward<__half>(p, plan, powers, s) : forward<__nv_bfloat16>(p, plan, nullptr, s);
}

}  // namespace ww

extern "C" {

int64_t ww_cross_attention_workspace(const ww_attention_t* p)
{
    ww::Plan plan;
    if (p == nullptr || ww::check_attention(*p) != WW_SUCCESS || !ww::make_plan(*p, ww::sm_count(), &plan)) return 0;
    return plan.part_bytes(p->D);
}

int ww_cross_attention(const ww_attention_t* p, void* stream)
{
    return p == nullptr ? WW_ERR_NULL_POINTER : ww::cross_attention(*p, nullptr, stream);
}

}  // extern "C"
