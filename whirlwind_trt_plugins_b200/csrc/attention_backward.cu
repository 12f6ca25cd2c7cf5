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
// The row operands stay in shared memory; each streamed tile is the K-major B
// operand of the two score products and, unchanged, the MN-major B operand of
// the accumulating ones; P and dS return to TMEM as their A operands.  Two
// tiles are in flight (S and dP of 64 columns each: 256 of 512 columns), one
// per warpgroup, so that products and elementwise work overlap.
//
// 16-bit ranges: P is kept as 2^6 P, and in fp16 dS is formed from dO 2^e with
// 2^e max|dO| in [1, 2): gradients as small as a mean over a batch leaves
// them stay in fp16's normal range.  Powers of two, taken out again at the end.
//
// Bound: per 128 x 64 tile 512 clocks of exponentials (16 per clock and SM) in
// each kernel against 8 D (dK, dV) and 6 D (dQ) clocks of products.
//
// dtable: a tile whose positions all lie in one bucket adds its plain sum.
// Otherwise dS goes through shared memory 32 columns at a time; a thread sums
// one diagonal j - i (one read and one add per value, no conflicts), diagonals
// are collected per CTA and joined to buckets, CTAs and warpgroups in order.
#include "attention.cuh"
#include "tensor_map.cuh"
#include "umma.cuh"

#include <algorithm>

namespace ww {
namespace {

constexpr int kRows = 128;
constexpr int kCols = 64;
constexpr int kShift = 6;         // P is kept times 2^kShift
constexpr int kPitch = 33;        // floats of a dS row in shared memory
constexpr int kThreads = 2 * 128 + 64;

struct BwdParams {
    CUtensorMap q, k, v, dout;  // boxes of 64 tokens
    const int32_t* k_lens;
    const uint8_t* key_mask;
    const void* table;
    const float* lse2;    // [B * Hq][Lq_pad] log2 units minus kShift; +inf: no gradient
    const float* delta;   // [B * Hq][Lq_pad]
    const uint32_t* top;  // bits of max |dO| (fp16)
    void* d1;             // keys: dk; queries: dq
    void* d2;             // keys: dv
    float* part;          // splits > 1: [splits][values of d1, then of d2] fp32
    float* table_part;    // queries: [B * Hq * blocks * splits][buckets]
    RelBuckets rel;
    int32_t B, Lq, Lk, Hq, Hk, D, Lq_pad;
    int32_t blocks, splits, q_tiles;
    int32_t q_b, q_h, k_b, k_h, v_b, v_h, g_b, g_h;
    int32_t max_entries;  // relative positions a CTA keeps
    float scale, scale2;
    int* err;
};

template <int DP, bool KEYS>
struct Layout {
    static constexpr int kRow = DP == 32 ? 64 : 128;   // bytes of an operand row
    static constexpr int kVals = kRow / 2;
    static constexpr int kChunks = DP * 2 / kRow;
    static constexpr int kRowChunk = kRows * kRow;     // row operand
    static constexpr int kRowBytes = kRows * DP * 2;
    static constexpr int kColChunk = kCols * kRow;     // streamed operand
    static constexpr int kColBytes = kCols * DP * 2;
    static constexpr int kStages = DP == 128 ? 2 : 4;
    static constexpr int kR1 = 0;
    static constexpr int kR2 = kRowBytes;
    static constexpr int kC = 2 * kRowBytes;                       // stages of C1, C2
    static constexpr int kVec = kC + kStages * 2 * kColBytes;      // KEYS: lse2, delta of 64 queries per stage
    static constexpr int kBar = kVec + (KEYS ? kStages * 2 * kCols * 4 : 0);
    static constexpr int kBias = kBar + 256;                       // bias tables, see below
};

template <int DP, bool KEYS>
struct Bars {
    static constexpr int kStages = Layout<DP, KEYS>::kStages;
    uint64_t r_full, c_full[kStages], c_empty[kStages], s_full[2], p_ready[2], done;
    uint32_t tmem;
};

// Shared memory after the barriers, with a bias:
//   buckets  [entries] bytes
//   KEYS:    values [2 warpgroups][entries] floats, rebuilt when the head changes
//   queries: values [entries], with a gradient also the diagonals
//            [2][entries], plain sums [8 warps][kMaxBuckets] and dS [2][128][33]
__host__ __device__ inline int bias_bytes(bool keys, int entries)
{
    const int e = (entries + 15) / 16 * 16;
    return keys ? e + 2 * e * 4 : e + 3 * e * 4 + 8 * kMaxBuckets * 4 + 2 * kRows * kPitch * 4;
}

template <typename T, int DP, bool KEYS, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1) attention_backward_kernel(const __grid_constant__ BwdParams p)
{
    using L = Layout<DP, KEYS>;
    using Bar = Bars<DP, KEYS>;
    constexpr int S = L::kStages;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    extern __shared__ uint8_t raw[];
    uint8_t* base = raw + ((1024 - (umma::smem_addr(raw) & 1023)) & 1023);
    const uint32_t sm = umma::smem_addr(base);
    Bar* bar = reinterpret_cast<Bar*>(base + L::kBar);
    const auto at = [](const uint64_t& b) { return umma::smem_addr(&b); };

    const int split = blockIdx.x % p.splits;
    int rest = blockIdx.x / p.splits;
    const int block = rest % p.blocks;
    rest /= p.blocks;
    const int heads = KEYS ? p.Hk : p.Hq, group = p.Hq / p.Hk;
    const int h = rest % heads, b = rest / heads;
    const int row0 = block * kRows;
    const int len = p.k_lens == nullptr ? p.Lk : min(max(__ldg(p.k_lens + b), 0), p.Lk);
    // streamed tiles of this CTA
    const int n_all = KEYS ? (row0 < len ? group * p.q_tiles : 0) : (len + kCols - 1) / kCols;
    const int first = static_cast<int>(static_cast<int64_t>(n_all) * split / p.splits);
    const int n = static_cast<int>(static_cast<int64_t>(n_all) * (split + 1) / p.splits) - first;

    const int warp = __shfl_sync(~0u, threadIdx.x / 32, 0), lane = threadIdx.x % 32;  // warp-uniform: roles branch as warps
    RelRange range;
    uint8_t* buckets = base + L::kBias;
    float* values = nullptr;  // bias of [range]: KEYS: of this warpgroup's current head
    const int entries = (p.max_entries + 15) / 16 * 16;
    if (BIAS) {
        // positions j - i - offset of the CTA's tiles, padded rows and columns included
        range = KEYS ? rel_range(p.rel, row0 - (p.q_tiles * kCols - 1) - p.rel.q_offset, row0 + kRows - 1 - p.rel.q_offset)
                     : rel_range(p.rel, first * kCols - (row0 + kRows - 1) - p.rel.q_offset,
                                 (first + n) * kCols - 1 - row0 - p.rel.q_offset);
        if (n > 0) build_buckets(p.rel, range, buckets, threadIdx.x, kThreads);
        values = reinterpret_cast<float*>(base + L::kBias + entries) + (KEYS && warp >= 4 ? entries : 0);
        if (!KEYS) {
            const T* table = static_cast<const T*>(p.table) + static_cast<int64_t>(h) * p.rel.total;
            if (n > 0)
                for (int e = threadIdx.x; e < range.count(); e += kThreads)
                    values[e] = bias_value<T>(table[rel_bucket(p.rel, range.lo + e)]) * kLog2eF;
            float* diag = values + entries;  // diagonals, then plain sums
            for (int e = threadIdx.x; e < 2 * entries + 8 * kMaxBuckets; e += kThreads) diag[e] = 0.0f;
        }
    }
    if (threadIdx.x == 0) {
        umma::mbar_init(at(bar->r_full), 1);
        for (int s = 0; s < S; ++s) {
            umma::mbar_init(at(bar->c_full[s]), 1);
            umma::mbar_init(at(bar->c_empty[s]), 1);
        }
        for (int s = 0; s < 2; ++s) {
            umma::mbar_init(at(bar->s_full[s]), 1);
            umma::mbar_init(at(bar->p_ready[s]), 4);  // one arrival per warp
        }
        umma::mbar_init(at(bar->done), 1);
        umma::mbar_fence_init();
    }
    if (warp == 8) umma::tmem_alloc(umma::smem_addr(&bar->tmem), 512);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    const uint32_t tmem = bar->tmem;
    // columns: S of both stages, dP of both stages, then the accumulators
    const auto s_col = [&](int st) { return tmem + st * kCols; };
    const auto dp_col = [&](int st) { return tmem + 2 * kCols + st * kCols; };
    const uint32_t acc1 = tmem + 4 * kCols, acc2 = acc1 + DP;

    if (warp == 9) {
        if (lane == 0 && n > 0) {
            const CUtensorMap* r1 = KEYS ? &p.k : &p.q;
            const CUtensorMap* r2 = KEYS ? &p.v : &p.dout;
            const CUtensorMap* c1 = KEYS ? &p.q : &p.k;
            const CUtensorMap* c2 = KEYS ? &p.dout : &p.v;
            const int r1b = KEYS ? p.k_b : p.q_b, r1h = KEYS ? p.k_h : p.q_h, r2b = KEYS ? p.v_b : p.g_b,
                      r2h = KEYS ? p.v_h : p.g_h;
            const int c1b = KEYS ? p.q_b : p.k_b, c1h = KEYS ? p.q_h : p.k_h, c2b = KEYS ? p.g_b : p.v_b,
                      c2h = KEYS ? p.g_h : p.v_h;
            const int rows_end = KEYS ? p.Lk : p.Lq;
            // a half of the row tile that lies beyond the tensor reads as zeros like any other place outside
            umma::mbar_arrive_expect_tx(at(bar->r_full), 2 * L::kRowBytes);
            for (int half = 0; half < 2; ++half)
                for (int c = 0; c < L::kChunks; ++c) {
                    const uint32_t off = c * L::kRowChunk + half * L::kColChunk;
                    const int l = min(row0 + half * kCols, rows_end);
                    umma::tma_load_4d(sm + L::kR1 + off, r1, c * L::kVals, h * r1h, l, b * r1b, at(bar->r_full));
                    umma::tma_load_4d(sm + L::kR2 + off, r2, c * L::kVals, h * r2h, l, b * r2b, at(bar->r_full));
                }
            bool ok = true;
            for (int i = 0; i < n && ok; ++i) {
                const int s = i % S;
                ok = umma::mbar_poll(at(bar->c_empty[s]), (i / S + 1) & 1);
                if (!ok) break;
                int ch = h / group, l = (first + i) * kCols;
                if (KEYS) {
                    ch = h * group + (first + i) / p.q_tiles;
                    l = (first + i) % p.q_tiles * kCols;
                }
                umma::mbar_arrive_expect_tx(at(bar->c_full[s]), 2 * L::kColBytes + (KEYS ? 2 * kCols * 4 : 0));
                const uint32_t to = sm + L::kC + s * 2 * L::kColBytes;
                for (int c = 0; c < L::kChunks; ++c) {
                    umma::tma_load_4d(to + c * L::kColChunk, c1, c * L::kVals, ch * c1h, l, b * c1b, at(bar->c_full[s]));
                    umma::tma_load_4d(to + L::kColBytes + c * L::kColChunk, c2, c * L::kVals, ch * c2h, l, b * c2b,
                                      at(bar->c_full[s]));
                }
                if (KEYS) {
                    const int64_t row = (static_cast<int64_t>(b) * p.Hq + ch) * p.Lq_pad + l;
                    const uint32_t vec = sm + L::kVec + s * 2 * kCols * 4;
                    umma::bulk_g2s(vec, p.lse2 + row, kCols * 4, at(bar->c_full[s]));
                    umma::bulk_g2s(vec + kCols * 4, p.delta + row, kCols * 4, at(bar->c_full[s]));
                }
            }
            if (!ok) record_device_error(p.err, kErrMbarTimeout | 0x30);
        }
    } else if (warp == 8) {
        if (n > 0) {
            // one lane issues, the warp runs as a whole with everything in uniform registers
            // (see attention_forward.cu)
            const uint32_t tm = __reduce_or_sync(~0u, tmem);
            const auto s_col = [&](int st) { return tm + st * kCols; };
            const auto dp_col = [&](int st) { return tm + 2 * kCols + st * kCols; };
            const uint32_t acc1 = tm + 4 * kCols, acc2 = acc1 + DP;
            constexpr bool bf = !kHalf;
            constexpr uint32_t id_s = umma::idesc_16bit(bf, kRows, kCols, false), id_a = umma::idesc_16bit(bf, kRows, DP, true);
            const uint64_t r_desc = umma::smem_desc_swizzled<L::kRow>(sm + L::kR1, 16);
            const uint64_t c_desc = umma::smem_desc_swizzled<L::kRow>(sm + L::kC, 16);
            const uint64_t a_desc = umma::smem_desc_swizzled<L::kRow>(sm + L::kC, L::kColChunk);
            const auto scores = [&](int i) {
                const uint64_t cd = umma::desc_advance(c_desc, i % S * 2 * L::kColBytes);
                const uint32_t to = s_col(i & 1), to2 = dp_col(i & 1);
                if (!umma::elect_one()) return;
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int j = 0; j < DP / 16; ++j)
                        umma::mma_f16_ss(x ? to2 : to,
                                         umma::desc_advance(r_desc, x * L::kRowBytes + j * 16 / L::kVals * L::kRowChunk +
                                                                        j * 16 % L::kVals * 2),
                                         umma::desc_advance(cd, x * L::kColBytes + j * 16 / L::kVals * L::kColChunk +
                                                                    j * 16 % L::kVals * 2),
                                         id_s, j > 0);
                umma::mma_commit(at(bar->s_full[i & 1]));
            };
            bool ok = umma::mbar_poll(at(bar->r_full), 0);
            for (int i = 0; i < 2 && i < n && ok; ++i) {
                ok = umma::mbar_poll(at(bar->c_full[i]), 0);
                if (ok) scores(i);
            }
            for (int i = 0; i < n && ok; ++i) {
                ok = umma::mbar_poll(at(bar->p_ready[i & 1]), (i >> 1) & 1);
                if (!ok) break;
                umma::fence_after_sync();
                const uint64_t ad = umma::desc_advance(a_desc, i % S * 2 * L::kColBytes);
                const uint32_t from = s_col(i & 1), from2 = dp_col(i & 1);
                if (umma::elect_one()) {
#pragma unroll
                for (int j = 0; j < kCols / 16; ++j) {
                    umma::mma_f16_ts(acc1, from2 + j * 8, umma::desc_advance(ad, j * 16 * L::kRow), id_a, i > 0 || j > 0);
                    if (KEYS)
                        umma::mma_f16_ts(acc2, from + j * 8, umma::desc_advance(ad, L::kColBytes + j * 16 * L::kRow), id_a,
                                         i > 0 || j > 0);
                }
                umma::mma_commit(at(bar->c_empty[i % S]));
                }
                __syncwarp();
                if (i + 2 < n) {
                    ok = umma::mbar_poll(at(bar->c_full[(i + 2) % S]), ((i + 2) / S) & 1);
                    if (ok) scores(i + 2);
                }
            }
            if (ok && umma::elect_one()) umma::mma_commit(at(bar->done));
            if (!ok && lane == 0) record_device_error(p.err, kErrMbarTimeout | 0x31);
        }
    } else {
        const int wg = warp / 4, r = threadIdx.x % 128;
        const uint32_t lanes = static_cast<uint32_t>(warp % 4) << 21;
        const int row = row0 + r;
        bool ok = true;  // once a wait has run out: no more waits, but every barrier is kept
        // fp16: f = 2^e, e = 127 - the biased exponent of max |dO|
        float f = 1.0f;
        if (kHalf) {
            const int top = static_cast<int>(__ldg(p.top) >> 23);  // biased exponent
            if (top > 0 && top < 255) f = __int_as_float((254 - top) << 23);
        }
        bool row_ok = row < (KEYS ? len : p.Lq);
        float my_lse = INFINITY, my_delta = 0.0f;
        if (KEYS) {
            if (row_ok && p.key_mask != nullptr) row_ok = __ldg(p.key_mask + static_cast<int64_t>(b) * p.Lk + row) != 0;
        } else if (row_ok) {
            const int64_t i = (static_cast<int64_t>(b) * p.Hq + h) * p.Lq_pad + row;
            my_lse = __ldg(p.lse2 + i);
            my_delta = __ldg(p.delta + i) * f;
        }
        const bool rows_ok = __all_sync(~0u, row_ok);
        const bool any_row = row0 + warp % 4 * 32 < (KEYS ? len : p.Lq);  // else this warp keeps the barriers only
        int built = -1;  // KEYS: head of `values`
        float* diag = values + entries + wg * entries;
        float* plain = values + 3 * entries + warp * kMaxBuckets;
        float* tile = values + 3 * entries + 8 * kMaxBuckets + wg * kRows * kPitch;
        if (BIAS && !KEYS && !any_row)
            for (int j = 0; j < 32; ++j) tile[r * kPitch + j] = 0.0f;
        for (int i = wg; i < n; i += 2) {
            const int col0 = KEYS ? (first + i) % p.q_tiles * kCols : (first + i) * kCols;
            uint32_t keep[2] = {~0u, ~0u};
            if (!KEYS) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int left = len - col0 - 32 * c;
                    keep[c] = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
                    if (p.key_mask != nullptr)
                        keep[c] &= __ballot_sync(~0u, lane < left && __ldg(p.key_mask + static_cast<int64_t>(b) * p.Lk +
                                                                          col0 + 32 * c + lane) != 0);
                }
            }
            const bool whole = (keep[0] & keep[1]) == ~0u;
            float flat = 0.0f;
            const float* mine = nullptr;  // bias of column 0 of this row
            int flat_bucket = 0;
            if (BIAS) {
                const int ch = KEYS ? h * group + (first + i) / p.q_tiles : h;
                const T* table = static_cast<const T*>(p.table) + static_cast<int64_t>(ch) * p.rel.total;
                if (KEYS && built != ch) {
                    warpgroup_sync(wg);
                    for (int e = r; e < range.count(); e += 128) values[e] = bias_value<T>(table[buckets[e]]) * kLog2eF;
                    warpgroup_sync(wg);
                    built = ch;
                }
                // j - i - offset over the tile
                const int lo = KEYS ? row0 - (col0 + kCols - 1) - p.rel.q_offset : col0 - (row0 + kRows - 1) - p.rel.q_offset;
                const int hi = lo + kRows + kCols - 2;
                flat_bucket = bucket_at(range, buckets, lo);
                if (flat_bucket == bucket_at(range, buckets, hi))
                    flat = bias_value<T>(table[flat_bucket]) * kLog2eF;
                else
                    mine = values + (KEYS ? row - col0 : col0 - row) - p.rel.q_offset - range.lo;
            }
            ok = ok && umma::mbar_poll(at(bar->s_full[wg]), (i >> 1) & 1);
            umma::fence_after_sync();
            const float* vec = reinterpret_cast<const float*>(base + L::kVec + (i % S) * 2 * kCols * 4);
            if (KEYS) ok = ok && umma::mbar_poll(at(bar->c_full[i % S]), (i / S) & 1);
            const float row_add = (BIAS ? flat : 0.0f) - (KEYS ? 0.0f : my_lse);
            float total = 0.0f;
            // sums of a half tile's dS along j - i: each thread a diagonal, column
            // j of row (j + 127 - r) mod 128: diagonal r - 127 until column r, r + 1
            // (r < 31) from there on
            const auto diagonals = [&](int c) {
                warpgroup_sync(wg);
                float run = 0.0f, left = 0.0f;
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    if (j == r + 1) {
                        left = run;
                        run = 0.0f;
                    }
                    run += tile[((j + 127 - r) & 127) * kPitch + j];
                }
                float* to = diag + col0 + 32 * c - row0 - p.rel.q_offset - range.lo;
                to[r - 127] += r < 31 ? left : run;
                if (r < 31) to[r + 1] += run;
            };
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t s[32], d[32];
                if (!any_row) {
                    if (!KEYS && BIAS) {
                        if (mine != nullptr) {
                            warpgroup_sync(wg);
                            diagonals(c);
                        }
                    }
                    continue;
                }
                umma::tmem_ld32(s_col(wg) + lanes + c * 32, s);
                umma::tmem_ld32(dp_col(wg) + lanes + c * 32, d);
                umma::tmem_wait_ld32(s);
                umma::tmem_wait_ld32(d);
                uint32_t pk[16], dk[16];
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    float add = row_add;
                    if (KEYS) add -= vec[32 * c + j];
                    if (BIAS) {
                        if (mine != nullptr) add += KEYS ? mine[-(32 * c + j)] : mine[32 * c + j];
                    }
                    float pr = exp2_approx(fmaf(f32(s[j]), p.scale2, add));
                    float ds;
                    if (KEYS) {
                        const float del = vec[kCols + 32 * c + j];
                        ds = kHalf ? pr * ((f32(d[j]) - del) * f) : pr * (f32(d[j]) - del);
                    } else {
                        ds = kHalf ? pr * fmaf(f32(d[j]), f, -my_delta) : pr * (f32(d[j]) - my_delta);
                    }
                    s[j] = __float_as_uint(pr);
                    d[j] = __float_as_uint(ds);
                }
                if (KEYS ? !rows_ok : !whole) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const bool in = KEYS ? row_ok : ((keep[c] >> j) & 1);
                        s[j] = in ? s[j] : 0u;
                        d[j] = in ? d[j] : 0u;
                    }
                }
                if (!KEYS && BIAS) {
                    if (mine == nullptr) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) total += f32(d[j]);
                    } else {
                        float* to = tile + r * kPitch;
                        warpgroup_sync(wg);
#pragma unroll
                        for (int j = 0; j < 32; ++j) to[j] = f32(d[j]);
                        diagonals(c);
                    }
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (KEYS) pk[j] = pack2<T>(f32(s[2 * j]), f32(s[2 * j + 1]));
                    dk[j] = pack2<T>(f32(d[2 * j]), f32(d[2 * j + 1]));
                }
                if (KEYS) umma::tmem_st16(s_col(wg) + lanes + c * 16, pk);
                umma::tmem_st16(dp_col(wg) + lanes + c * 16, dk);
            }
            if (!KEYS && BIAS && mine == nullptr) {
                for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
                if (lane == 0) plain[flat_bucket] += total;
            }
            if (!KEYS && !whole) {
                // rows of K behind masked keys: 0 in place of whatever they hold
                ok = ok && umma::mbar_poll(at(bar->c_full[i % S]), (i / S) & 1);
                if (r < kCols && !((keep[(r >> 5) & 1] >> lane) & 1)) {
                    const uint32_t to = sm + L::kC + (i % S) * 2 * L::kColBytes + r * L::kRow;
                    for (int c = 0; c < L::kChunks; ++c)
#pragma unroll
                        for (int j = 0; j < L::kRow; j += 16) umma::st_shared_v4(to + c * L::kColChunk + j, 0, 0, 0, 0);
                }
                umma::fence_proxy_async_smem();
            }
            umma::tmem_wait_st();
            umma::fence_before_sync();
            __syncwarp();
            if (lane == 0) umma::mbar_arrive(at(bar->p_ready[wg]));
        }
        if (n > 0) ok = ok && umma::mbar_poll(at(bar->done), 0);
        umma::fence_after_sync();
        if (!ok) record_device_error(p.err, kErrMbarTimeout | 0x32);
        // keys: warpgroup 0 writes dk, 1 dv; queries: each half of dq
        const int L_ = KEYS ? p.Lk : p.Lq;
        const int64_t at_row = ((static_cast<int64_t>(b) * L_ + row) * heads + h) * p.D;
        const int64_t size = static_cast<int64_t>(p.B) * L_ * heads * p.D;
        const bool second = KEYS && wg == 1;
        const float mul = second ? 1.0f / (1 << kShift) : p.scale / (1 << kShift) / f;
        const uint32_t acc = second ? acc2 : acc1;
        constexpr int kSpan = KEYS ? DP : DP / 2;
        const int begin = KEYS ? 0 : wg * kSpan;
#pragma unroll
        for (int c = 0; c < kSpan; c += 16) {
            uint32_t o[16];
            const int d0 = begin + c;
            if (n > 0) {
                umma::tmem_ld16(acc + lanes + d0, o);
                umma::tmem_wait_ld16(o);
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = 0;
            }
            if (row >= L_) continue;
            if (KEYS && !row_ok) {  // a masked key: 0, whatever a skipped warp left in its lanes
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = 0;
            }
            if (p.splits > 1) {
                float* to = p.part + (static_cast<int64_t>(split) * (KEYS ? 2 : 1) + second) * size + at_row + d0;
#pragma unroll
                for (int j = 0; j < 16; j += 4)
                    if (d0 + j < p.D)
                        *reinterpret_cast<float4*>(to + j) =
                            make_float4(f32(o[j]) * mul, f32(o[j + 1]) * mul, f32(o[j + 2]) * mul, f32(o[j + 3]) * mul);
            } else {
                T* to = static_cast<T*>(second ? p.d2 : p.d1) + at_row + d0;
#pragma unroll
                for (int j = 0; j < 16; j += 8)
                    if (d0 + j < p.D)
                        *reinterpret_cast<uint4*>(to + j) = make_uint4(
                            pack2<T>(f32(o[j]) * mul, f32(o[j + 1]) * mul), pack2<T>(f32(o[j + 2]) * mul, f32(o[j + 3]) * mul),
                            pack2<T>(f32(o[j + 4]) * mul, f32(o[j + 5]) * mul),
                            pack2<T>(f32(o[j + 6]) * mul, f32(o[j + 7]) * mul));
            }
        }
        umma::fence_before_sync();
    }
    __syncthreads();
    if (warp == 8) {
        umma::fence_after_sync();
        umma::tmem_dealloc(tmem, 512);
    }
    if (BIAS && !KEYS) {
        // buckets of this CTA: each warp every 8th bucket, its lanes over the entries
        const float* diag = values + entries;
        const float* plain = values + 3 * entries;
        float f = 1.0f;
        if (kHalf) {
            const int top = static_cast<int>(__ldg(p.top) >> 23);
            if (top > 0 && top < 255) f = __int_as_float((254 - top) << 23);
        }
        float* to = p.table_part + static_cast<int64_t>(blockIdx.x) * p.rel.total;
        for (int t = warp; t < p.rel.total; t += kThreads / 32) {
            float sum = 0.0f;
            if (n > 0)
                for (int e = lane; e < range.count(); e += 32)
                    if (buckets[e] == t) sum += diag[e] + diag[entries + e];
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            if (lane == 0) {
                for (int w = 0; w < 8; ++w) sum += plain[w * kMaxBuckets + t];
                to[t] = sum / (1 << kShift) / f;
            }
        }
    }
}

// delta = rowsum(dO * O) and lse in log2 units, both laid out [B * Hq][Lq_pad]
// with rows of no gradient (lse -inf, padding) at lse2 = +inf; for fp16 also
// max |dO| (an integer maximum of non-negative floats: no order).  kLanes >= D / 8
// lanes per row, 8 values each.
template <typename T, int kLanes>
__global__ void __launch_bounds__(256) attention_delta_kernel(const __grid_constant__ ww_attention_t a, float* lse2,
                                                              float* delta, uint32_t* top, int Lq_pad)
{
    const int64_t item = static_cast<int64_t>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
    const int lane = threadIdx.x % kLanes;
    const int64_t rows = static_cast<int64_t>(a.B) * Lq_pad * a.Hq;
    const int h = static_cast<int>(item % a.Hq);
    const int64_t bi = item / a.Hq;
    const int b = static_cast<int>(bi / Lq_pad), i = static_cast<int>(bi % Lq_pad);
    const bool live = item < rows && i < a.Lq;
    float sum = 0.0f, mx = 0.0f;
    if (live && lane * 8 < a.D) {
        const T* g = static_cast<const T*>(a.dout) + b * a.dout_strides[0] + i * a.dout_strides[1] + h * a.dout_strides[2];
        const T* o = static_cast<const T*>(a.out) + ((static_cast<int64_t>(b) * a.Lq + i) * a.Hq + h) * a.D;
        const uint4 gu = *reinterpret_cast<const uint4*>(g + lane * 8);
        const uint4 ou = *reinterpret_cast<const uint4*>(o + lane * 8);
        const T* ge = reinterpret_cast<const T*>(&gu);
        const T* oe = reinterpret_cast<const T*>(&ou);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sum = fmaf(to_float(ge[j]), to_float(oe[j]), sum);
            mx = fmaxf(mx, fabsf(to_float(ge[j])));
        }
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (item < rows && lane == 0) {
        const int64_t to = (static_cast<int64_t>(b) * a.Hq + h) * Lq_pad + i;
        const float l = live ? a.lse[(static_cast<int64_t>(b) * a.Hq + h) * a.Lq + i] : -INFINITY;
        lse2[to] = l == -INFINITY ? INFINITY : l * kLog2eF - kShift;
        delta[to] = sum;
    }
    if (std::is_same<T, __half>::value) {
        __shared__ uint32_t block_top;
        if (threadIdx.x == 0) block_top = 0;
        __syncthreads();
        const uint32_t m = __reduce_max_sync(~0u, __float_as_uint(mx));
        if (threadIdx.x % 32 == 0) atomicMax(&block_top, m);
        __syncthreads();
        if (threadIdx.x == 0 && block_top > 0) atomicMax(top, block_top);
    }
}

// Sums of the splits in order; 4 values per thread.
template <typename T>
__global__ void __launch_bounds__(256) attention_sum_kernel(const float* part, int splits, int64_t stride, T* out, int64_t n)
{
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    float4 s = make_float4(0, 0, 0, 0);
    for (int k = 0; k < splits; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(part + k * stride + i);
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
    }
    *reinterpret_cast<uint2*>(out + i) = make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
}

// Table gradient of one head: the CTAs' buckets in order.  Each of 32 warps takes
// every 32nd CTA (four loads in flight), 32 buckets at a time, then the warps'
// sums in order.
template <typename T>
__global__ void __launch_bounds__(1024) attention_table_kernel(const float* part, T* out, int B, int Hq, int per_head, int total)
{
    __shared__ float sums[32][33];
    const int h = blockIdx.x, t = blockIdx.y * 32 + threadIdx.x % 32, w = threadIdx.x / 32;
    float s = 0.0f;
    if (t < total) {
#pragma unroll 4
        for (int n = w; n < B * per_head; n += 32)
            s += part[((static_cast<int64_t>(n / per_head) * Hq + h) * per_head + n % per_head) * total + t];
    }
    sums[w][threadIdx.x % 32] = s;
    __syncthreads();
    if (w == 0 && t < total) {
        s = 0.0f;
        for (int n = 0; n < 32; ++n) s += sums[n][threadIdx.x];
        out[h * total + t] = from_float<T>(s);
    }
}

// How a call runs and where its workspace is.
struct Plan {
    int q_blocks, k_blocks, q_splits, k_splits, Lq_pad;
    int64_t lse2, delta, part, table, bytes;  // byte offsets; the maximum of |dO| stands first
};

int splits_for(int64_t ctas, int64_t tiles, int sms)
{
    if (ctas <= 0 || ctas >= sms || tiles < 8) return 1;
    return static_cast<int>(std::min<int64_t>({sms / ctas, tiles / 4, 64}));
}

Plan make_plan(const ww_attention_t& p, int sms) noexcept
{
    Plan r;
    r.q_blocks = (p.Lq + kRows - 1) / kRows;
    r.k_blocks = (p.Lk + kRows - 1) / kRows;
    r.Lq_pad = (p.Lq + kCols - 1) / kCols * kCols;
    const int64_t q_ctas = i64(r.q_blocks) * p.B * p.Hq, k_ctas = i64(r.k_blocks) * p.B * p.Hk;
    r.q_splits = splits_for(q_ctas, (p.Lk + kCols - 1) / kCols, sms);
    r.k_splits = splits_for(k_ctas, i64(r.Lq_pad / kCols) * (p.Hq / p.Hk), sms);
    const int64_t rows = i64(p.B) * p.Hq * r.Lq_pad;
    const int64_t q_part = r.q_splits > 1 ? r.q_splits * i64(p.B) * p.Lq * p.Hq * p.D * 4 : 0;
    const int64_t k_part = r.k_splits > 1 ? 2 * r.k_splits * i64(p.B) * p.Lk * p.Hk * p.D * 4 : 0;
    r.lse2 = 256;
    r.delta = r.lse2 + rows * 4;
    r.part = r.delta + rows * 4;  // one after the other: both kernels use the same place
    r.table = r.part + std::max(q_part, k_part);
    r.bytes = r.table + (p.bias_table != nullptr ? q_ctas * r.q_splits * p.num_buckets * 4 : 0);
    return r;
}

template <typename T, int DP, bool KEYS, bool BIAS>
int launch_one(const BwdParams& f, int64_t ctas, cudaStream_t stream) noexcept
{
    using L = Layout<DP, KEYS>;
    const auto kernel = attention_backward_kernel<T, DP, KEYS, BIAS>;
    const int bytes = 1024 + L::kBias + (BIAS ? bias_bytes(KEYS, f.max_entries) : 0);
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
        return launch_status("cross_attention_backward");
    kernel<<<static_cast<unsigned>(ctas), kThreads, bytes, stream>>>(f);
    return launch_status("cross_attention_backward");
}

template <typename T, bool KEYS>
int launch(const BwdParams& f, int64_t ctas, cudaStream_t stream) noexcept
{
    if (ctas == 0) return WW_SUCCESS;
    if (ctas > 0x7fffffff) return WW_ERR_UNSUPPORTED;
    const int dp = f.D <= 32 ? 32 : f.D <= 64 ? 64 : 128;
    if (f.table != nullptr)
        return dp == 32 ? launch_one<T, 32, KEYS, true>(f, ctas, stream)
             : dp == 64 ? launch_one<T, 64, KEYS, true>(f, ctas, stream) : launch_one<T, 128, KEYS, true>(f, ctas, stream);
    return dp == 32 ? launch_one<T, 32, KEYS, false>(f, ctas, stream)
         : dp == 64 ? launch_one<T, 64, KEYS, false>(f, ctas, stream) : launch_one<T, 128, KEYS, false>(f, ctas, stream);
}

template <typename T>
int sum_parts(const float* part, int splits, int64_t stride, void* out, int64_t n, cudaStream_t stream) noexcept
{
    attention_sum_kernel<T><<<static_cast<unsigned>((n / 4 + 255) / 256), 256, 0, stream>>>(part, splits, stride,
                                                                                           static_cast<T*>(out), n);
    return launch_status("cross_attention_backward");
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
    f.top = reinterpret_cast<uint32_t*>(ws);
    f.lse2 = reinterpret_cast<float*>(ws + plan.lse2);
    f.delta = reinterpret_cast<float*>(ws + plan.delta);
    f.part = reinterpret_cast<float*>(ws + plan.part);
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
        if (!bf && cudaMemsetAsync(ws, 0, 4, stream) != cudaSuccess) return launch_status("cross_attention_backward");
        const int64_t rows = i64(p.B) * plan.Lq_pad * p.Hq;
        const int per = p.D <= 32 ? 64 : p.D <= 64 ? 32 : 16;  // rows of a block
        const int64_t blocks = (rows + per - 1) / per;
        if (blocks > 0x7fffffff) return WW_ERR_UNSUPPORTED;
        const auto kernel = per == 64 ? attention_delta_kernel<T, 4> : per == 32 ? attention_delta_kernel<T, 8>
                                                                                 : attention_delta_kernel<T, 16>;
        kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(p, const_cast<float*>(f.lse2), const_cast<float*>(f.delta),
                                                                  reinterpret_cast<uint32_t*>(ws), plan.Lq_pad);
        st = launch_status("cross_attention_backward");
    }
    const int far = 2 * (p.max_distance + kRelMargin) + 1;
    if (st == WW_SUCCESS && has_k) {
        f.d1 = p.dk;
        f.d2 = p.dv;
        f.blocks = plan.k_blocks;
        f.splits = plan.k_splits;
        f.max_entries = std::min(far, plan.Lq_pad + kRows);
        st = launch<T, true>(f, i64(plan.k_blocks) * p.B * p.Hk * plan.k_splits, stream);
        const int64_t n = i64(p.B) * p.Lk * p.Hk * p.D;
        if (st == WW_SUCCESS && plan.k_splits > 1) st = sum_parts<T>(f.part, plan.k_splits, 2 * n, p.dk, n, stream);
        if (st == WW_SUCCESS && plan.k_splits > 1) st = sum_parts<T>(f.part + n, plan.k_splits, 2 * n, p.dv, n, stream);
    }
    if (st == WW_SUCCESS && has_q) {
        f.d1 = p.dq;
        f.blocks = plan.q_blocks;
        f.splits = plan.q_splits;
        f.max_entries = std::min(far, (p.Lk + kCols - 1) / kCols * kCols + kRows);
        st = launch<T, false>(f, i64(plan.q_blocks) * p.B * p.Hq * plan.q_splits, stream);
        const int64_t n = i64(p.B) * p.Lq * p.Hq * p.D;
        if (st == WW_SUCCESS && plan.q_splits > 1) st = sum_parts<T>(f.part, plan.q_splits, n, p.dq, n, stream);
    }
    if (st == WW_SUCCESS && p.bias_table != nullptr) {
        attention_table_kernel<T><<<dim3(p.Hq, (p.num_buckets + 31) / 32), 1024, 0, stream>>>(
            f.table_part, static_cast<T*>(p.dbias_table), has_q ? p.B : 0, p.Hq, plan.q_blocks * plan.q_splits, p.num_buckets);
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
    if (p == nullptr || ww::check_attention(*p) != WW_SUCCESS) return 0;
    return ww::make_plan(*p, ww::sm_count()).bytes;
}

int ww_cross_attention_backward(const ww_attention_t* p, void* stream)
{
    if (p == nullptr) return WW_ERR_NULL_POINTER;
    int st = ww::check_attention(*p);
    if (st == WW_SUCCESS) st = ww::check_attention_backward(*p, ww::make_plan(*p, ww::sm_count()).bytes);
    if (st != WW_SUCCESS) return st;
    ww::DeviceInfo d;
    if ((st = ww::current_device_info(&d)) != WW_SUCCESS) return st;
    const ww::Plan plan = ww::make_plan(*p, d.sm_count);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return p->dtype == WW_DTYPE_HALF ? ww::backward<__half>(*p, plan, s) : ww::backward<__nv_bfloat16>(*p, plan, s);
}

}  // extern "C"
