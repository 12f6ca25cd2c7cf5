// attention_int8.cu -- ww_cross_attention with keys and values in 8 bits, for few
// query rows per key head; more rows: keys and values brought to 16 bits first (by_copies).
//
//   s_ij = (q_i . kq_j) ks_j scale log2(e) + bias,   l_i = sum_j 2^(s_ij - m_i)
//   o_i = sum_j 2^(s_ij + log2(vs_j) - n_i) vq_j,    out_i = o_i 2^(n_i - m_i) / l_i
//
// A key's scale is a factor of its scores, a value's goes into the exponent of its
// weight: the weights have a running maximum n of their own, so that P in fp16 (times
// 2^6) keeps its precision whatever the values' scales are, and the sum is formed beside it.
// Bound: HBM -- every key and value is read once, as one byte.  The bytes are
// brought to fp16 in registers, exactly (1024 + byte by a permutation, less 1152),
// and go through mma.sync m16n8k16 with 16 keys, or 16 dims of the values, as its M
// side and 8 rows (query heads of the key head x tokens) as its N side: what lanes
// convert is used once for all rows.  Queries are scaled by a power of two to fp16's
// upper range, whatever their type.
// Two blocks of 6 warps (4 for more than 8 rows) per SM.  Each warp runs alone over every 6th tile
// of 32 keys of its block's share: one lane keeps a ring of TMA loads in flight (swizzled rows, read back by
// ldmatrix), and no barrier joins the warps before the end.  Sums of scores belong to a
// lane until then; O is rescaled only when n has grown by 2^8.  The keys are split over
// blocks until the GPU is full: up to 4 are a cluster that joins its parts through shared
// memory, more are joined by attention_join_kernel, in order either way.
//
// Measured, bf16: one token of 2 x 32 heads on 8 key heads of 128 against 40001 keys with a bias,
// 169 MB: 36 us and 3 to join, 4.6 TB/s (5.6 between its start and end); 64 x 8 key heads
// of 128, 1250 keys, 170 MB: 39 us.
#include "attention_token.cuh"
#include "rows.cuh"
#include "tensor_map.cuh"
#include "umma.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace ww {

int dequantise_valid(const ww_kv_cache_t& p, const uint8_t* mask, float2* powers, const char* name, void* stream) noexcept;  // kv_cache.cu

namespace {

constexpr int kKeys = 32;          // of a warp's tile
// Splits that are a cluster and join themselves.  8 items of 4 key heads of 64 against up to 1500
// keys: 8.5 us and 10.1 with a second launch, a call 14 us and 18.  Clusters of 8 blocks of an
// SM each do not all find room at once: 2 x 8 key heads of 128, 40001 keys, 60 us and 37.
constexpr int kCluster = 4;
constexpr int kShort = 32;          // tiles of a cluster's block up to which a call takes no more splits
constexpr int kMostRows = 128;     // of a key head, in blocks of up to 32, that run without copies
constexpr float kRescale = 8.0f;   // log2 growth of a maximum that is left in P
constexpr float kHead = 6.0f;      // P times 2^6

struct Int8Params {
    CUtensorMap k, v;
    const float *ks, *vs;
    const void* q;
    void* out;
    float* lse;
    const int32_t* k_lens;
    const uint8_t* key_mask;
    const void* table;
    float* part_o;
    float* part_lse;
    RelBuckets rel;
    int64_t q_strides[3], ks_strides[2], vs_strides[2];
    int32_t B, Lq, Lk, Hq, Hk, D, rows;
    int32_t splits;
    int32_t k_b, k_h, v_b, v_h;
    int32_t max_entries;
    int32_t joined;  // the splits are a cluster
    float scale2;
    int* err;
};

template <int DP, int NB>
struct Layout {
    static constexpr int kTile = kKeys * DP;
    static constexpr int kWarps = NB == 1 ? 6 : 4;  // as registers allow two blocks per SM
    static constexpr int kStages = DP == 128 ? (NB == 1 ? 2 : 3) : DP == 64 ? 4 : 6;
    static constexpr int kRows = NB * 8;
    static constexpr int kRing = (kStages * 2 * kTile > kRows * DP * 4 ? kStages * 2 * kTile : kRows * DP * 4);  // of a warp; its rows at the end
    static constexpr int kQPitch = DP * 2 + 16;  // bytes
    static constexpr int kQ = kWarps * kRing;
    static constexpr int kRowScale = kQ + kRows * kQPitch;
    static constexpr int kBar = kRowScale + kRows * 4;
    static constexpr int kMl = kBar + kWarps * kStages * 8;     // n, maximum and sum of [warp][row]
    static constexpr int kBias = kMl + kWarps * kRows * 12;     // [heads][buckets] values, [entries] buckets
    static constexpr int kBytes = kBias + 1024;
    static constexpr int kItems = (kRows * (DP / 8) + kWarps * 32 - 1) / (kWarps * 32);  // 8 values of a row, of a thread at the end
    static_assert(kRing % 1024 == 0, "swizzled tiles");
    static_assert(kRows * DP * 4 + kRows * 8 <= kWarps * kRing, "a block's rows for its cluster");
};

// 16-byte piece j of row r of a swizzled tile of rows of DP bytes.
template <int DP>
__device__ __forceinline__ uint32_t piece(uint32_t tile, int r, int j)
{
    const int turn = DP == 128 ? r & 7 : DP == 64 ? (r >> 1) & 3 : (r >> 2) & 1;
    return tile + r * DP + ((j ^ turn) << 4);
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t saddr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(saddr)
                 : "memory");
}

// 8x8 matrix of 16-bit values transposed over the warp.
__device__ __forceinline__ uint32_t transpose(uint32_t x)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

// Two signed bytes of w (with their sign bits turned) as fp16: 1024 + 128 + byte, less 1152.
template <int SELECT>
__device__ __forceinline__ uint32_t to_half2(uint32_t w)
{
    const uint32_t u = __byte_perm(w, 0x64646464u, SELECT);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}

template <typename T, int DP, int NB>
__global__ void __launch_bounds__(Layout<DP, NB>::kWarps * 32, 2) attention_int8_kernel(const __grid_constant__ Int8Params p)
{
    using L = Layout<DP, NB>;
    constexpr int S = L::kStages, kRows = L::kRows, kWarps = L::kWarps;
    extern __shared__ uint8_t raw[];
    uint8_t* base = raw + ((1024 - (umma::smem_addr(raw) & 1023)) & 1023);
    const uint32_t sm = umma::smem_addr(base);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g8 = lane / 4, t4 = lane % 4;
    const uint32_t ring = sm + warp * L::kRing, bars = sm + L::kBar + warp * S * 8;

    if (p.splits > 1 && !p.joined) start_launch_behind();  // the join, which waits for this grid's end
    const int split = blockIdx.x % p.splits;
    const int g = blockIdx.x / p.splits % p.Hk, b = blockIdx.x / p.splits / p.Hk;
    const int row0 = blockIdx.y * kRows, rows = min(kRows, p.rows - row0);
    const int len = p.k_lens == nullptr ? p.Lk : min(max(__ldg(p.k_lens + b), 0), p.Lk);
    const int all = (len + kKeys - 1) / kKeys;
    int first, count;
    part_of(all, split, p.splits, first, count);
    const int last = first + count;
    const int n = (last - first - warp + kWarps - 1) / kWarps;  // tiles of this warp: first + warp + kWarps i
    const int group = p.Hq / p.Hk;

    const auto load = [&](int i) {  // lane 0
        const int s = i % S, key = (first + warp + kWarps * i) * kKeys;
        umma::mbar_arrive_expect_tx(bars + s * 8, 2 * L::kTile);
        const uint32_t to = ring + s * 2 * L::kTile;
        umma::tma_load_4d(to, &p.k, 0, g * p.k_h, key, b * p.k_b, bars + s * 8);
        umma::tma_load_4d(to + L::kTile, &p.v, 0, g * p.v_h, key, b * p.v_b, bars + s * 8);
    };
    if (lane == 0) {
        for (int s = 0; s < S; ++s) umma::mbar_init(bars + s * 8, 1);
        umma::mbar_fence_init();
        umma::fence_proxy_async_smem();
        for (int i = 0; i < S && i < n; ++i) load(i);
    }
    // query rows, a warp a row: row r is head g * group + r / Lq, token r % Lq; the rest zeros.
    // A row is multiplied by a power of two that brings its largest value to [2^14, 2^15).
    float* row_scales = reinterpret_cast<float*>(base + L::kRowScale);
    constexpr int kQueries = (kRows + kWarps - 1) / kWarps;  // of a warp, their loads under way together
    uint2 raw_q[kQueries];
    const int d = lane * 4;
#pragma unroll
    for (int i = 0; i < kQueries; ++i) {
        const int r = warp + i * kWarps;
        raw_q[i] = make_uint2(0, 0);
        if (r < rows && d < p.D)
            raw_q[i] = __ldg(reinterpret_cast<const uint2*>(static_cast<const T*>(p.q) + b * p.q_strides[0] + ((row0 + r) % p.Lq) * p.q_strides[1] +
                                                            (g * group + (row0 + r) / p.Lq) * p.q_strides[2] + d));
    }
#pragma unroll
    for (int i = 0; i < kQueries; ++i) {
        const int r = warp + i * kWarps;
        if (r >= kRows) break;
        const T* t = reinterpret_cast<const T*>(&raw_q[i]);
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = to_float(t[j]);
        const float top = row_max<32>(max_nan(max_nan(fabsf(x[0]), fabsf(x[1])), max_nan(fabsf(x[2]), fabsf(x[3]))), nullptr);
        int e = 0;  // 0 for rows that hold NaN, infinities or nothing
        if (top > 0.0f && top < INFINITY) e = 14 - max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100);
        const float f = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
        if (d < DP)
            *reinterpret_cast<uint2*>(base + L::kQ + r * L::kQPitch + d * 2) =
                make_uint2(pack2<__half>(x[0] * f, x[1] * f), pack2<__half>(x[2] * f, x[3] * f));
        if (lane == 0) row_scales[r] = p.scale2 * __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    }
    // bias: the heads' values by bucket, buckets by position over this block's keys
    const bool biased = p.rel.per_side != 0;
    const int head0 = row0 / p.Lq, heads = (row0 + rows - 1) / p.Lq - head0 + 1;  // of this block, within the key head's
    float* values = reinterpret_cast<float*>(base + L::kBias);
    uint8_t* buckets = base + L::kBias + (biased ? heads * p.rel.total * 4 : 0);
    RelRange range;
    if (biased) {
        for (int e = threadIdx.x; e < heads * p.rel.total; e += kWarps * 32)
            values[e] = bias_value<T>(static_cast<const T*>(p.table)[(static_cast<int64_t>(g) * group + head0) * p.rel.total + e]) * kLog2eF;
        range = rel_range(p.rel, first * kKeys - (p.Lq - 1) - p.rel.q_offset, last * kKeys - 1 - p.rel.q_offset);
        if (last > first) build_buckets(p.rel, range, buckets, threadIdx.x, kWarps * 32);
    }
    __syncthreads();

    // this lane's rows: 2 t4 + {0, 1} of each 8; its keys: g8 + 8 {0 .. 3}
    float o[NB][DP / 16][4], top_n[NB][2], top_m[NB][2], sum[NB][2], rscale[NB][2];
    const float* tables[NB][2];
    int token[NB][2];
#pragma unroll
    for (int x = 0; x < NB; ++x) {
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) o[x][i][0] = o[x][i][1] = o[x][i][2] = o[x][i][3] = 0.0f;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int r = x * 8 + 2 * t4 + z;
            top_n[x][z] = top_m[x][z] = -INFINITY;
            sum[x][z] = 0.0f;
            rscale[x][z] = row_scales[r];
            tables[x][z] = values + (min(row0 + r, row0 + rows - 1) / p.Lq - head0) * p.rel.total;
            token[x][z] = (row0 + r) % p.Lq;
        }
    }
    // queries: B fragments, dims 4 t4 + {0 .. 3} of each 16 of row g8 of each 8; kept where registers allow
    constexpr bool kKeep = NB <= 2;
    uint2 qf[kKeep ? NB : 1][kKeep ? DP / 16 : 1];
    const uint8_t* q_at = base + L::kQ + g8 * L::kQPitch + t4 * 8;
    if constexpr (kKeep)
#pragma unroll
        for (int x = 0; x < NB; ++x)
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) qf[x][d] = *reinterpret_cast<const uint2*>(q_at + x * 8 * L::kQPitch + d * 32);

    const float* ks = p.ks + b * p.ks_strides[0] + g * p.ks_strides[1];
    const float* vs = p.vs + b * p.vs_strides[0] + g * p.vs_strides[1];
    float key_scale = 0.0f, value_scale = 0.0f;  // of key `lane` of the tile to come
    uint8_t byte = 1;
    const auto ahead = [&](int i) {
        const int key = (first + warp + kWarps * i) * kKeys + lane;
        if (key < len) {
            key_scale = __ldg(ks + key);
            value_scale = __ldg(vs + key);
            if (p.key_mask != nullptr) byte = __ldg(p.key_mask + static_cast<int64_t>(b) * p.Lk + key);
        }
    };
    if (n > 0) ahead(0);
    const int mat = (lane & 7) + (lane & 8), half = lane >> 4;  // row and piece of a lane's ldmatrix address
    bool ok = true;
    for (int i = 0; i < n; ++i) {
        const int s = i % S, key0 = (first + warp + kWarps * i) * kKeys;
        const uint32_t kt = ring + s * 2 * L::kTile, vt = kt + L::kTile;
        const uint32_t keep = __ballot_sync(~0u, key0 + lane < len && byte != 0);
        const float my_k = key_scale;
        float my_v;  // log2 of the value's scale
        asm("lg2.approx.f32 %0, %1;" : "=f"(my_v) : "f"(value_scale));
        if (i + 1 < n) ahead(i + 1);
        ok = ok && umma::mbar_poll(bars + s * 8, (i / S) & 1);
        float sc[NB][2][4];
#pragma unroll
        for (int x = 0; x < NB; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h) sc[x][h][0] = sc[x][h][1] = sc[x][h][2] = sc[x][h][3] = 0.0f;
#pragma unroll
        for (int d = 0; d < DP / 16; d += 2)
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // 16 keys x 32 dims
                uint32_t w[4];
                ldmatrix_x4(piece<DP>(kt, h * 16 + mat, d + half), w);
#pragma unroll
                for (int z = 0; z < 4; ++z) w[z] ^= 0x80808080u;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const uint32_t a0 = to_half2<0x4140>(w[2 * y]), a1 = to_half2<0x4140>(w[2 * y + 1]),
                                   a2 = to_half2<0x4342>(w[2 * y]), a3 = to_half2<0x4342>(w[2 * y + 1]);
#pragma unroll
                    for (int x = 0; x < NB; ++x) {
                        const uint2 q = kKeep ? qf[kKeep ? x : 0][kKeep ? d + y : 0]
                                              : *reinterpret_cast<const uint2*>(q_at + x * 8 * L::kQPitch + (d + y) * 32);
                        umma::mma_16x8x16_f16f32(sc[x][h], a0, a1, a2, a3, q.x, q.y);
                    }
                }
            }
        int bucket = 0;
        bool one = true;  // the tile's positions lie in one bucket for every token
        const int rel0 = key0 - p.rel.q_offset;
        if (biased) {
            bucket = bucket_at(range, buckets, rel0 - (p.Lq - 1));
            one = bucket == bucket_at(range, buckets, rel0 + kKeys - 1);
        }
        uint32_t pf[NB][4];  // P, keys x rows: 8 keys each
        {
            float kk[4], vv[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                kk[c] = __shfl_sync(~0u, my_k, c * 8 + g8);
                vv[c] = __shfl_sync(~0u, my_v, c * 8 + g8);
            }
#pragma unroll
            for (int x = 0; x < NB; ++x) {
                float w[4][2], v[2][4];
                if (one) {  // a tile's bias is one value a row, or none
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const float flat = biased ? tables[x][z][bucket] : 0.0f;
#pragma unroll
                        for (int c = 0; c < 4; ++c) v[z][c] = fmaf(sc[x][c / 2][c % 2 * 2 + z], kk[c] * rscale[x][z], flat);
                    }
                } else {
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const uint8_t* by = buckets + rel0 + g8 - token[x][z] - range.lo;
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            v[z][c] = fmaf(sc[x][c / 2][c % 2 * 2 + z], kk[c] * rscale[x][z], tables[x][z][by[c * 8]]);
                    }
                }
                if (keep != ~0u) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (!((keep >> (c * 8 + g8)) & 1)) {
                            v[0][c] = v[1][c] = -INFINITY;
                            vv[c] = 0.0f;  // whatever the place holds
                        }
                }
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const float m = fmaxf(fmaxf(fmaxf(v[z][0], v[z][1]), fmaxf(v[z][2], v[z][3])), top_m[x][z]), ms = m == -INFINITY ? 0.0f : m;
                    float add = 0.0f;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        add += exp2_approx(v[z][c] - ms);
                        w[c][z] = v[z][c] + vv[c];
                    }
                    sum[x][z] = fmaf(sum[x][z], exp2_approx(top_m[x][z] - ms), add);
                    top_m[x][z] = m;
                }
                const float h0 = fmaxf(fmaxf(w[0][0], w[1][0]), fmaxf(w[2][0], w[3][0]));
                const float h1 = fmaxf(fmaxf(w[0][1], w[1][1]), fmaxf(w[2][1], w[3][1]));
                if (__any_sync(~0u, h0 > top_n[x][0] + kRescale || h1 > top_n[x][1] + kRescale)) {
                    float f[2];
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        float top = z ? h1 : h0;
#pragma unroll
                        for (int e = 4; e < 32; e *= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, e));
                        const float nn = fmaxf(top_n[x][z], top);
                        f[z] = top_n[x][z] == -INFINITY ? 0.0f : exp2_approx(top_n[x][z] - nn);
                        top_n[x][z] = nn;
                    }
#pragma unroll
                    for (int e = 0; e < DP / 16; ++e) {
                        o[x][e][0] *= f[0];
                        o[x][e][1] *= f[1];
                        o[x][e][2] *= f[0];
                        o[x][e][3] *= f[1];
                    }
                }
                const float n0 = top_n[x][0] == -INFINITY ? 0.0f : top_n[x][0] - kHead, n1 = top_n[x][1] == -INFINITY ? 0.0f : top_n[x][1] - kHead;
#pragma unroll
                for (int c = 0; c < 4; ++c) pf[x][c] = transpose(pack2<__half>(exp2_approx(w[c][0] - n0), exp2_approx(w[c][1] - n1)));
            }
        }
#pragma unroll
        for (int d = 0; d < DP / 16; d += 2)
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // 16 keys x 32 dims
                uint32_t w[4];
                umma::ldmatrix_x4_trans(piece<DP>(vt, h * 16 + mat, d + half), w);
#pragma unroll
                for (int z = 0; z < 4; ++z) w[z] ^= 0x80808080u;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const uint32_t a0 = to_half2<0x4240>(w[2 * y]), a1 = to_half2<0x4341>(w[2 * y]),
                                   a2 = to_half2<0x4240>(w[2 * y + 1]), a3 = to_half2<0x4341>(w[2 * y + 1]);
#pragma unroll
                    for (int x = 0; x < NB; ++x) umma::mma_16x8x16_f16f32(o[x][d + y], a0, a1, a2, a3, pf[x][2 * h], pf[x][2 * h + 1]);
                }
            }
        __syncwarp();  // the tile has been read
        if (lane == 0 && i + S < n && ok) load(i + S);
    }
    if (!ok) record_device_error(p.err, kErrMbarTimeout | 0x41);

    // the warps' rows: each puts its own in place of its ring; o of dims 2 g8 + {0, 1} of each 16
    float* mine = reinterpret_cast<float*>(base + warp * L::kRing);
    float* ml = reinterpret_cast<float*>(base + L::kMl);  // [warp][row] x {n, m, sum}
    __syncwarp();
#pragma unroll
    for (int x = 0; x < NB; ++x)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int r = x * 8 + 2 * t4 + z;
            float m = top_m[x][z];
#pragma unroll
            for (int e = 4; e < 32; e *= 2) m = fmaxf(m, __shfl_xor_sync(~0u, m, e));
            float l = sum[x][z] * (top_m[x][z] == -INFINITY ? 1.0f : exp2_approx(top_m[x][z] - m));
#pragma unroll
            for (int e = 4; e < 32; e *= 2) l += __shfl_xor_sync(~0u, l, e);
            if (g8 == 0) {
                float* to = ml + (warp * kRows + r) * 3;
                to[0] = top_n[x][z];
                to[1] = m;
                to[2] = l;
            }
#pragma unroll
            for (int e = 0; e < DP / 16; ++e)
                *reinterpret_cast<float2*>(mine + r * DP + e * 16 + 2 * g8) = make_float2(o[x][e][z], o[x][e][2 + z]);
        }
    __syncthreads();
    // the warps' rows joined: unnormalised values, the maximum and the sum
    float v[L::kItems][8], tops[L::kItems], totals[L::kItems];
    const int pieces = p.D / 8, items = rows * pieces;
#pragma unroll
    for (int n = 0; n < L::kItems; ++n) {
        const int e = threadIdx.x + n * kWarps * 32;
        tops[n] = -INFINITY;
        totals[n] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[n][j] = 0.0f;
        if (e >= items) continue;
        const int r = e / pieces, d = e % pieces * 8;
        for (int w = 0; w < kWarps; ++w) tops[n] = fmaxf(tops[n], ml[(w * kRows + r) * 3 + 1]);
        const float ms = tops[n] == -INFINITY ? 0.0f : tops[n];
        for (int w = 0; w < kWarps; ++w) {
            const float* x = ml + (w * kRows + r) * 3;
            totals[n] += x[1] == -INFINITY ? x[2] : exp2_approx(x[1] - ms) * x[2];  // a NaN sum has no maximum
            // a warp without keys, or whose values are all 0, has n = -inf and zeros
            const float f = x[0] == -INFINITY ? 1.0f : exp2_approx(x[0] - kHead - ms);
            const float* from = reinterpret_cast<const float*>(base + w * L::kRing) + r * DP + d;
            for (int j = 0; j < 8; ++j) v[n][j] += f * from[j];
        }
    }
    const auto finish = [&](int r, int d, float top, float total, const float (&o)[8]) {
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        const int h = g * group + (row0 + r) / p.Lq, i = (row0 + r) % p.Lq;
        const int64_t row = (static_cast<int64_t>(b) * p.Lq + i) * p.Hq + h;
        const float lse2 = total == 0.0f ? -INFINITY : (top == -INFINITY ? 0.0f : top) + log2f(total);
        if (p.splits > 1 && !p.joined) {
            const int64_t part = static_cast<int64_t>(blockIdx.x) * p.rows + row0 + r;  // [item][split][row]
            float* to = p.part_o + part * p.D + d;
            *reinterpret_cast<float4*>(to) = make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
            *reinterpret_cast<float4*>(to + 4) = make_float4(o[4] * inv, o[5] * inv, o[6] * inv, o[7] * inv);
            if (d == 0) p.part_lse[part] = lse2;
        } else {
            *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row * p.D + d) =
                make_uint4(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv),
                           pack2<T>(o[4] * inv, o[5] * inv), pack2<T>(o[6] * inv, o[7] * inv));
            if (d == 0 && p.lse != nullptr) p.lse[(static_cast<int64_t>(b) * p.Hq + h) * p.Lq + i] = lse2 * kLn2F;
        }
    };
    if (!p.joined) {
#pragma unroll
        for (int n = 0; n < L::kItems; ++n) {
            const int e = threadIdx.x + n * kWarps * 32;
            if (e < items) finish(e / pieces, e % pieces * 8, tops[n], totals[n], v[n]);
        }
        return;
    }
    // the cluster's blocks put theirs into their shared memory; each joins a share of the rows
    // from all of them, in order
    float* block_o = reinterpret_cast<float*>(base);
    float2* block_ml = reinterpret_cast<float2*>(base + kRows * DP * 4);
    __syncthreads();  // the warps' rows have been read
#pragma unroll
    for (int n = 0; n < L::kItems; ++n) {
        const int e = threadIdx.x + n * kWarps * 32;
        if (e >= items) continue;
        float4* to = reinterpret_cast<float4*>(block_o + e * 8);
        to[0] = make_float4(v[n][0], v[n][1], v[n][2], v[n][3]);
        to[1] = make_float4(v[n][4], v[n][5], v[n][6], v[n][7]);
        if (e % pieces == 0) block_ml[e / pieces] = make_float2(tops[n], totals[n]);
    }
    const auto cluster = cooperative_groups::this_cluster();
    cluster.sync();
    const int e0 = items * split / p.splits, e1 = items * (split + 1) / p.splits;
    for (int e = e0 + threadIdx.x; e < e1; e += kWarps * 32) {
        const int r = e / pieces;
        float top = -INFINITY, total = 0.0f, o[8] = {};
        for (int c = 0; c < p.splits; ++c) top = fmaxf(top, cluster.map_shared_rank(block_ml, c)[r].x);
        const float ms = top == -INFINITY ? 0.0f : top;
        for (int c = 0; c < p.splits; ++c) {
            const float2 x = cluster.map_shared_rank(block_ml, c)[r];
            const float4* from = reinterpret_cast<const float4*>(cluster.map_shared_rank(block_o, c) + e * 8);
            const float f = x.x == -INFINITY ? 1.0f : exp2_approx(x.x - ms);  // zeros, or a NaN sum
            const float4 lo = from[0], hi = from[1];
            total += f * x.y;
            o[0] += f * lo.x;
            o[1] += f * lo.y;
            o[2] += f * lo.z;
            o[3] += f * lo.w;
            o[4] += f * hi.x;
            o[5] += f * hi.y;
            o[6] += f * hi.z;
            o[7] += f * hi.w;
        }
        finish(r, e % pieces * 8, top, total, o);
    }
    cluster.sync();  // until the others have read this block's
}

template <typename T, int DP, int NB>
int launch(const Int8Params& f, int64_t items, cudaStream_t stream) noexcept
{
    using L = Layout<DP, NB>;
    const auto kernel = attention_int8_kernel<T, DP, NB>;
    static_assert(L::kBytes + NB * 8 * kMaxBuckets * 4 + kMaxPositions <= kMaxShared, "shared memory");
    const int bytes = L::kBytes + (f.table != nullptr ? std::min(L::kRows, f.Hq / f.Hk) * f.rel.total * 4 + f.max_entries : 0);
    static std::atomic<uint64_t> raised{0};
    if (!allow_shared_memory(reinterpret_cast<const void*>(kernel), raised)) return launch_status("cross_attention_int8");
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(f.splits);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(items * f.splits), (f.rows + L::kRows - 1) / L::kRows);
    cfg.blockDim = L::kWarps * 32;
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = f.joined ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, f);
    return launch_status("cross_attention_int8");
}

template <typename T, int DP>
int launch_rows(const Int8Params& f, int64_t items, cudaStream_t stream) noexcept
{
    return f.rows <= 8 ? launch<T, DP, 1>(f, items, stream) : f.rows <= 16 ? launch<T, DP, 2>(f, items, stream) : launch<T, DP, 4>(f, items, stream);
}

// How a call runs: rows against the 8-bit values, keys split over blocks; or 16-bit
// copies in the workspace and the kernels of ww_cross_attention.
struct Plan {
    bool few, joined;  // joined: the splits are a cluster, which joins them itself
    int rows, row_blocks, splits;
    int64_t part_rows(const ww_attention_t& p) const { return splits > 1 && !joined ? i64(p.B) * p.Hk * splits * rows : 0; }
    void without_parts()
    {
        splits = std::min(splits, kCluster);
        joined = splits > 1;
    }
};

// Copies cost 5 bytes a value and three launches, but are converted once for all rows.  us in 8 bits and by copies:
// more than 64 rows (converted 3 or 4 times), 8 x 8 key heads of 64 and 128, 1500 keys, 128 rows 33 and 38, 48 and 46,
// 1 x 8, 40001 keys 80 and 76, 120 and 105.
// Short keys of more blocks than are resident (a block's start and end): 64 x 8, 100 keys, 32 rows of 64 21 and 21, 48 rows of 128 46 and 27.
constexpr int64_t kManyKeys = 1 << 17;  // of all items and key heads
constexpr int kShortKeys = 512;
bool by_copies(const ww_attention_t& p, int64_t rows, int sms) noexcept
{
    if (rows > kMostRows) return true;
    if (p.dtype == WW_DTYPE_BF16) return false;  // whose rounding of keys and values shows: 0.4 % of the result, 0.17 its own
    const int64_t heads = i64(p.B) * p.Hk, row_blocks = (rows + 31) / 32;
    return (rows > 64 && heads * p.Lk >= kManyKeys) || (rows > 32 && p.Lk < kShortKeys && p.Lk > 0 && heads * row_blocks > 2 * sms);
}

Plan make_plan(const ww_attention_t& p, int sms, bool copies_fit = true) noexcept
{
    Plan r{};
    const int64_t rows = i64(p.Hq / p.Hk) * p.Lq;
    r.few = rows <= kMostRows && !(copies_fit && by_copies(p, rows, sms));
    if (!r.few) return r;
    r.rows = static_cast<int>(rows);
    r.row_blocks = (r.rows + 31) / 32;
    const int64_t items = i64(p.B) * p.Hk * r.row_blocks, tiles = (p.Lk + kKeys - 1) / kKeys;
    // two blocks per SM; a block has a tile for each of its warps at least
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>({items > 0 ? 2 * sms / items : 1, tiles / 6, 128}));
    r.splits = static_cast<int>(most);
    // short keys: a cluster, which saves a launch
    if (most > kCluster && tiles <= kCluster * kShort) r.splits = kCluster;
    r.joined = r.splits > 1 && r.splits <= kCluster;
    return r;
}

int64_t aligned(int64_t n) noexcept { return (n + 255) / 256 * 256; }

// Workspace of the 16-bit form: (powers,) keys, values, then that of ww_cross_attention.
int64_t copy_bytes(const ww_attention_t& p) noexcept { return aligned(i64(p.B) * p.Lk * p.Hk * p.D * 2); }

// In front of them in fp16, whose range is narrower than the scales': a power of two for each head's keys and values, by which
// the copies are divided and which scores and results take back.  A workspace of the copies alone does without.
int64_t power_bytes(const ww_attention_t& p) noexcept { return p.dtype == WW_DTYPE_HALF ? aligned(i64(p.B) * p.Hk * 8) : 0; }

ww_attention_t of_copies(const ww_attention_int8_t& a, bool powers) noexcept
{
    ww_attention_t p = a.attention;
    char* ws = static_cast<char*>(p.workspace);
    const int64_t n = copy_bytes(p);
    if (ws == nullptr) ws = reinterpret_cast<char*>(static_cast<uintptr_t>(256));  // sizes only
    const int64_t before = powers ? power_bytes(p) : 0;
    ws += before;
    p.k = ws;
    p.v = ws + n;
    p.workspace = ws + 2 * n;
    p.workspace_bytes -= 2 * n + before;
    for (int64_t* s : {p.k_strides, p.v_strides}) {
        s[0] = i64(p.Lk) * p.Hk * p.D;
        s[1] = i64(p.Hk) * p.D;
        s[2] = p.D;
    }
    return p;
}

int64_t workspace(const ww_attention_int8_t& a, const Plan& plan) noexcept
{
    const ww_attention_t& p = a.attention;
    if (p.B == 0 || p.Lq == 0) return 0;
    if (plan.few) return plan.part_rows(p) * (p.D + 1) * 4;
    const ww_attention_t q = of_copies(a, true);
    return power_bytes(p) + 2 * copy_bytes(p) + ww_cross_attention_workspace(&q);
}

int check(const ww_attention_int8_t& a) noexcept
{
    ww_attention_t p = a.attention;
    // the caches' strides are in bytes; check_attention counts 2 to a value
    const bool has_k = p.B > 0 && p.Lk > 0;
    const int n[3] = {p.B, p.Lk, p.Hk};
    for (int64_t* s : {p.k_strides, p.v_strides})
        for (int i = 0; i < 3; ++i) {
            if (has_k && n[i] > 1 && s[i] >= 0 && s[i] % 16 != 0) return WW_ERR_MISALIGNED;
            if (s[i] > 0) s[i] = 8;
        }
    const int st = check_attention(p);
    if (st != WW_SUCCESS) return st;
    if (p.D % 16 != 0) return WW_ERR_UNSUPPORTED;
    if (!has_k) return WW_SUCCESS;
    if (i64(p.B) * p.Hk > (1 << 22) || i64(p.B) * p.Lk >= INT32_MAX || i64(p.B) * p.Lk * p.Hk >= INT32_MAX) return WW_ERR_UNSUPPORTED;
    if (a.k_scale == nullptr || a.v_scale == nullptr) return WW_ERR_NULL_POINTER;
    if (reinterpret_cast<uintptr_t>(a.k_scale) % 4 != 0 || reinterpret_cast<uintptr_t>(a.v_scale) % 4 != 0) return WW_ERR_MISALIGNED;
    for (const int64_t(*s)[2] : {&a.k_scale_strides, &a.v_scale_strides})
        if ((p.B > 1 && (*s)[0] < 0) || (p.Hk > 1 && (*s)[1] < 0)) return WW_ERR_INVALID_SHAPE;
    return WW_SUCCESS;
}

template <typename T>
int few_rows(const ww_attention_int8_t& a, const Plan& plan, cudaStream_t stream) noexcept
{
    const ww_attention_t& p = a.attention;
    Int8Params f{};
    const int dp = p.D <= 32 ? 32 : p.D <= 64 ? 64 : 128;
    const int nk[3] = {p.B, p.Lk, p.Hk};
    if (p.Lk > 0 && (!encode_bytes_map(&f.k, p.k, p.D, nk, p.k_strides, dp, kKeys) ||
                     !encode_bytes_map(&f.v, p.v, p.D, nk, p.v_strides, dp, kKeys)))
        return WW_ERR_UNSUPPORTED;
    f.ks = a.k_scale;
    f.vs = a.v_scale;
    f.q = p.q;
    f.out = p.out;
    f.lse = p.lse;
    f.k_lens = p.k_lens;
    f.key_mask = p.key_mask;
    f.table = p.bias_table;
    if (p.bias_table != nullptr) {
        make_buckets(p.num_buckets, p.max_distance, p.bidirectional, p.q_offset, &f.rel);
        f.max_entries = static_cast<int>(std::min<int64_t>(rel_positions(p.max_distance), i64(p.Lk) + 2 * kKeys + p.Lq));
    }
    f.part_o = static_cast<float*>(p.workspace);
    f.part_lse = f.part_o + plan.part_rows(p) * p.D;
    for (int i = 0; i < 3; ++i) f.q_strides[i] = p.q_strides[i];
    for (int i = 0; i < 2; ++i) {
        f.ks_strides[i] = a.k_scale_strides[i];
        f.vs_strides[i] = a.v_scale_strides[i];
    }
    f.B = p.B;
    f.Lq = p.Lq;
    f.Lk = p.Lk;
    f.Hq = p.Hq;
    f.Hk = p.Hk;
    f.D = p.D;
    f.rows = plan.rows;
    f.splits = plan.splits;
    f.joined = plan.joined;
    f.k_b = p.k_strides[0] != 0;
    f.k_h = p.k_strides[2] != 0;
    f.v_b = p.v_strides[0] != 0;
    f.v_h = p.v_strides[2] != 0;
    f.scale2 = p.scale * kLog2eF;
    f.err = device_error_slot();
    if (f.err == nullptr) return WW_ERR_DEVICE;
    const int64_t items = i64(p.B) * p.Hk;
    const int st = dp == 32 ? launch_rows<T, 32>(f, items, stream) : dp == 64 ? launch_rows<T, 64>(f, items, stream) : launch_rows<T, 128>(f, items, stream);
    if (st != WW_SUCCESS || plan.splits == 1 || plan.joined) return st;
    return attention_join_launch(p, static_cast<int>(items), plan.splits, plan.rows, f.part_o, f.part_lse, "cross_attention_int8", stream);
}

int sm_count() noexcept
{
    DeviceInfo d;
    return current_device_info(&d) == WW_SUCCESS ? d.sm_count : 148;
}

}  // namespace
}  // namespace ww

extern "C" {

int64_t ww_cross_attention_int8_workspace(const ww_attention_int8_t* p)
{
    return p == nullptr || ww::check(*p) != WW_SUCCESS ? 0 : ww::workspace(*p, ww::make_plan(p->attention, ww::sm_count()));
}

int ww_cross_attention_int8(const ww_attention_int8_t* a, void* stream)
{
    if (a == nullptr) return WW_ERR_NULL_POINTER;
    const ww_attention_t& p = a->attention;
    int st = ww::check(*a);
    if (st != WW_SUCCESS || p.B == 0 || p.Lq == 0) return st;
    ww::Plan plan = ww::make_plan(p, ww::sm_count(), p.workspace != nullptr);
    if (plan.few) {
        if (p.workspace == nullptr) plan.without_parts();
        else if (ww::workspace(*a, plan) > p.workspace_bytes) return WW_ERR_UNSUPPORTED;
    } else {
        if (p.Lk > 0 && p.workspace == nullptr) return WW_ERR_NULL_POINTER;
        if (2 * ww::copy_bytes(p) > p.workspace_bytes) return WW_ERR_UNSUPPORTED;
    }
    ww::DeviceInfo d;
    if ((st = ww::current_device_info(&d)) != WW_SUCCESS) return st;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (plan.few) return p.dtype == WW_DTYPE_HALF ? ww::few_rows<__half>(*a, plan, s) : ww::few_rows<__nv_bfloat16>(*a, plan, s);
    const bool has_powers = p.Lk > 0 && ww::power_bytes(p) > 0 && ww::power_bytes(p) + 2 * ww::copy_bytes(p) <= p.workspace_bytes;
    ww_attention_t q = ww::of_copies(*a, has_powers);
    if (ww_cross_attention_workspace(&q) > q.workspace_bytes) q.workspace = nullptr;  // keys are not split then
    ww_kv_cache_t c{};
    c.k_cache = static_cast<int8_t*>(const_cast<void*>(p.k));
    c.v_cache = static_cast<int8_t*>(const_cast<void*>(p.v));
    c.k_scale = const_cast<float*>(a->k_scale);
    c.v_scale = const_cast<float*>(a->v_scale);
    c.lens = p.k_lens;
    c.k_out = const_cast<void*>(q.k);
    c.v_out = const_cast<void*>(q.v);
    for (int i = 0; i < 3; ++i) {
        c.k_cache_strides[i] = p.k_strides[i];
        c.v_cache_strides[i] = p.v_strides[i];
    }
    for (int i = 0; i < 2; ++i) {
        c.k_scale_strides[i] = a->k_scale_strides[i];
        c.v_scale_strides[i] = a->v_scale_strides[i];
    }
    c.dtype = p.dtype;
    c.B = p.B;
    c.places = p.Lk;
    c.H = p.Hk;
    c.D = p.D;
    float2* powers = has_powers ? static_cast<float2*>(p.workspace) : nullptr;
    if (p.Lk > 0 && (st = ww::dequantise_valid(c, p.key_mask, powers, "cross_attention_int8", stream)) != WW_SUCCESS) return st;
    return ww::cross_attention(q, powers, stream);
}

}  // extern "C"
