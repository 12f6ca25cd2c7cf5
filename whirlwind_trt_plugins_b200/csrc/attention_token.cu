// attention_token.cu -- ww_cross_attention for a few query rows per key head
// (one token of a decoder against an encoder's states, with the query heads
// that share a key head as further rows).
//
// Bound: HBM -- every key and value is read once, 4 flops per byte and row.
// The rows of a key head (query heads x tokens, up to 16 or 32) are one M tile
// of mma.sync m16n8k16, so that shared heads read their keys once; tcgen05's
// 128 rows would be almost all padding.
// Each of 8 warps runs alone over every 8th tile of 16 or 32 keys of its CTA's
// share: one lane keeps a ring of TMA loads in flight (swizzled rows, read back
// by ldmatrix without conflicts; up to 128 KB per SM), the warp computes scores,
// the running maximum and sum and O in registers, and no barrier joins the warps
// before the end.  O is rescaled only when a maximum has grown by 2^8.
// The keys are split over CTAs until the GPU is full; the partial rows are
// joined by attention_join_kernel (attention_forward.cu) in order.
//
// Measured, bf16: one token of 2 x 32 heads on 8 key heads of 128 against 40001 keys
// with a bias, 328 MB: 55 us, 6.0 TB/s, and 6 us to join.  Eight items of up to 1500
// keys, 16 heads on 4 of 64: 9 us, and 6 to join.
#include "attention_token.cuh"
#include "tensor_map.cuh"
#include "umma.cuh"

#include <algorithm>

namespace ww {
namespace {

constexpr int kWarps = 8;
constexpr float kRescale = 8.0f;  // log2 growth of a maximum that is left in P

// Keys of a warp's tile: 8 KB of keys and values at D = 64 and 128.
constexpr int tile_keys(int dp) { return dp == 128 ? 16 : 32; }

struct TokenParams {
    CUtensorMap k, v;
    const void* q;
    void* out;
    float* lse;
    const int32_t* k_lens;
    const uint8_t* key_mask;
    const void* table;
    float* part_o;
    float* part_lse;
    RelBuckets rel;
    int64_t q_strides[3];
    int32_t B, Lq, Lk, Hq, Hk, D, rows;
    int32_t splits;
    int32_t k_b, k_h, v_b, v_h;
    int32_t max_entries;
    float scale2;
    int* err;
};

template <int DP, int MB>
struct Layout {
    static constexpr int kKeys = tile_keys(DP);
    static constexpr int kRow = DP == 32 ? 64 : 128;
    static constexpr int kChunks = DP * 2 / kRow;
    static constexpr int kChunkBytes = kKeys * kRow;
    static constexpr int kTileBytes = kKeys * DP * 2;
    static constexpr int kStages = DP == 32 ? 4 : 3;
    static constexpr int kRing = kStages * 2 * kTileBytes;            // of a warp
    static constexpr int kQPitch = DP * 2 + 16;                       // bytes, ldmatrix without conflicts
    static constexpr int kQ = kWarps * kRing;
    static constexpr int kBar = kQ + MB * 16 * kQPitch;
    static constexpr int kMl = kBar + kWarps * kStages * 8;           // maximum and sum of [warp][row]
    static constexpr int kBias = kMl + kWarps * MB * 16 * 8;          // [heads][buckets] values, [entries] buckets
    static constexpr int kBytes = kBias + 1024;
    static_assert(MB * 16 * DP * 4 <= kRing, "a warp's rows replace its ring at the end");
};

// 16-byte piece j of row r of a swizzled tile.
template <int kRow>
__device__ __forceinline__ uint32_t piece(uint32_t tile, int r, int j)
{
    return kRow == 128 ? tile + r * 128 + ((j ^ (r & 7)) << 4) : tile + r * 64 + ((j ^ ((r >> 1) & 3)) << 4);
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t saddr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(saddr)
                 : "memory");
}

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    umma::mma_16x8x16_f16f32(d, a[0], a[1], a[2], a[3], b0, b1);
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                 "{%8, %9}, {%0, %1, %2, %3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int DP, int MB>
__global__ void __launch_bounds__(kWarps * 32, 1) attention_token_kernel(const __grid_constant__ TokenParams p)
{
    using L = Layout<DP, MB>;
    constexpr int S = L::kStages, kKeys = L::kKeys;
    constexpr int kRows = MB * 16;
    extern __shared__ uint8_t raw[];
    uint8_t* base = raw + ((1024 - (umma::smem_addr(raw) & 1023)) & 1023);
    const uint32_t sm = umma::smem_addr(base);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t ring = sm + warp * L::kRing, bars = sm + L::kBar + warp * S * 8;

    const int split = blockIdx.x % p.splits;
    const int g = blockIdx.x / p.splits % p.Hk, b = blockIdx.x / p.splits / p.Hk;
    const int len = p.k_lens == nullptr ? p.Lk : min(max(__ldg(p.k_lens + b), 0), p.Lk);
    const int all = (len + kKeys - 1) / kKeys;
    int first, count;
    part_of(all, split, p.splits, first, count);
    const int last = first + count;
    const int n = (last - first - warp + kWarps - 1) / kWarps;  // tiles of this warp: first + warp + kWarps i
    const int group = p.Hq / p.Hk;

    const auto load = [&](int i) {  // lane 0
        const int s = i % S, key = (first + warp + kWarps * i) * kKeys;
        umma::mbar_arrive_expect_tx(bars + s * 8, 2 * L::kTileBytes);
#pragma unroll
        for (int c = 0; c < L::kChunks; ++c) {
            const uint32_t to = ring + s * 2 * L::kTileBytes + c * L::kChunkBytes;
            umma::tma_load_4d(to, &p.k, c * L::kRow / 2, g * p.k_h, key, b * p.k_b, bars + s * 8);
            umma::tma_load_4d(to + L::kTileBytes, &p.v, c * L::kRow / 2, g * p.v_h, key, b * p.v_b, bars + s * 8);
        }
    };
    if (lane == 0) {
        for (int s = 0; s < S; ++s) umma::mbar_init(bars + s * 8, 1);
        umma::mbar_fence_init();
        umma::fence_proxy_async_smem();
        for (int i = 0; i < S && i < n; ++i) load(i);
    }
    // query rows: row r is head g * group + r / Lq, token r % Lq; the rest zeros
    for (int e = threadIdx.x; e < kRows * (DP / 8); e += kWarps * 32) {
        const int r = e / (DP / 8), d = e % (DP / 8) * 8;
        uint4 u = make_uint4(0, 0, 0, 0);
        if (r < p.rows && d < p.D)
            u = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + b * p.q_strides[0] +
                                                (r % p.Lq) * p.q_strides[1] + (g * group + r / p.Lq) * p.q_strides[2] + d);
        *reinterpret_cast<uint4*>(base + L::kQ + r * L::kQPitch + d * 2) = u;
    }
    // bias: the heads' values by bucket, buckets by position over this CTA's keys
    const bool biased = p.rel.per_side != 0;
    float* values = reinterpret_cast<float*>(base + L::kBias);
    uint8_t* buckets = base + L::kBias + (biased ? group * p.rel.total * 4 : 0);
    RelRange range;
    if (biased) {
        for (int e = threadIdx.x; e < group * p.rel.total; e += kWarps * 32)
            values[e] = bias_value<T>(static_cast<const T*>(p.table)[static_cast<int64_t>(g) * group * p.rel.total + e]) * kLog2eF;
        range = rel_range(p.rel, first * kKeys - (p.Lq - 1) - p.rel.q_offset, last * kKeys - 1 - p.rel.q_offset);
        if (last > first) build_buckets(p.rel, range, buckets, threadIdx.x, kWarps * 32);
    }
    __syncthreads();
    const uint32_t q_at = sm + L::kQ + (lane % 16) * L::kQPitch + (lane / 16) * 16;

    float o[MB][DP / 8][4];
    float m[MB][2], l[MB][2];
#pragma unroll
    for (int x = 0; x < MB; ++x) {
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) o[x][i][0] = o[x][i][1] = o[x][i][2] = o[x][i][3] = 0.0f;
        m[x][0] = m[x][1] = -INFINITY;
        l[x][0] = l[x][1] = 0.0f;
    }
    // query fragments of a single M tile stay in registers
    uint32_t qf[MB == 1 ? DP / 16 : 1][4];
    if (MB == 1)
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) ldmatrix_x4(q_at + d * 32, qf[d]);
    uint8_t byte = 0;  // of the key mask, for the tile to come
    const auto mask_byte = [&](int i) {
        const int key = (first + warp + kWarps * i) * kKeys + lane;
        byte = lane < kKeys && key < len ? __ldg(p.key_mask + static_cast<int64_t>(b) * p.Lk + key) : 0;
    };
    if (p.key_mask != nullptr && n > 0) mask_byte(0);
    constexpr uint32_t kAll = kKeys == 32 ? ~0u : (1u << (kKeys & 31)) - 1;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
        const int s = i % S, key0 = (first + warp + kWarps * i) * kKeys;
        const uint32_t kt = ring + s * 2 * L::kTileBytes, vt = kt + L::kTileBytes;
        uint32_t keep = len - key0 >= kKeys ? kAll : (1u << (len - key0)) - 1;
        if (p.key_mask != nullptr) {
            keep &= __ballot_sync(~0u, byte != 0);
            if (i + 1 < n) mask_byte(i + 1);
        }
        ok = ok && umma::mbar_poll(bars + s * 8, (i / S) & 1);
        if (keep != kAll) {
            // rows of V behind masked keys: 0 in place of whatever they hold
            __syncwarp();
            if (lane < kKeys && !((keep >> lane) & 1))
                for (int c = 0; c < L::kChunks; ++c)
#pragma unroll
                    for (int j = 0; j < L::kRow; j += 16)
                        umma::st_shared_v4(vt + c * L::kChunkBytes + lane * L::kRow + j, 0, 0, 0, 0);
            __syncwarp();
        }
        float sc[MB][kKeys / 8][4];
#pragma unroll
        for (int x = 0; x < MB; ++x)
#pragma unroll
            for (int nb = 0; nb < kKeys / 8; ++nb) sc[x][nb][0] = sc[x][nb][1] = sc[x][nb][2] = sc[x][nb][3] = 0.0f;
#pragma unroll
        for (int d = 0; d < DP; d += 32) {
            uint32_t a[MB][2][4];
#pragma unroll
            for (int x = 0; x < MB; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    if (MB == 1) {
#pragma unroll
                        for (int z = 0; z < 4; ++z) a[x][y][z] = qf[MB == 1 ? d / 16 + y : 0][z];
                    } else {
                        ldmatrix_x4(q_at + x * 16 * L::kQPitch + d * 2 + y * 32, a[x][y]);
                    }
                }
            const uint32_t chunk = kt + d * 2 / L::kRow * L::kChunkBytes;
#pragma unroll
            for (int nb = 0; nb < kKeys / 8; ++nb) {
                uint32_t kb[4];  // 8 keys x 32 dims
                ldmatrix_x4(piece<L::kRow>(chunk, nb * 8 + lane % 8, d * 2 % L::kRow / 16 + lane / 8), kb);
#pragma unroll
                for (int x = 0; x < MB; ++x) {
                    mma<T>(sc[x][nb], a[x][0], kb[0], kb[1]);
                    mma<T>(sc[x][nb], a[x][1], kb[2], kb[3]);
                }
            }
        }
        // scores in log2 units; this lane: rows lane / 4 (+ 8), keys 2 (lane % 4) + {0, 1} of each 8
        int bucket = 0;
        bool one = true;  // the tile's positions lie in one bucket for every token
        const int rel0 = key0 - p.rel.q_offset;
        if (biased) {
            bucket = bucket_at(range, buckets, rel0 - (p.Lq - 1));
            one = bucket == bucket_at(range, buckets, rel0 + kKeys - 1);
        }
#pragma unroll
        for (int x = 0; x < MB; ++x)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int r = x * 16 + y * 8 + lane / 4;
                const float* table = biased && r < p.rows ? values + r / p.Lq * p.rel.total : nullptr;
                const uint8_t* by = buckets + rel0 - (r % p.Lq) - range.lo;
                const float flat = table != nullptr ? table[bucket] : 0.0f;
                float top = -INFINITY;
#pragma unroll
                for (int nb = 0; nb < kKeys / 8; ++nb)
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const int c = nb * 8 + 2 * (lane % 4) + z;
                        const float bias = !one && table != nullptr ? table[by[c]] : flat;
                        float v = fmaf(sc[x][nb][2 * y + z], p.scale2, bias);
                        v = (keep >> c) & 1 ? v : -INFINITY;
                        sc[x][nb][2 * y + z] = v;
                        top = fmaxf(top, v);
                    }
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                if (__any_sync(~0u, top > m[x][y] + kRescale || i == 0)) {
                    const float mn = fmaxf(m[x][y], top);
                    const float f = m[x][y] == -INFINITY ? 0.0f : exp2_approx(m[x][y] - mn);
                    m[x][y] = mn;
                    l[x][y] *= f;
#pragma unroll
                    for (int e = 0; e < DP / 8; ++e) {
                        o[x][e][2 * y] *= f;
                        o[x][e][2 * y + 1] *= f;
                    }
                }
                const float ms = m[x][y] == -INFINITY ? 0.0f : m[x][y];
#pragma unroll
                for (int nb = 0; nb < kKeys / 8; ++nb)
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const float pr = exp2_approx(sc[x][nb][2 * y + z] - ms);
                        l[x][y] += pr;
                        sc[x][nb][2 * y + z] = pr;
                    }
            }
#pragma unroll
        for (int h = 0; h < kKeys / 16; ++h) {  // 16 keys each
            uint32_t a[MB][4];
#pragma unroll
            for (int x = 0; x < MB; ++x) {
                a[x][0] = pack2<T>(sc[x][2 * h][0], sc[x][2 * h][1]);
                a[x][1] = pack2<T>(sc[x][2 * h][2], sc[x][2 * h][3]);
                a[x][2] = pack2<T>(sc[x][2 * h + 1][0], sc[x][2 * h + 1][1]);
                a[x][3] = pack2<T>(sc[x][2 * h + 1][2], sc[x][2 * h + 1][3]);
            }
#pragma unroll
            for (int d = 0; d < DP; d += 16) {
                uint32_t vb[4];  // 16 keys x 16 dims
                const uint32_t chunk = vt + d * 2 / L::kRow * L::kChunkBytes;
                umma::ldmatrix_x4_trans(
                    piece<L::kRow>(chunk, h * 16 + lane % 16, d * 2 % L::kRow / 16 + lane / 16), vb);
#pragma unroll
                for (int x = 0; x < MB; ++x) {
                    mma<T>(o[x][d / 8], a[x], vb[0], vb[1]);
                    mma<T>(o[x][d / 8 + 1], a[x], vb[2], vb[3]);
                }
            }
        }
        umma::fence_proxy_async_smem();  // this tile's reads and zeroed rows before the next load into its place
        __syncwarp();
        if (lane == 0 && i + S < n && ok) load(i + S);
    }
    if (!ok) record_device_error(p.err, kErrMbarTimeout | 0x40);

    // the warps' rows: each puts its own, unnormalised, in place of its ring
    float* mine = reinterpret_cast<float*>(base + warp * L::kRing);
    float2* ml = reinterpret_cast<float2*>(base + L::kMl);
    __syncwarp();
#pragma unroll
    for (int x = 0; x < MB; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const int r = x * 16 + y * 8 + lane / 4;
            float sum = l[x][y];
            sum += __shfl_xor_sync(~0u, sum, 1);
            sum += __shfl_xor_sync(~0u, sum, 2);
            if (lane % 4 == 0) ml[warp * kRows + r] = make_float2(m[x][y], sum);
#pragma unroll
            for (int e = 0; e < DP / 8; ++e)
                *reinterpret_cast<float2*>(mine + r * DP + e * 8 + 2 * (lane % 4)) =
                    make_float2(o[x][e][2 * y], o[x][e][2 * y + 1]);
        }
    __syncthreads();
    for (int e = threadIdx.x; e < p.rows * (p.D / 8); e += kWarps * 32) {
        const int r = e / (p.D / 8), d = e % (p.D / 8) * 8;
        float top = -INFINITY;
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w * kRows + r].x);
        const float ms = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f, v[8] = {};
        for (int w = 0; w < kWarps; ++w) {
            const float2 x = ml[w * kRows + r];
            const float f = exp2_approx(x.x - ms);
            sum += f * x.y;
            const float* from = reinterpret_cast<const float*>(base + w * L::kRing) + r * DP + d;
            for (int j = 0; j < 8; ++j) v[j] += f * from[j];
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int h = g * group + r / p.Lq, i = r % p.Lq;
        const int64_t row = (static_cast<int64_t>(b) * p.Lq + i) * p.Hq + h;
        const float lse2 = sum == 0.0f ? -INFINITY : ms + log2f(sum);
        if (p.splits > 1) {
            const int64_t part = static_cast<int64_t>(blockIdx.x) * p.rows + r;  // [item][split][row]
            float* to = p.part_o + part * p.D + d;
            *reinterpret_cast<float4*>(to) = make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
            *reinterpret_cast<float4*>(to + 4) = make_float4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
            if (d == 0) p.part_lse[part] = lse2;
        } else {
            *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row * p.D + d) =
                make_uint4(pack2<T>(v[0] * inv, v[1] * inv), pack2<T>(v[2] * inv, v[3] * inv),
                           pack2<T>(v[4] * inv, v[5] * inv), pack2<T>(v[6] * inv, v[7] * inv));
            if (d == 0 && p.lse != nullptr) p.lse[(static_cast<int64_t>(b) * p.Hq + h) * p.Lq + i] = lse2 * kLn2F;
        }
    }
}

template <typename T, int DP, int MB>
int launch(const TokenParams& f, int64_t ctas, cudaStream_t stream) noexcept
{
    using L = Layout<DP, MB>;
    const auto kernel = attention_token_kernel<T, DP, MB>;
    static_assert(L::kBytes + MB * 16 * kMaxBuckets * 4 + kMaxPositions <= kMaxShared, "shared memory");
    const int bytes = L::kBytes + (f.table != nullptr ? f.Hq / f.Hk * f.rel.total * 4 + f.max_entries : 0);
    static std::atomic<uint64_t> raised{0};
    if (!allow_shared_memory(reinterpret_cast<const void*>(kernel), raised)) return launch_status("cross_attention");
    kernel<<<static_cast<unsigned>(ctas), kWarps * 32, bytes, stream>>>(f);
    return launch_status("cross_attention");
}

template <typename T>
int tokens(const ww_attention_t& p, int splits, float* part_o, float* part_lse, cudaStream_t stream) noexcept
{
    TokenParams f;
    const int dp = p.D <= 32 ? 32 : p.D <= 64 ? 64 : 128;
    constexpr bool bf = !std::is_same<T, __half>::value;
    const int nk[3] = {p.B, p.Lk, p.Hk};
    if (p.Lk > 0 && (!encode_vectors_map(&f.k, bf, p.k, p.D, nk, p.k_strides, dp == 32 ? 32 : 64, tile_keys(dp)) ||
                     !encode_vectors_map(&f.v, bf, p.v, p.D, nk, p.v_strides, dp == 32 ? 32 : 64, tile_keys(dp))))
        return WW_ERR_UNSUPPORTED;
    f.q = p.q;
    f.out = p.out;
    f.lse = p.lse;
    f.k_lens = p.k_lens;
    f.key_mask = p.key_mask;
    f.table = p.bias_table;
    if (p.bias_table != nullptr)
        make_buckets(p.num_buckets, p.max_distance, p.bidirectional, p.q_offset, &f.rel);
    f.max_entries = 0;
    if (p.bias_table != nullptr)
        f.max_entries = static_cast<int>(std::min<int64_t>(rel_positions(p.max_distance), i64(p.Lk) + 64 + p.Lq));
    f.part_o = part_o;
    f.part_lse = part_lse;
    for (int i = 0; i < 3; ++i) f.q_strides[i] = p.q_strides[i];
    f.B = p.B;
    f.Lq = p.Lq;
    f.Lk = p.Lk;
    f.Hq = p.Hq;
    f.Hk = p.Hk;
    f.D = p.D;
    f.rows = p.Hq / p.Hk * p.Lq;
    f.splits = splits;
    f.k_b = p.k_strides[0] != 0;
    f.k_h = p.k_strides[2] != 0;
    f.v_b = p.v_strides[0] != 0;
    f.v_h = p.v_strides[2] != 0;
    f.scale2 = p.scale * kLog2eF;
    f.err = device_error_slot();
    if (f.err == nullptr) return WW_ERR_DEVICE;
    const int64_t ctas = i64(p.B) * p.Hk * splits;
    if (f.rows <= 16)
        return dp == 32 ? launch<T, 32, 1>(f, ctas, stream)
             : dp == 64 ? launch<T, 64, 1>(f, ctas, stream) : launch<T, 128, 1>(f, ctas, stream);
    return dp == 32 ? launch<T, 32, 2>(f, ctas, stream)
         : dp == 64 ? launch<T, 64, 2>(f, ctas, stream) : launch<T, 128, 2>(f, ctas, stream);
}

}  // namespace

// Shared heads read their keys once in this form, and few items are split into
// shares without a wide tile's start.  Neither: the tiles of attention_forward.cu.
// fp16, this form and those tiles:
//   64 x 8 key heads of 64, 1024 keys: one token of a head 40 us and 30, two heads 40 and 51,
//   four heads 41 and 95; 512 x 8 of 32, 200 keys: 93 and 64, two heads 97 and 122
//   8 x 8 key heads of 64, 8192 keys, one token 32 us and 36; 1 x 8, 16384 keys 24 and 34
bool token_form(const ww_attention_t& p, int sms) noexcept
{
    return i64(p.Hq / p.Hk) * p.Lq <= 32 && (p.Hq > p.Hk || i64(p.B) * p.Hk <= sms);
}

int token_splits(const ww_attention_t& p, int sms) noexcept
{
    const int keys = tile_keys(p.D <= 32 ? 32 : p.D <= 64 ? 64 : 128);
    const int64_t ctas = i64(p.B) * p.Hk, tiles = (p.Lk + keys - 1) / keys;
    if (ctas <= 0 || ctas >= sms) return 1;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({sms / ctas, tiles / kWarps, 128})));
}

int attention_token_launch(const ww_attention_t& p, int splits, float* part_o, float* part_lse,
                           cudaStream_t stream) noexcept
{
    return p.dtype == WW_DTYPE_HALF ? tokens<__half>(p, splits, part_o, part_lse, stream)
                                    : tokens<__nv_bfloat16>(p, splits, part_o, part_lse, stream);
}

}  // namespace ww
