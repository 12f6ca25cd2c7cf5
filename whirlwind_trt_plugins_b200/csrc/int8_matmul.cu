// int8_matmul.cu -- products in 8-bit integers with a scale for each token and
// each channel, and the 8-bit form of 16- or 32-bit activations in front of them.
//
//   out[m, n] = xs[m] ws[n] sum_k xq[m, k] wq[n, k] + bias[n]
//
// The sums are whole numbers in 32 bits, exact (K < 2^17), so that neither tiles nor
// shares of K change a result; (sum xs) ws + bias in fp32, one rounding to the output's type.
//
// Tiles: tcgen05 kind::i8, accumulators in TMEM, operands by TMA in swizzled rows
// of 128 bytes.  One producer warp, one warp that issues, 16 (8 for narrow tiles) that
// write out: each takes 32 rows and 32 or 64 columns of a tile, from TMEM through shared memory to a TMA
// store, while the next tile's products run into the other half of TMEM.
// Blocks are persistent; tiles go in bands of rows so that operands are read from L2.
// Where the tokens do not fill a tile only their rows are loaded, and the ring has more stages.
// Large products take two SMs for a 256 x 256 tile (cta_group::2): each holds half
// the rows and half the channels and reads each operand once.
// Up to 8 tokens: the weights' bytes are the bound.  One round of blocks shares the
// channels; a warp's load is 512 bytes of a channel, so that a lane's 16 bytes of the
// tokens stay in registers over all channels; dp4a, and eight integer sums at a time joined
// over the warp.  The weights' loads are under way before the tokens have been brought to
// 8 bits.
//
// Measured, tokens given in 8 bits: 8192^3 329 us (3340 Tera-operations a second, the rate of kind::i8);
// 469248 x 256 x 768 149 us, 841 MB, most of them written (5.7 TB/s); 64 x 8192 x 8192 17.5 us and 128 x 1024 x 131072 31, HBM and the
// start; 16 x 4096 x 4096 9.2 us, 150 ns a block of K of a single round.  One token: 4096 x 4096 7.2 us with
// its 8-bit form, 4096 x 131072 85 us (6.3 TB/s).
#include "rows.cuh"
#include "tensor_map.cuh"
#include "umma.cuh"

#include <algorithm>

namespace ww {

int quantise_rows(const ww_layer_norm_t& p, const char* name, void* stream) noexcept;  // layer_norm.cu

namespace {

constexpr int kBlockK = 128;  // bytes of a row of a stage
constexpr int kTileM = 128;   // rows of an SM's tile

struct MatmulParams {
    CUtensorMap a, b, c;
    const float *xs, *ws;
    const void* bias;
    void* out;
    int32_t M, N, k_blocks;
    int32_t m_tiles, n_tiles, band;
    int32_t behind;  // the operands are written by the launch before
    int32_t stored;  // the output is stored by TMA
    int32_t a_bytes, block, stages;  // bytes of a block of K: of the tokens, in all; stages of the ring
    int* err;
};

// U: blocks of K of a stage.  A stage costs its two barriers (waits, arrivals) whatever it holds, 150 ns next to the 95 of a
// block's products in tiles of 64 channels: those take 2 at a time, 4 where the tokens leave room for three stages.
// One round of 8 tiles, 16 tokens, K = 8192: 18.1 us with 1, 14.7 with 2, 12.3 with 4.
constexpr int kFewRows = 32;  // of a tile, up to which 4 blocks are a stage
template <int BN, bool PAIR, int U, typename O>
struct Tiles {
    static constexpr int kUnit = U;
    static constexpr int kA = kTileM * kBlockK;
    static constexpr int kB = (PAIR ? BN / 2 : BN) * kBlockK;
    static constexpr int kStage = kA + kB;
    static constexpr int kRing = (BN == 64 ? 6 : sizeof(O) == 2 ? 5 : 4) * kStage;
    static constexpr int kMostStages = 16;  // where the tokens do not fill a tile
    static constexpr int kWarps = BN == 64 ? 8 : 16;  // that write out
    static constexpr int kThreads = 128 + 32 * kWarps;
    static constexpr int kColumns = BN * 4 / kWarps;  // of such a warp
    static constexpr int kChunk = 32;                      // of them staged at a time
    static constexpr int kChunkRow = kChunk * sizeof(O);   // 64 or 128 bytes
    static constexpr int kStaging = 32 * kChunkRow;
    static constexpr int kBuffers = BN == 64 ? 2 : 1;  // of a warp
    static constexpr int kOut = kRing;
    static constexpr int kScales = kOut + kWarps * kBuffers * kStaging;
    static constexpr int kBar = kScales + kWarps * kColumns * 8;
    static constexpr int kBytes = kBar + (2 * kMostStages + 4) * 8 + 16 + 1024;
    static constexpr int kTmem = 2 * BN;
    static_assert(kBytes <= kMaxShared, "shared memory");
    static_assert(kRing + kA <= kBytes, "products may read a whole tile from the last stage on");
    static_assert(kRing >= 2 * U * (U == 4 ? kFewRows * kBlockK + kB : kStage), "two stages");
};

// ---- instructions of a pair of SMs ----

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// Address of `saddr` in the shared memory of block `rank` of the cluster.
__device__ __forceinline__ uint32_t in_block(uint32_t saddr, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" : : : "memory");
}

// Tells the other SM that this one's tensor memory has been read.  Relaxed: the reads are in
// registers (tcgen05.wait::ld), nothing written here is read there; a release would wait
// for the stores to memory under way (1700 clocks of 5000 a tile).
__device__ __forceinline__ void arrive_cluster(uint32_t bar)
{
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" : : "r"(bar) : "memory");
}

template <bool PAIR>
__device__ __forceinline__ void load_tile(uint32_t dst, const void* map, int x, int y, uint32_t bar)
{
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                     "[%0], [%1, {%2, %3}], [%4];\n"
                     : : "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                     "[%0], [%1, {%2, %3}], [%4];\n"
                     : : "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

__device__ __forceinline__ void store_tile(const void* map, uint32_t src, int x, int y)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];\n"
                 : : "l"(map), "r"(x), "r"(y), "r"(src) : "memory");
}

__device__ __forceinline__ void commit_store() { asm volatile("cp.async.bulk.commit_group;\n" : : : "memory"); }

template <bool PAIR>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
                     : : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
                     : : "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

// Arrive on the barrier (of both SMs) when the products issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar)
{
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n"
                     : : "r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
    else
        umma::mma_commit(bar);
}

template <bool PAIR>
__device__ __forceinline__ void tmem_get(uint32_t to, uint32_t columns)
{
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" : : "r"(to), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" : : : "memory");
    } else {
        umma::tmem_alloc(to, columns);
    }
}

template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t at, uint32_t columns)
{
    if constexpr (PAIR)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" : : "r"(at), "r"(columns) : "memory");
    else
        umma::tmem_dealloc(at, columns);
}

// Bounded wait of a warp, the same answer in every lane.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity)
{
    return __all_sync(~0u, umma::mbar_poll(bar, parity));
}

// Instruction descriptor of kind::i8: signed operands, K-major both, 32-bit sums.
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N)
{
    return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

// Tile t: bands of `band` tiles of rows, the rows of a band first.
__device__ __forceinline__ void tile_at(const MatmulParams& p, int t, int& m, int& n)
{
    const int whole = p.band * p.n_tiles, first = t / whole * p.band, rows = min(p.band, p.m_tiles - first);
    t %= whole;
    m = first + t % rows;
    n = t / rows;
}

template <typename O>
__device__ __forceinline__ void pack_row(const Pair (&v)[4], uint32_t to0, uint32_t to1)
{
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) unpair(v[i], f[2 * i], f[2 * i + 1]);
    if constexpr (sizeof(O) == 4) {
        umma::st_shared_v4(to0, __float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        umma::st_shared_v4(to1, __float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
    } else {
        umma::st_shared_v4(to0, pack2<O>(f[0], f[1]), pack2<O>(f[2], f[3]), pack2<O>(f[4], f[5]), pack2<O>(f[6], f[7]));
    }
}

template <int BN, bool PAIR, int U, typename O>
__global__ void __launch_bounds__(Tiles<BN, PAIR, U, O>::kThreads, 1) int8_matmul_kernel(const __grid_constant__ MatmulParams p)
{
    using L = Tiles<BN, PAIR, U, O>;
    const int S = p.stages;
    extern __shared__ uint8_t raw[];
    uint8_t* base = raw + ((1024 - (umma::smem_addr(raw) & 1023)) & 1023);
    const uint32_t sm = umma::smem_addr(base);
    const uint32_t full = sm + L::kBar, empty = full + L::kMostStages * 8, done = empty + L::kMostStages * 8, freed = done + 16, slot = freed + 16;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = PAIR ? cluster_rank() : 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            umma::mbar_init(full + s * 8, 1);
            umma::mbar_init(empty + s * 8, 1);
        }
        for (int i = 0; i < 2; ++i) {
            umma::mbar_init(done + i * 8, 1);
            umma::mbar_init(freed + i * 8, L::kWarps * (PAIR ? 2 : 1));
        }
        umma::mbar_fence_init();
        umma::tma_prefetch_desc(&p.a);
        umma::tma_prefetch_desc(&p.b);
    }
    if (warp == 2) tmem_get<PAIR>(slot, L::kTmem);
    umma::fence_before_sync();
    __syncthreads();
    if (PAIR) cluster_sync();
    umma::fence_after_sync();
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(slot) : "memory");
    if (p.behind) wait_for_launches_before();
    const int tiles = p.m_tiles * p.n_tiles, step = PAIR ? gridDim.x / 2 : gridDim.x, start = PAIR ? blockIdx.x / 2 : blockIdx.x;
    bool ok = true;

    if (warp == 0 && umma::elect_one()) {  // loads
        int s = 0;
        uint32_t parity = 1, to = sm;
        for (int t = start; t < tiles && ok; t += step) {
            int m, n;
            tile_at(p, t, m, n);
            const int row = (m * (PAIR ? 2 : 1) + static_cast<int>(rank)) * kTileM, channel = n * BN + static_cast<int>(rank) * (BN / 2);
            for (int k = 0; k < p.k_blocks && ok; k += L::kUnit) {  // blocks beyond the last are zeros
                ok = umma::mbar_poll(empty + s * 8, parity);
                if (ok) {
                    const uint32_t bar = PAIR ? in_block(full + s * 8, 0) : full + s * 8;
                    if (rank == 0) umma::mbar_arrive_expect_tx(full + s * 8, L::kUnit * p.block * (PAIR ? 2 : 1));
#pragma unroll
                    for (int u = 0; u < L::kUnit; ++u) {
                        load_tile<PAIR>(to + u * p.block, &p.a, (k + u) * kBlockK, row, bar);
                        load_tile<PAIR>(to + u * p.block + p.a_bytes, &p.b, (k + u) * kBlockK, channel, bar);
                    }
                }
                to += L::kUnit * p.block;
                if (++s == S) {
                    s = 0;
                    to = sm;
                    parity ^= 1;
                }
            }
        }
    } else if (warp == 1 && rank == 0 && umma::elect_one()) {  // products
        constexpr uint32_t idesc = idesc_i8(PAIR ? 2 * kTileM : kTileM, BN);
        const uint64_t a0 = umma::smem_desc_swizzled<128>(sm, 1024), b0 = umma::smem_desc_swizzled<128>(sm + p.a_bytes, 1024);
        int s = 0, i = 0, at = 0;
        uint32_t parity = 0;
        for (int t = start; t < tiles && ok; t += step, ++i) {
            ok = umma::mbar_poll(freed + (i & 1) * 8, ((i >> 1) & 1) ^ 1);
            umma::fence_after_sync();
            const uint32_t d = tmem + (i & 1) * BN;
            for (int k = 0; k < p.k_blocks && ok; k += L::kUnit) {
                ok = umma::mbar_poll(full + s * 8, parity);
                umma::fence_after_sync();
                if (ok) {
#pragma unroll
                    for (int u = 0; u < L::kUnit; ++u) {
                        const uint64_t a = umma::desc_advance(a0, at + u * p.block), b = umma::desc_advance(b0, at + u * p.block);
#pragma unroll
                        for (int j = 0; j < kBlockK / 32; ++j)
                            mma_i8<PAIR>(d, umma::desc_advance(a, j * 32), umma::desc_advance(b, j * 32), idesc, k > 0 || u > 0 || j > 0);
                    }
                    commit<PAIR>(empty + s * 8);
                    if (k + L::kUnit >= p.k_blocks) commit<PAIR>(done + (i & 1) * 8);
                }
                at += L::kUnit * p.block;
                if (++s == S) {
                    s = at = 0;
                    parity ^= 1;
                }
            }
        }
    } else if (warp >= 4) {  // results
        const int quarter = warp % 4, part = warp / 4 - 1, w = warp - 4;
        constexpr int kMine = L::kColumns / 32;  // columns of a lane whose scales it brings
        const uint32_t bar = PAIR ? in_block(freed, 0) : freed;
        float* scales = reinterpret_cast<float*>(base + L::kScales) + w * 2 * L::kColumns;  // [columns] of ws, of the bias
        int row0, column0, buffer = 0;
        float ws[kMine], xs;
        O bs[kMine];  // converted when they are used: the loads stay under way
        const auto ahead = [&](int t) {
            int m, n;
            tile_at(p, t, m, n);
            row0 = (m * (PAIR ? 2 : 1) + static_cast<int>(rank)) * kTileM + quarter * 32;
            column0 = n * BN + part * L::kColumns;
#pragma unroll
            for (int c = 0; c < kMine; ++c) {
                const int x = column0 + c * 32 + lane;
                ws[c] = x < p.N ? __ldg(p.ws + x) : 0.0f;
                bs[c] = from_float<O>(0.0f);
                if (x < p.N && p.bias != nullptr) bs[c] = static_cast<const O*>(p.bias)[x];
            }
            xs = row0 + lane < p.M ? __ldg(p.xs + row0 + lane) : 0.0f;
        };
        if (start < tiles) ahead(start);
        int i = 0;
        for (int t = start; t < tiles && ok; t += step, ++i) {
            __syncwarp();  // the scales before have been read
#pragma unroll
            for (int c = 0; c < kMine; ++c) {
                scales[c * 32 + lane] = ws[c];
                scales[L::kColumns + c * 32 + lane] = to_float(bs[c]);
            }
            __syncwarp();
            const Pair x2 = pair(xs, xs);
            const int my_row0 = row0, my_column0 = column0;
            if (t + step < tiles) ahead(t + step);
            ok = wait(done + (i & 1) * 8, (i >> 1) & 1);
            umma::fence_after_sync();
            if (!ok) break;
            const uint32_t from = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (i & 1) * BN + part * L::kColumns;
#pragma unroll 1
            for (int c = 0; c < L::kColumns; c += L::kChunk, buffer = L::kBuffers - 1 - buffer) {
                const int my_out = L::kOut + (w * L::kBuffers + buffer) * L::kStaging;
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;\n" : : "n"(L::kBuffers - 1) : "memory");
                __syncwarp();
                uint32_t v[32];
                umma::tmem_ld32(from + c, v);
                umma::tmem_wait_ld32(v);
                if (c + L::kChunk == L::kColumns) {  // TMEM has been read
                    umma::fence_before_sync();
                    __syncwarp();
                    if (lane == 0) {
                        if (PAIR) arrive_cluster(bar + (i & 1) * 8);
                        else umma::mbar_arrive(bar + (i & 1) * 8);
                    }
                }
#pragma unroll
                for (int j = 0; j < L::kChunk; j += 8) {
                    Pair f[4];
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        const float4 m = *reinterpret_cast<const float4*>(scales + c + j + 4 * z);
                        const float4 a = *reinterpret_cast<const float4*>(scales + L::kColumns + c + j + 4 * z);
                        const uint32_t* q = v + j + 4 * z;
                        f[2 * z] = fma2(mul2(pair(__int2float_rn(q[0]), __int2float_rn(q[1])), x2), pair(m.x, m.y), pair(a.x, a.y));
                        f[2 * z + 1] = fma2(mul2(pair(__int2float_rn(q[2]), __int2float_rn(q[3])), x2), pair(m.z, m.w), pair(a.z, a.w));
                    }
                    // 16-byte piece of the row, swizzled as the TMA store reads it
                    const int piece = j * static_cast<int>(sizeof(O)) / 16;
                    const int turn = L::kChunkRow == 128 ? lane & 7 : (lane >> 1) & 3;
                    const uint32_t at = sm + my_out + lane * L::kChunkRow;
                    pack_row<O>(f, at + ((piece ^ turn) << 4), at + (((piece + 1) ^ turn) << 4));
                }
                const int x = my_column0 + c;
                if (p.stored) {
                    umma::fence_proxy_async_smem();
                    __syncwarp();
                    // Of two buffers one is free when all groups but the last have been read, which has to be the other one's: a
                    // chunk that lies outside the output is an empty group.
                    const bool within = x < p.N && my_row0 < p.M;
                    if (lane == 0 && within) store_tile(&p.c, sm + my_out, x, my_row0);
                    if (lane == 0 && (within || L::kBuffers > 1)) commit_store();
                } else {  // rows that do not start on 16 bytes
                    __syncwarp();
                    for (int r = 0; r < 32 && my_row0 + r < p.M; ++r) {
                        const int turn = L::kChunkRow == 128 ? r & 7 : (r >> 1) & 3;
                        const int byte = lane * static_cast<int>(sizeof(O));
                        const uint8_t* from_row = base + my_out + r * L::kChunkRow + (((byte >> 4) ^ turn) << 4) + (byte & 15);
                        if (x + lane < p.N)
                            static_cast<O*>(p.out)[static_cast<int64_t>(my_row0 + r) * p.N + x + lane] = *reinterpret_cast<const O*>(from_row);
                    }
                    __syncwarp();
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;\n" : : : "memory");
    }
    if (!ok && (warp < 4 || lane == 0)) record_device_error(p.err, kErrMbarTimeout | 0x50);
    __syncwarp();
    umma::fence_before_sync();
    __syncthreads();
    if (PAIR) cluster_sync();  // until neither SM's barriers or TMEM are used by the other
    umma::fence_after_sync();
    if (warp == 2) tmem_free<PAIR>(tmem, L::kTmem);
}

// ---- few tokens ----

constexpr int kFewTokens = 8;
constexpr int kFewWarps = 16;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kSlice = 512;             // bytes of K of a warp's load
constexpr int kFewShared = 160 * 1024;  // bytes of the tokens in 8 bits
constexpr int kFewChannels = 1 << 18;   // whose sums fit beside them
constexpr int kFewAhead = 8;            // loads that a warp has under way

struct FewParams {
    const void* x;  // activations, or
    const int8_t* xq;
    const float *xs, *ws;
    const int8_t* wq;
    const void* bias;
    void* out;
    int64_t x_stride, xq_stride, w_stride;
    int32_t M, K, N, pitch;  // pitch: bytes between the tokens in shared memory
    int32_t channels;        // of a block
    int32_t x_pieces;        // x can be read 16 bytes at a time
    int32_t behind;          // xq is written by the launch before
};

// 16 bytes of a row at k < K; what lies beyond K is 0.
__device__ __forceinline__ uint4 load_row(const int8_t* row, int k, int K)
{
    uint4 u = __ldg(reinterpret_cast<const uint4*>(row + k));
    const auto keep = [&](uint32_t& w, int at) {  // the word's bytes before K
        const int n = K - k - at;
        if (n < 4) w = n <= 0 ? 0 : w & (0xffffffffu >> (32 - 8 * n));
    };
    if (k + 16 > K) {
        keep(u.x, 0);
        keep(u.y, 4);
        keep(u.z, 8);
        keep(u.w, 12);
    }
    return u;
}

template <typename O, int TOKENS>
__global__ void __launch_bounds__(kFewThreads, 1) int8_few_kernel(const __grid_constant__ FewParams p)
{
    constexpr int kAhead = kFewAhead;
    extern __shared__ __align__(16) uint8_t tokens[];  // [M][pitch], then the sums [channels][tokens], then
    int* sums = reinterpret_cast<int*>(tokens + p.M * p.pitch);
    float* scale = reinterpret_cast<float*>(sums + p.channels * TOKENS);
    uint32_t* top = reinterpret_cast<uint32_t*>(scale + TOKENS);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int n0 = blockIdx.x * p.channels, channels = min(p.channels, p.N - n0);
    const int slices = (p.K + kSlice - 1) / kSlice, end = slices * kSlice;
    // This warp's rows: [row0, channels) in steps of `by`, of slices slice0, slice0 + 16, ..., kAhead
    // rows (places beyond the channels included) at a time.  The first loads are under way before
    // the tokens are there.  Bytes beyond K meet zeros of the tokens.
    const int by = slices < kFewWarps ? kFewWarps / slices : 1, row0 = slices < kFewWarps ? warp / slices : 0;
    const int slice0 = slices < kFewWarps ? warp % slices : warp;
    const int turns = row0 < by && row0 < channels ? (channels - row0 + by * kAhead - 1) / (by * kAhead) : 0;
    const int count = slice0 < slices ? turns * ((slices - slice0 + kFewWarps - 1) / kFewWarps) : 0;
    uint4 w[kAhead];
    const auto load = [&](int i, int slice, int r0) {  // row i of those from r0 on
        const int row = r0 + i * by, k = slice * kSlice + lane * 16;
        w[i] = make_uint4(0, 0, 0, 0);
        if (row < channels && k < p.K) w[i] = __ldg(reinterpret_cast<const uint4*>(p.wq + (n0 + row) * p.w_stride + k));
    };
    if (count > 0)
#pragma unroll
        for (int i = 0; i < kAhead; ++i) load(i, slice0, row0);
    for (int e = threadIdx.x; e < p.channels * TOKENS; e += kFewThreads) sums[e] = 0;
    if (threadIdx.x < TOKENS) top[threadIdx.x] = 0;
    if (p.behind) wait_for_launches_before();
    constexpr int kBatch = TOKENS < 4 ? TOKENS : 4;  // tokens whose loads are under way together
    if (p.x != nullptr) {
        // the tokens in 8 bits: each token's largest magnitude (its bits order like the
        // values, NaN above all), then its whole numbers, from L1 again
        constexpr int V = 16 / static_cast<int>(sizeof(O));
        __syncthreads();
        for (int m0 = 0; m0 < p.M; m0 += kBatch) {
            float a[kBatch] = {};
            if (p.x_pieces) {
                for (int k = threadIdx.x * V; k < p.K; k += kFewThreads * V) {
                    Piece<O, V> r[kBatch][1];
                    Pair f[V / 2];
#pragma unroll
                    for (int j = 0; j < kBatch; ++j)
                        if (m0 + j < p.M) r[j][0].load(static_cast<const O*>(p.x) + (m0 + j) * p.x_stride + k);
                        else r[j][0].clear();
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) {
                        values_of<O, V, 1>(r[j], f);
                        a[j] = max_nan(a[j], largest(f));
                    }
                }
            } else {
#pragma unroll 4
                for (int k = threadIdx.x; k < p.K; k += kFewThreads)
#pragma unroll
                    for (int j = 0; j < kBatch; ++j)
                        if (m0 + j < p.M) a[j] = max_nan(a[j], fabsf(to_float(static_cast<const O*>(p.x)[(m0 + j) * p.x_stride + k])));
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const uint32_t u = __reduce_max_sync(~0u, __float_as_uint(a[j]) & 0x7fffffffu);
                if (lane == 0 && m0 + j < p.M) atomicMax(top + m0 + j, u);
            }
        }
        __syncthreads();
        if (threadIdx.x < p.M) scale[threadIdx.x] = row_scale(__uint_as_float(top[threadIdx.x])).scale;
        for (int m0 = 0; m0 < p.M; m0 += kBatch) {
            float inv[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j) inv[j] = row_scale(__uint_as_float(top[min(m0 + j, p.M - 1)])).inv;
            int8_t* to = reinterpret_cast<int8_t*>(tokens) + m0 * p.pitch;
            if (p.x_pieces) {
                for (int k = threadIdx.x * V; k < end; k += kFewThreads * V) {
                    Piece<O, V> r[kBatch][1];
                    Pair f[V / 2];
#pragma unroll
                    for (int j = 0; j < kBatch; ++j)
                        if (m0 + j < p.M && k < p.K) r[j][0].load(static_cast<const O*>(p.x) + (m0 + j) * p.x_stride + k);
                        else r[j][0].clear();
#pragma unroll
                    for (int j = 0; j < kBatch; ++j) {
                        if (m0 + j >= p.M) continue;
                        values_of<O, V, 1>(r[j], f);
                        store_piece_int8<V>(to + j * p.pitch + k, f, inv[j], 0);
                    }
                }
            } else {
#pragma unroll 4
                for (int k = threadIdx.x; k < end; k += kFewThreads)
#pragma unroll
                    for (int j = 0; j < kBatch; ++j)
                        if (m0 + j < p.M)
                            to[j * p.pitch + k] = k < p.K ? quantise(to_float(static_cast<const O*>(p.x)[(m0 + j) * p.x_stride + k]), inv[j]) : 0;
            }
        }
    } else {
        if (threadIdx.x < p.M) scale[threadIdx.x] = __ldg(p.xs + threadIdx.x);
        for (int m0 = 0; m0 < p.M; m0 += kBatch)
            for (int k = threadIdx.x * 16; k < end; k += kFewThreads * 16) {
                uint4 u[kBatch];
#pragma unroll
                for (int j = 0; j < kBatch; ++j)
                    u[j] = m0 + j < p.M && k < p.K ? load_row(p.xq + (m0 + j) * p.xq_stride, k, p.K) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < kBatch; ++j)
                    if (m0 + j < p.M) *reinterpret_cast<uint4*>(tokens + (m0 + j) * p.pitch + k) = u[j];
            }
    }
    __syncthreads();
    uint4 x[TOKENS];
    constexpr int kAtOnce = 8 / TOKENS;  // rows whose eight sums are joined over the warp together
    int slice = slice0, r0 = row0;
    for (int n = 0; n < count; ++n) {
        if (r0 == row0)
#pragma unroll
            for (int m = 0; m < TOKENS; ++m)
                x[m] = m < p.M ? *reinterpret_cast<const uint4*>(tokens + m * p.pitch + slice * kSlice + lane * 16) : make_uint4(0, 0, 0, 0);
        const bool wraps = r0 + by * kAhead >= channels;
        const int next_slice = wraps ? slice + kFewWarps : slice, next_r0 = wraps ? row0 : r0 + by * kAhead;
#pragma unroll
        for (int i = 0; i < kAhead; i += kAtOnce) {
            int v[8];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const uint4 a = w[i + j];
                if (n + 1 < count) load(i + j, next_slice, next_r0);
#pragma unroll
                for (int m = 0; m < TOKENS; ++m) {
                    int d = __dp4a(static_cast<int>(a.x), static_cast<int>(x[m].x), 0);
                    d = __dp4a(static_cast<int>(a.y), static_cast<int>(x[m].y), d);
                    d = __dp4a(static_cast<int>(a.z), static_cast<int>(x[m].z), d);
                    v[j * TOKENS + m] = __dp4a(static_cast<int>(a.w), static_cast<int>(x[m].w), d);
                }
            }
            // eight sums over 32 lanes: half of them change sides at each of three steps
#pragma unroll
            for (int half = 4; half > 0; half /= 2) {
                const bool upper = lane & (half * 4);
#pragma unroll
                for (int j = 0; j < half; ++j) {
                    const int give = upper ? v[j] : v[j + half];
                    v[j] = (upper ? v[j + half] : v[j]) + __shfl_xor_sync(~0u, give, half * 4);
                }
            }
            v[0] += __shfl_xor_sync(~0u, v[0], 2);
            v[0] += __shfl_xor_sync(~0u, v[0], 1);
            // value lane / 4; the slices' sums are whole numbers, so that their order does not matter
            const int row = r0 + (i + lane / 4 / TOKENS) * by, m = lane / 4 % TOKENS;
            if (lane % 4 == 0 && row < channels && m < p.M) atomicAdd(sums + row * TOKENS + m, v[0]);
        }
        slice = next_slice;
        r0 = next_r0;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.M * channels; e += kFewThreads) {
        const int m = e / channels, c = e - m * channels;
        const float b = p.bias == nullptr ? 0.0f : to_float(static_cast<const O*>(p.bias)[n0 + c]);
        static_cast<O*>(p.out)[static_cast<int64_t>(m) * p.N + n0 + c] =
            from_float<O>(fmaf(__int2float_rn(sums[c * TOKENS + m]) * scale[m], __ldg(p.ws + n0 + c), b));
    }
}

// ---- host ----

int pitch_of(int k) noexcept { return (k + 15) / 16 * 16; }

// Bytes between tokens in shared memory: whole slices.
int few_pitch(int k) noexcept { return (k + kSlice - 1) / kSlice * kSlice; }

// Few tokens that every block brings to 8 bits by itself; more are brought there once.  4096 values
// a token against 4096 channels, in the blocks and before them: one token 7.2 us and 8.9, 4
// tokens 9.2 and 11.2, 8 tokens 14.9 and 12.1.
bool few_alone(const ww_int8_matmul_t& p) noexcept { return p.x == nullptr || i64(p.M) * p.K <= 16384; }

template <int BN, bool PAIR, int U, typename O>
int launch_tiles(MatmulParams& f, int tiles, int sms, cudaStream_t stream) noexcept
{
    using L = Tiles<BN, PAIR, U, O>;
    const auto kernel = int8_matmul_kernel<BN, PAIR, U, O>;
    static std::atomic<uint64_t> raised{0};
    if (!allow_shared_memory(reinterpret_cast<const void*>(kernel), raised)) return launch_status("int8_matmul");
    cudaLaunchAttribute attr[2]{};
    cudaLaunchConfig_t cfg{};
    if (f.behind) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (PAIR) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = 2;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    cfg.gridDim = PAIR ? 2 * std::min(tiles, sms / 2) : std::min(tiles, sms);
    cfg.blockDim = L::kThreads;
    cfg.dynamicSmemBytes = L::kBytes;
    cfg.stream = stream;
    cfg.attrs = attr;
    cudaLaunchKernelEx(&cfg, kernel, f);
    return launch_status("int8_matmul");
}

// Channels of a tile: 64 or 128 on an SM, 256 x 256 on a pair; the form whose rounds end
// soonest, by clocks of a block of K and of a round's start and end (fitted to the times below).
// us with 64, 128, 256 channels: 16 x 4096 x 14336 15.5, 14.6, 16.9; 64 x 8192 x 8192 17.3, 21.5, 24.9; 300 x 4096 x 4096
// 16.6, 13.3, 15.6; 1777 x 1000 x 1111 10.8, 9.4, 12.5; 1024 x 4096 x 4096 29.9, 23.3, 17.1; 2048^3 17.3, 14.3, 11.9;
// 19200 x 320 x 320 10.0, 9.0, 10.3; 500 x 2048 x 700 8.2, 9.8, 13.4; 469248 x 256 x 768 -, 184, 149.
struct TileForm {
    int channels;
    int64_t clocks;
};

TileForm tile_form(const ww_int8_matmul_t& p, int sms) noexcept
{
    const int64_t k_blocks = (p.K + kBlockK - 1) / kBlockK;
    const auto time = [&](int rows, int channels, int slots, int block, int round) {
        const int64_t tiles = ((i64(p.M) + rows - 1) / rows) * ((i64(p.N) + channels - 1) / channels);
        return (tiles + slots - 1) / slots * (k_blocks * block + round);
    };
    const int64_t narrow = time(kTileM, 64, sms, p.M <= kFewRows ? 290 : 360, 800), one = time(kTileM, 128, sms, 540, 1000),
                  two = time(2 * kTileM, 256, sms / 2, 690, 2400);
    if (two <= narrow && two <= one) return {256, two};
    return one <= narrow ? TileForm{128, one} : TileForm{64, narrow};
}

// Whether up to 8 tokens take the form of their own: one always does; more where it is expected to end before the tiles
// do (dp4a costs 0.2 or 0.3 ps a weight with 4 or 8 tokens), the 8-bit form of the tokens in a launch before them included.
// us in their own form and in tiles, 4 tokens: 4096 x 4096 8.1 and 9.3, 8192 x 8192 17.6 and 15.8, 1024 x 131072 32 and 25;
// 8 tokens: 4096 x 512 6.3 and 7.8, 1024 x 1024 6.1 and 4.6, 4096 x 4096 10.6 and 9.4, 8192 x 8192 24 and 16.  One: 4096 x 131072 85 and 138.
bool few_form(const ww_int8_matmul_t& p, int sms) noexcept
{
    if (p.M > kFewTokens || i64(p.M) * few_pitch(p.K) > kFewShared || p.N > kFewChannels) return false;
    if (p.M == 1) return true;
    const int64_t own = (p.M <= 4 ? 700'000 : 1'900'000) + i64(p.N) * p.K * (p.M <= 4 ? 200 : 300) / 1000;   // ps
    const int64_t tiles = tile_form(p, sms).clocks * 526 + (p.x != nullptr && few_alone(p) ? 1'700'000 : 0);  // at 1.9 GHz
    return own <= tiles;
}

// Rows of a tile of tokens that are loaded: of a tile that the tokens do not fill, only those.
// The products then read on into what lies behind them, in shared memory, for rows that are not written out.
int loaded_rows(int m) noexcept { return std::min(kTileM, (m + 7) / 8 * 8); }

template <int BN, bool PAIR, int U, typename O>
int run_tiles(const ww_int8_matmul_t& p, bool behind, int sms, int* err, cudaStream_t stream) noexcept
{
    using L = Tiles<BN, PAIR, U, O>;
    MatmulParams f;
    const int a_rows = loaded_rows(p.M);
    f.a_bytes = a_rows * kBlockK;
    f.block = f.a_bytes + L::kB;
    f.stages = std::min(L::kMostStages, L::kRing / (L::kUnit * f.block));
    if (!encode_rows_map(&f.a, WW_DTYPE_INT8, p.x_q, p.M, p.K, p.x_q_stride, kBlockK, a_rows) ||
        !encode_rows_map(&f.b, WW_DTYPE_INT8, p.w_q, p.N, p.K, p.w_stride, kBlockK, PAIR ? BN / 2 : BN))
        return WW_ERR_UNSUPPORTED;
    f.stored = i64(p.N) * static_cast<int>(sizeof(O)) % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
    if (f.stored && !encode_rows_map(&f.c, p.dtype, p.out, p.M, p.N, p.N, L::kChunk, 32)) return WW_ERR_UNSUPPORTED;
    f.xs = p.x_scale;
    f.ws = p.w_scale;
    f.bias = p.bias;
    f.out = p.out;
    f.M = p.M;
    f.N = p.N;
    f.k_blocks = (p.K + kBlockK - 1) / kBlockK;
    const int rows = PAIR ? 2 * kTileM : kTileM;
    f.m_tiles = (p.M + rows - 1) / rows;
    f.n_tiles = (p.N + BN - 1) / BN;
    f.band = 8;
    f.behind = behind;
    f.err = err;
    const int64_t tiles = i64(f.m_tiles) * f.n_tiles;
    if (tiles > INT_MAX / 2) return WW_ERR_UNSUPPORTED;
    return launch_tiles<BN, PAIR, U, O>(f, static_cast<int>(tiles), sms, stream);
}

// Channels of a block in the form for few tokens: one round of blocks, at least 4 channels each.
int few_channels(int n, int sms) noexcept { return std::max(4, (n + sms - 1) / sms); }

template <typename O>
int few(const ww_int8_matmul_t& p, bool behind, int sms, cudaStream_t stream) noexcept
{
    FewParams f{p.x, p.x_q, p.x_scale, p.w_scale, p.w_q, p.bias, p.out, p.x_stride, p.x_q_stride, p.w_stride, p.M, p.K, p.N, few_pitch(p.K),
                few_channels(p.N, sms), 0, behind};
    constexpr int V = 16 / static_cast<int>(sizeof(O));
    f.x_pieces = p.K % V == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && (p.M == 1 || p.x_stride % V == 0);
    const int form = p.M == 1 ? 0 : p.M <= 4 ? 1 : 2, tokens = form == 0 ? 1 : 4 * form;
    const auto kernel = form == 0 ? int8_few_kernel<O, 1> : form == 1 ? int8_few_kernel<O, 4> : int8_few_kernel<O, 8>;
    static std::atomic<uint64_t> raised[3];
    if (!allow_shared_memory(reinterpret_cast<const void*>(kernel), raised[form])) return launch_status("int8_matmul");
    const int bytes = p.M * f.pitch + f.channels * tokens * 4 + tokens * 8;
    const dim3 grid((p.N + f.channels - 1) / f.channels);
    if (behind) launch_behind(kernel, grid, dim3(kFewThreads), bytes, stream, f);
    else kernel<<<grid, kFewThreads, bytes, stream>>>(f);
    return launch_status("int8_matmul");
}

template <typename O>
int matmul(const ww_int8_matmul_t& p, int sms, cudaStream_t stream) noexcept
{
    const bool is_few = few_form(p, sms);
    if (is_few && few_alone(p)) return few<O>(p, false, sms, stream);
    ww_int8_matmul_t c = p;
    if (p.x != nullptr) {
        ww_layer_norm_t r{};
        c.x = nullptr;
        c.x_q_stride = r.y_q_stride = pitch_of(p.K);
        c.x_q = r.y_q = static_cast<int8_t*>(p.workspace);
        c.x_scale = r.y_scale = reinterpret_cast<float*>(r.y_q + i64(p.M) * r.y_q_stride);
        r.x = p.x;
        r.x_stride = p.x_stride;
        r.dtype = p.dtype;
        r.rows = p.M;
        r.N = p.K;
        const int st = quantise_rows(r, "int8_matmul", stream);
        if (st != WW_SUCCESS) return st;
    }
    const bool behind = p.x != nullptr;
    if (is_few) return few<O>(c, behind, sms, stream);
    int* err = device_error_slot();
    if (err == nullptr) return WW_ERR_DEVICE;
    switch (tile_form(c, sms).channels) {
    case 256: return run_tiles<256, true, 1, O>(c, behind, sms, err, stream);
    case 128: return run_tiles<128, false, 1, O>(c, behind, sms, err, stream);
    default:
        return loaded_rows(c.M) <= kFewRows ? run_tiles<64, false, 4, O>(c, behind, sms, err, stream)
                                            : run_tiles<64, false, 2, O>(c, behind, sms, err, stream);
    }
}

int check(const ww_int8_matmul_t& p) noexcept
{
    if (p.dtype != WW_DTYPE_HALF && p.dtype != WW_DTYPE_BF16 && p.dtype != WW_DTYPE_FLOAT) return WW_ERR_INVALID_DTYPE;
    if (p.M < 0 || p.N < 0 || p.K <= 0) return WW_ERR_INVALID_SHAPE;
    if (p.K >= (1 << 17)) return WW_ERR_UNSUPPORTED;
    if (p.M == 0 || p.N == 0) return WW_SUCCESS;
    if (p.w_q == nullptr || p.w_scale == nullptr || p.out == nullptr) return WW_ERR_NULL_POINTER;
    if ((p.x == nullptr) == (p.x_q == nullptr) || (p.x_q != nullptr && p.x_scale == nullptr)) return WW_ERR_NULL_POINTER;
    const int bytes = p.dtype == WW_DTYPE_FLOAT ? 4 : 2;
    const auto off = [](const void* q, int by) { return reinterpret_cast<uintptr_t>(q) % by != 0; };
    if (p.w_stride < p.K || (p.x_q != nullptr && p.x_q_stride < p.K && p.M > 1) || (p.x != nullptr && p.x_stride < 0)) return WW_ERR_INVALID_SHAPE;
    if (off(p.w_q, 16) || p.w_stride % 16 != 0 || off(p.x_q, 16) || (p.x_q != nullptr && p.M > 1 && p.x_q_stride % 16 != 0)) return WW_ERR_MISALIGNED;
    if (off(p.x, bytes) || off(p.bias, bytes) || off(p.out, bytes) || off(p.x_scale, 4) || off(p.w_scale, 4)) return WW_ERR_MISALIGNED;
    return WW_SUCCESS;
}

int sm_count() noexcept
{
    DeviceInfo d;
    return current_device_info(&d) == WW_SUCCESS ? d.sm_count : 148;
}

int64_t workspace(const ww_int8_matmul_t& p, int sms) noexcept
{
    if (p.x == nullptr || p.M == 0 || p.N == 0 || (few_form(p, sms) && few_alone(p))) return 0;
    return i64(p.M) * pitch_of(p.K) + i64(p.M) * 4;
}

}  // namespace
}  // namespace ww

extern "C" {

int64_t ww_int8_matmul_workspace(const ww_int8_matmul_t* p)
{
    return p == nullptr || ww::check(*p) != WW_SUCCESS ? 0 : ww::workspace(*p, ww::sm_count());
}

int ww_int8_matmul(const ww_int8_matmul_t* p, void* stream)
{
    if (p == nullptr) return WW_ERR_NULL_POINTER;
    int st = ww::check(*p);
    if (st != WW_SUCCESS || p->M == 0 || p->N == 0) return st;
    const int64_t need = ww::workspace(*p, ww::sm_count());
    if (need > 0) {
        if (p->workspace == nullptr) return WW_ERR_NULL_POINTER;
        if (reinterpret_cast<uintptr_t>(p->workspace) % 16 != 0) return WW_ERR_MISALIGNED;
        if (p->workspace_bytes < need) return WW_ERR_UNSUPPORTED;
    }
    ww::DeviceInfo d;
    if ((st = ww::current_device_info(&d)) != WW_SUCCESS) return st;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return p->dtype == WW_DTYPE_HALF ? ww::matmul<__half>(*p, d.sm_count, s)
         : p->dtype == WW_DTYPE_BF16 ? ww::matmul<__nv_bfloat16>(*p, d.sm_count, s) : ww::matmul<float>(*p, d.sm_count, s);
}

}  // extern "C"
