// layer_norm.cu -- layer norm of token rows, optionally of a residual sum and
// with an 8-bit result, its gradient, and the 8-bit form of rows by itself.
//
//   h = x + r (rounded to its type, as it is kept),  m = mean h,  v = mean (h - m)^2
//   xh = (h - m) rsqrt(v + eps),  y = xh w + b        8 bits: rows.cuh
//
// and backwards, with g = dy w:
//
//   dx = rstd (g - mean g - xh mean(g xh)) + dsum,  dw = sum over rows of dy xh,  db = sum of dy.
//
// Bound: HBM (forward 2 values per element moved, 4 with a residual; backward 3,
// 4 with dsum; about 10 flops).  A row stays in registers between its sums (the
// variance from the deviations; rows far from zero once more, so that a large mean costs no digits), held by a
// group of 4 to 32 lanes or, where a warp's registers do not hold it, by a block;
// loads are 16 bytes a lane where rows start on 16 bytes, else single values, or pairs for long rows.
// Both directions run one resident round of blocks, the next rows' loads under way
// while rows are computed: in registers, or for the gradient of rows of more than a piece a
// lane in rings in shared memory.  In the gradient a lane owns the same columns of all its
// rows, so the weight's and bias's sums stay in registers; they are joined per
// block in shared memory and over blocks by a second kernel, both in a fixed order.
// Rows beyond a block's registers are read again from L2 for each step.
//
// Measured: 469248 rows of 256, fp16, 480 MB: 78 us, 6.1 TB/s; their gradient with dsum,
// bf16, 961 MB: 153 us with the join, 6.3 TB/s.  Gradient of 9001 rows of 1337, fp32, 144 MB:
// 31 us (single loads; pieces of 16 bytes with the rows' ends masked took 52).
// 40000 rows of 1337 in fp16, single loads of 2 bytes: 82 us for 214 MB, instructions.
#include "rows.cuh"
#include "umma.cuh"

#include <algorithm>
#include <cmath>

namespace ww {
namespace {

constexpr int kBlock = 256;
constexpr int kLongBlock = 1024;
// Rows of a group that are under way at a time, and blocks of a resident round, by V (values
// of a piece), pieces a lane and lanes a row.
// Rows of 256 in fp16, forward: 2 rows and 4 blocks 78 us; 3 blocks 85, 4 rows and 2 blocks 81,
// 1 row and 6 blocks 89.  Their gradient with dsum, bf16: 2 rows and 2 blocks 153 us; 1 row and
// 3 blocks 194.
__host__ __device__ constexpr int rows_at_once(int v, int pieces, int group) { return v > 1 && pieces == 1 && group > 0 ? 2 : 1; }
// Three pieces a lane, 80000 rows of 640: fp16 3 blocks (which spill) 49.7 us and 2 45.6, with a residual 89 and 69.6; 100000 of 320 in
// fp32 45 and 52, with a residual 90 and 86.
__host__ __device__ constexpr int forward_blocks(int v, int pieces, bool residual)
{
    return pieces == 1 ? 4 : pieces >= 4 || (pieces == 3 && (v == 8 || residual)) ? 2 : 3;
}
constexpr int kBackwardBlocks = 2;
// Threads of an SM's blocks where a block holds a row.  Gradient of 9001 rows of 1337 in
// fp32 (8 single values a lane): 768 threads 33.5 us; 512 and 1024, which spills, 40 and 38.
// Forward, the same rows: 768 20.9 us, 1024, of which not all are resident, 27.
int forward_threads(bool pieces) { return pieces ? 1024 : 768; }
int backward_threads(int per_lane) { return per_lane == 8 ? 768 : 512; }
// Blocks of a row that the compiler keeps registers for, so that these threads fit.
__host__ __device__ constexpr int row_blocks(int v, int pieces) { return v == 1 && pieces == 8 ? 3 : 1; }

struct NormParams {
    const void *x, *r, *w, *b;
    void *y, *sum;
    int8_t* q;
    float *scale, *mean, *rstd;
    const void *dy, *dsum;
    void* dx;
    float* part;  // [blocks][2][N]
    int64_t xs, rs, qs, gs, ds;  // elements between rows
    int32_t rows, N, norm;
    float eps, inv_n;
    int32_t shift, odd;  // pairs: whether row 0 begins off their grid, whether every other row does
    int32_t stages;      // of a ring
    int* err;
};

// Columns by which the pairs of a group's rows are shifted (rows a step apart begin alike).
template <int V>
__device__ __forceinline__ int pair_shift(const NormParams& p, int64_t row)
{
    return V == 2 ? (p.shift + static_cast<int>(row & 1) * p.odd) & 1 : 0;
}

template <int E>
__device__ __forceinline__ float sum_of(const Pair (&f)[E])
{
    Pair s = f[0];
#pragma unroll
    for (int i = 1; i < E; ++i) s = add2(s, f[i]);
    return both(s);
}

// f less the mean, 0 beyond the row; the sum of their squares.
template <int V, int P, int GROUP, int E>
__device__ __forceinline__ float deviations(Pair (&f)[E], float mean, int n, const Columns<V, P, GROUP>& column)
{
    const Pair nm = pair(-mean, -mean);
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = add2(f[i], nm);
    clear_beyond(f, n, column);
    Pair s = mul2(f[0], f[0]);
#pragma unroll
    for (int i = 1; i < E; ++i) s = fma2(f[i], f[i], s);
    return both(s);
}

// Values of a row and its residual, rounded to their type as they are kept.
template <typename T, int V, int P>
__device__ __forceinline__ void add_residual(Pair (&f)[P * V / 2], const Piece<T, V> (&r)[P])
{
    Pair g[P * V / 2];
    values_of<T, V, P>(r, g);
#pragma unroll
    for (int i = 0; i < P * V / 2; ++i) {
        float a, c;
        unpair(add2(f[i], g[i]), a, c);
        f[i] = pair(to_float(from_float<T>(a)), to_float(from_float<T>(c)));
    }
}

// Whether a row's deviations are so far below its mean (32 times) that the mean's own rounding, 2^-24 of it for each
// addition and for the product with 1 / N, shows in them.
__device__ __forceinline__ bool mean_far(float mean, float variance) { return mean != 0.0f && variance <= mean * mean * 0x1p-10f; }

// The rows of a block.  R rows of a group of lanes at a time, those of the block's next step loaded ahead.  Returns whether one is far
// from its deviations; then the block (GROUP: the warp) goes over its rows again, with FAR, and writes those rows anew: their
// deviations less what these leave of the mean.  Of a row of one value they are a few units in its last place, all equal,
// whose sum is exact, and so is its quotient by N: what remains is 0.  (Done at once, with the next rows under way in
// registers, it costs the other rows 3 to 20 % of their time.)  469248 rows of 256, fp16: 78 us without such rows, 147 with one
// in 1000, 215 where all are.
template <typename T, int V, int P, int GROUP, int R, bool RES, bool FAR>
__device__ __forceinline__ bool norm_rows(const NormParams& p, float (&red)[2][GROUP ? 1 : 3][32 * R])
{
    constexpr int E = P * V / 2;
    constexpr int kGroups = GROUP ? kBlock / (GROUP ? GROUP : 1) : 1;  // rows of a block side by side
    const int lane = GROUP ? threadIdx.x % (GROUP ? GROUP : 1) : threadIdx.x;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kGroups * R);
    int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kGroups * R) + (GROUP ? threadIdx.x / (GROUP ? GROUP : 1) : 0);
    const Columns<V, P, GROUP> column(pair_shift<V>(p, row0));
    const T* xp = static_cast<const T*>(p.x) + row0 * p.xs + column.first;
    const T* rp = RES ? static_cast<const T*>(p.r) + row0 * p.rs + column.first : nullptr;
    // weights: kept where they are few, else from L1 for each row
    constexpr bool kKeep = E <= 4 || V == 2;
    Pair w[E], b[E];
    const auto weights = [&] {
        Piece<T, V> wr[P], br[P];
        load_weights(wr, static_cast<const T*>(p.w), p.N, column);
        load_weights(br, static_cast<const T*>(p.b), p.N, column);
        values_of<T, V, P>(wr, w);
        values_of<T, V, P>(br, b);
        if (p.w == nullptr)
#pragma unroll
            for (int i = 0; i < E; ++i) w[i] = pair(1.0f, 1.0f);
    };
    if (kKeep) weights();
    // what lies beyond a row, and rows beyond the last, are zeros
    Piece<T, V> xr[R][P], rr[RES ? R : 1][P];
    const auto load = [&](int64_t at) {
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const bool is = at + j * kGroups < p.rows;
                load_piece<true>(xr[j][i], xp + j * kGroups * p.xs + i * column.kNext, i, p.N, is, column);
                if constexpr (RES) load_piece<true>(rr[j][i], rp + j * kGroups * p.rs + i * column.kNext, i, p.N, is, column);
            }
    };
    if (!FAR) load(row0);
    int turn = 0;
    bool any_far = false;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * (kGroups * R); base < p.rows; base += step, row0 += step, turn ^= 1) {
        Pair f[R][E];
        bool far[R] = {};
        if (FAR) load(row0);
        const auto real = [&](int j) { return row0 + j * kGroups < p.rows && (!FAR || far[j]); };  // written
#pragma unroll
        for (int j = 0; j < R; ++j) {
            values_of<T, V, P>(xr[j], f[j]);
            if constexpr (RES) add_residual<T, V, P>(f[j], rr[j]);
        }
        if (FAR || base + step < p.rows) {
            xp += step * p.xs;
            if constexpr (RES) rp += step * p.rs;
            if (!FAR) load(row0 + step);
        }
        if (RES && !FAR && p.sum != nullptr)
#pragma unroll
            for (int j = 0; j < R; ++j) {
                T* to = static_cast<T*>(p.sum) + (row0 + j * kGroups) * p.N;
#pragma unroll
                for (int i = 0; i < P; ++i)
                    if (real(j)) store_row_piece(to + column(i), f[j], i, p.N, column);
            }
        if (p.norm) {
            float v[R], mean[R];
#pragma unroll
            for (int j = 0; j < R; ++j) v[j] = sum_of(f[j]);
            row_sums<GROUP>(v, red[turn][0]);
#pragma unroll
            for (int j = 0; j < R; ++j) {
                mean[j] = v[j] * p.inv_n;
                if (!FAR && lane == 0 && p.mean != nullptr && real(j)) p.mean[row0 + j * kGroups] = mean[j];
                v[j] = deviations(f[j], mean[j], p.N, column);
            }
            row_sums<GROUP>(v, red[turn][GROUP ? 0 : 1]);
#pragma unroll
            for (int j = 0; j < R; ++j) {
                far[j] = mean_far(mean[j], v[j] * p.inv_n);
                any_far = any_far || far[j];
            }
            if constexpr (FAR) {
#pragma unroll
                for (int j = 0; j < R; ++j) v[j] = sum_of(f[j]);
                row_sums<GROUP>(v, red[turn][0]);
#pragma unroll
                for (int j = 0; j < R; ++j) {
                    const float c = __fdiv_rn(v[j], static_cast<float>(p.N));
                    if (lane == 0 && p.mean != nullptr && real(j)) p.mean[row0 + j * kGroups] = mean[j] + c;
                    v[j] = deviations(f[j], c, p.N, column);
                }
                row_sums<GROUP>(v, red[turn][GROUP ? 0 : 1]);
            }
            if (!kKeep) weights();
#pragma unroll
            for (int j = 0; j < R; ++j) {
                const float rstd = rsqrtf(fmaf(v[j], p.inv_n, p.eps));
                if (lane == 0 && p.rstd != nullptr && real(j)) p.rstd[row0 + j * kGroups] = rstd;
                const Pair r2 = pair(rstd, rstd);
#pragma unroll
                for (int i = 0; i < E; ++i) f[j][i] = fma2(mul2(f[j][i], r2), w[i], b[i]);
            }
        }
        if (p.q != nullptr) {
            float top[R];
            RowScale k[R];
#pragma unroll
            for (int j = 0; j < R; ++j) top[j] = largest(f[j]);
            row_maxima<GROUP>(top, red[turn][GROUP ? 0 : 2]);
            row_scales<GROUP>(top, k);
#pragma unroll
            for (int j = 0; j < R; ++j) {
                if (!real(j)) continue;
                if (lane == 0) p.scale[row0 + j * kGroups] = k[j].scale;
                int8_t* to = p.q + (row0 + j * kGroups) * p.qs;
#pragma unroll
                for (int i = 0; i < P; ++i)
                    if (column(i) < p.N) store_piece_int8<V>(to + column(i), f[j], k[j].inv, i, column.has(i, 0, p.N), column.has(i, 1, p.N));
            }
        } else {
#pragma unroll
            for (int j = 0; j < R; ++j) {
                T* to = static_cast<T*>(p.y) + (row0 + j * kGroups) * p.N;
#pragma unroll
                for (int i = 0; i < P; ++i)
                    if (real(j)) store_row_piece(to + column(i), f[j], i, p.N, column);
            }
        }
    }
    return __any_sync(~0u, any_far);  // a block's threads have the same sums
}

// At a kernel's end, as a function: nothing is kept across it, and the kernel's registers are its own.
template <typename T, int V, int P, int GROUP, int R, bool RES>
__device__ __noinline__ void far_rows(const NormParams& p, float (&red)[2][GROUP ? 1 : 3][32 * R])
{
    norm_rows<T, V, P, GROUP, R, RES, true>(p, red);
}

template <typename T, int V, int P, int GROUP, int R, bool RES>
__global__ void __launch_bounds__(GROUP ? kBlock : row_threads(V, P, false), GROUP ? forward_blocks(V, P, RES) : row_blocks(V, P))
    layer_norm_kernel(const __grid_constant__ NormParams p)
{
    __shared__ float red[2][GROUP ? 1 : 3][32 * R];
    if (norm_rows<T, V, P, GROUP, R, RES, false>(p, red)) far_rows<T, V, P, GROUP, R, RES>(p, red);
}

// Rows of a residual sum, each held by a block: the rows to come lie in a ring in shared memory, filled by bulk copies.
// us with the next row in registers, and so: 10000 rows of 8192, bf16, 133 and 108 (655 MB, 6.1 TB/s); 10000 of 4096, fp32, 115 and 104.
// Not for rows without a residual (20000 of 4096 61 and 74), nor for those that warps hold (100000 of 1024 141 and 148).
template <typename T, int V>
__global__ void __launch_bounds__(row_threads(V, 2, false), 1) layer_norm_ring_kernel(const __grid_constant__ NormParams p)
{
    constexpr int P = 2, E = P * V / 2;
    extern __shared__ __align__(16) uint8_t ring[];  // stages of a row of x and one of the residual, their barriers, the sums
    const int S = p.stages;
    const bool leader = threadIdx.x == 0;
    const Columns<V, P, 0> column;
    const uint32_t row_bytes = p.N * static_cast<uint32_t>(sizeof(T)), stage = 2 * row_bytes;
    const uint32_t to = umma::smem_addr(ring), bars = to + S * stage;
    float (&red)[2][3][32] = *reinterpret_cast<float (*)[2][3][32]>(ring + static_cast<uint32_t>(S) * (stage + 8));
    int64_t ahead = blockIdx.x;
    const auto fill = [&](int s) {  // the leader
        if (ahead >= p.rows) return;
        umma::mbar_arrive_expect_tx(bars + s * 8, stage);
        umma::bulk_g2s(to + s * stage, static_cast<const T*>(p.x) + ahead * p.xs, row_bytes, bars + s * 8);
        umma::bulk_g2s(to + s * stage + row_bytes, static_cast<const T*>(p.r) + ahead * p.rs, row_bytes, bars + s * 8);
        ahead += gridDim.x;
    };
    if (leader) {
        for (int s = 0; s < S; ++s) umma::mbar_init(bars + s * 8, 1);
        umma::mbar_fence_init();
        for (int s = 0; s < S; ++s) fill(s);
    }
    __syncthreads();  // the barriers are there
    int s = 0, turn = 0;
    uint32_t parity = 0;
    bool ok = true, far = false;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        ok = ok && umma::mbar_poll(bars + s * 8, parity);  // once given up, no wait and no copy follows
        Pair f[E];
        {
            Piece<T, V> x[P], y[P];  // zeros beyond the row
            const T* from = reinterpret_cast<const T*>(ring + static_cast<uint32_t>(s) * stage);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                x[i].clear();
                y[i].clear();
                if (column(i) < p.N) {
                    x[i].load_shared(from + column(i));
                    y[i].load_shared(from + p.N + column(i));
                }
            }
            values_of<T, V, P>(x, f);
            add_residual<T, V, P>(f, y);
        }
        if (p.sum != nullptr)
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (column(i) < p.N) store_piece<T, V>(static_cast<T*>(p.sum) + row * p.N + column(i), f, i);
        const float mean = row_sum<0>(sum_of(f), red[turn][0]) * p.inv_n;
        if (leader) {
            if (ok) fill(s);  // the sum's barrier: the stage has been read
            if (p.mean != nullptr) p.mean[row] = mean;
        }
        const float squares = row_sum<0>(deviations(f, mean, p.N, column), red[turn][1]);
        const float rstd = rsqrtf(fmaf(squares, p.inv_n, p.eps));
        far = far || mean_far(mean, squares * p.inv_n);
        if (leader && p.rstd != nullptr) p.rstd[row] = rstd;
        const Pair r2 = pair(rstd, rstd);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if (column(i) >= p.N) continue;
            Piece<T, V> raw[2][1];
            Pair w[V / 2], b[V / 2];
            raw[1][0].clear();
            if (p.w != nullptr) raw[0][0].load(static_cast<const T*>(p.w) + column(i));
            if (p.b != nullptr) raw[1][0].load(static_cast<const T*>(p.b) + column(i));
            values_of<T, V, 1>(raw[0], w);
            values_of<T, V, 1>(raw[1], b);
#pragma unroll
            for (int e = 0; e < V / 2; ++e) {
                if (p.w == nullptr) w[e] = pair(1.0f, 1.0f);
                f[i * V / 2 + e] = fma2(mul2(f[i * V / 2 + e], r2), w[e], b[e]);
            }
        }
        if (p.q != nullptr) {
            const RowScale k = row_scale(row_max<0>(largest(f), red[turn][2]));
            if (leader) p.scale[row] = k.scale;
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (column(i) < p.N) store_piece_int8<V>(p.q + row * p.qs + column(i), f, k.inv, i);
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (column(i) < p.N) store_piece<T, V>(static_cast<T*>(p.y) + row * p.N + column(i), f, i);
        }
        if (++s == S) {
            s = 0;
            parity ^= 1;
        }
    }
    if (!ok) record_device_error(p.err, kErrMbarTimeout | 0x61);
    if (__any_sync(~0u, far)) far_rows<T, V, P, 0, 1, true>(p, red);  // the same rows, the same lanes
}

// A row of any length by a block, read again for each step, its mean found (FAR: what that lacks as well); returns
// whether it is far from its deviations.
template <typename T, bool FAR>
__device__ __forceinline__ bool norm_long_row(const NormParams& p, float (&red)[3][32])
{
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.xs;
    const T* r = p.r == nullptr ? nullptr : static_cast<const T*>(p.r) + row * p.rs;
    const auto at = [&](int c) { return r == nullptr ? to_float(x[c]) : to_float(from_float<T>(to_float(x[c]) + to_float(r[c]))); };
    float mean = 0.0f, rest = 0.0f, rstd = 1.0f;
    bool far = false;
    if (p.norm) {
        float s = 0.0f;
        for (int c = threadIdx.x; c < p.N; c += kLongBlock) s += at(c);
        mean = row_sum<0>(s, red[0]) * p.inv_n;
        if constexpr (FAR) {
            s = 0.0f;
            for (int c = threadIdx.x; c < p.N; c += kLongBlock) s += at(c) - mean;
            rest = __fdiv_rn(row_sum<0>(s, red[2]), static_cast<float>(p.N));
        }
        s = 0.0f;
        for (int c = threadIdx.x; c < p.N; c += kLongBlock) {
            const float d = FAR ? at(c) - mean - rest : at(c) - mean;
            s = fmaf(d, d, s);
        }
        const float variance = row_sum<0>(s, red[1]) * p.inv_n;
        rstd = rsqrtf(variance + p.eps);
        far = mean_far(mean, variance);
        if (threadIdx.x == 0) {
            if (p.mean != nullptr) p.mean[row] = mean + rest;
            if (p.rstd != nullptr) p.rstd[row] = rstd;
        }
    }
    if (!FAR && p.sum != nullptr)
        for (int c = threadIdx.x; c < p.N; c += kLongBlock) static_cast<T*>(p.sum)[row * p.N + c] = from_float<T>(at(c));
    const auto value = [&](int c) {
        float v = at(c);
        if (!p.norm) return v;
        v = (FAR ? v - mean - rest : v - mean) * rstd;
        if (p.w == nullptr) return v;
        return fmaf(v, to_float(static_cast<const T*>(p.w)[c]), p.b == nullptr ? 0.0f : to_float(static_cast<const T*>(p.b)[c]));
    };
    if (p.q == nullptr) {
        for (int c = threadIdx.x; c < p.N; c += kLongBlock) static_cast<T*>(p.y)[row * p.N + c] = from_float<T>(value(c));
        return far;
    }
    float top = 0.0f;
    for (int c = threadIdx.x; c < p.N; c += kLongBlock) top = max_nan(top, fabsf(value(c)));
    const RowScale k = row_scale(row_max<0>(top, red[2]));
    if (threadIdx.x == 0) p.scale[row] = k.scale;
    for (int c = threadIdx.x; c < p.N; c += kLongBlock)
        p.q[row * p.qs + c] = quantise(value(c), k.inv);
    return far;
}

template <typename T>
__device__ __noinline__ void far_long_row(const NormParams& p, float (&red)[3][32])
{
    norm_long_row<T, true>(p, red);
}

// Rows of any length, a block each.
template <typename T>
__global__ void __launch_bounds__(kLongBlock) layer_norm_long_kernel(const __grid_constant__ NormParams p)
{
    __shared__ float red[3][32];
    if (norm_long_row<T, false>(p, red)) far_long_row<T>(p, red);
}

template <typename T, int V, int P, int GROUP, int R, bool DSUM>
__global__ void __launch_bounds__(GROUP ? kBlock : row_threads(V, P, true), GROUP ? kBackwardBlocks : row_blocks(V, P)) layer_norm_backward_kernel(const __grid_constant__ NormParams p)
{
    constexpr int E = P * V / 2;
    constexpr int kGroups = GROUP ? kBlock / (GROUP ? GROUP : 1) : 1;  // rows of a block side by side
    constexpr int kJoin = GROUP ? kBlock * P * V : 1;                  // values of a block's rows
    __shared__ float joined[kJoin];
    __shared__ float red[2][GROUP ? 1 : 64 * R];
    const int lane = GROUP ? threadIdx.x % (GROUP ? GROUP : 1) : threadIdx.x;
    const int group = GROUP ? threadIdx.x / (GROUP ? GROUP : 1) : 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kGroups * R);
    int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kGroups * R) + group;
    const Columns<V, P, GROUP> column(pair_shift<V>(p, row0));
    Pair w[E], dw[E], db[E];
    {
        Piece<T, V> raw[P];
        load_weights(raw, static_cast<const T*>(p.w), p.N, column);
        values_of<T, V, P>(raw, w);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        dw[i] = db[i] = pair(0.0f, 0.0f);
        if (p.w == nullptr) w[i] = pair(1.0f, 1.0f);
    }
    // What lies beyond the row stays 0 in dy, and with it in every sum; so do rows beyond the last.  x is 0 there as well,
    // with a mean of 0 (-mean rstd times 0 is NaN where it passes fp32's range); few single values, where that is a
    // select each, take the row's last value instead (rows of 1337 in fp32 31 us and 32.4; 16 values a lane would spill).
    constexpr bool kLast = V == 1 && P <= 8;
    // one condition for a piece of all tensors, or each its own (300000 rows of 101, fp16, 115 and 95 us; 100000 of 401 74 and 83)
    constexpr bool kTogether = V > 2 || P == 16;
    const T* xp = static_cast<const T*>(p.x) + row0 * p.xs + column.first;
    const T* gp = static_cast<const T*>(p.dy) + row0 * p.gs + column.first;
    const T* sp = DSUM ? static_cast<const T*>(p.dsum) + row0 * p.ds + column.first : nullptr;
    T* to = static_cast<T*>(p.dx) + row0 * p.N + column.first;
    const int64_t x_step = step * p.xs, g_step = step * p.gs, s_step = step * p.ds, to_step = step * p.N;
    Piece<T, V> xr[R][P], gr[R][P], sr[DSUM ? R : 1][P];
    float mean[R], rstd[R];
    const auto load = [&](int64_t at) {  // rows at + j kGroups, from the pointers
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const bool real = at + j * kGroups < p.rows;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                if constexpr (kTogether) {
                    if (real && column(i) < p.N) {
                        xr[j][i].load(xp + j * kGroups * p.xs + i * column.kNext);
                        gr[j][i].load(gp + j * kGroups * p.gs + i * column.kNext);
                        if constexpr (DSUM) sr[j][i].load(sp + j * kGroups * p.ds + i * column.kNext);
                    } else {
                        xr[j][i].clear();
                        gr[j][i].clear();
                        if constexpr (DSUM) sr[j][i].clear();
                    }
                    continue;
                }
                if constexpr (kLast) {
                    xr[j][i].clear();
                    if (real) xr[j][i].load(xp + j * kGroups * p.xs + (min(column(i), p.N - 1) - column.first));
                } else {
                    load_piece<false>(xr[j][i], xp + j * kGroups * p.xs + i * column.kNext, i, p.N, real, column);
                }
                load_piece<false>(gr[j][i], gp + j * kGroups * p.gs + i * column.kNext, i, p.N, real, column);
                if constexpr (DSUM) load_piece<false>(sr[j][i], sp + j * kGroups * p.ds + i * column.kNext, i, p.N, real, column);
            }
            mean[j] = real ? __ldg(p.mean + at + j * kGroups) : 0.0f;
            rstd[j] = real ? __ldg(p.rstd + at + j * kGroups) : 0.0f;
        }
    };
    load(row0);
    int turn = 0;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * (kGroups * R); base < p.rows; base += step, row0 += step, to += to_step, turn ^= 1) {
        Pair xh[R][E], g[R][E], d[DSUM ? R : 1][E];
        float rs[R], v[2 * R];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            values_of<T, V, P>(xr[j], xh[j]);
            values_of<T, V, P>(gr[j], g[j]);
            if constexpr (DSUM) values_of<T, V, P>(sr[j], d[j]);
            rs[j] = rstd[j];
            const Pair r2 = pair(rs[j], rs[j]);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const bool out0 = !kLast && !column.has(2 * i / V, 2 * i % V, p.N), out1 = !kLast && !column.has((2 * i + 1) / V, (2 * i + 1) % V, p.N);
                xh[j][i] = mul2(add2(xh[j][i], pair(out0 ? 0.0f : -mean[j], out1 ? 0.0f : -mean[j])), r2);
            }
        }
        if (base + step < p.rows) {
            xp += x_step;
            gp += g_step;
            if constexpr (DSUM) sp += s_step;
            load(row0 + step);
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
            Pair s1 = pair(0.0f, 0.0f), s2 = s1;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                dw[i] = fma2(g[j][i], xh[j][i], dw[i]);
                db[i] = add2(db[i], g[j][i]);
                g[j][i] = mul2(g[j][i], w[i]);
                s1 = add2(s1, g[j][i]);
                s2 = fma2(g[j][i], xh[j][i], s2);
            }
            v[2 * j] = both(s1);
            v[2 * j + 1] = both(s2);
        }
        row_sums<GROUP>(v, red[turn]);
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const float m1 = v[2 * j] * p.inv_n, m2 = v[2 * j + 1] * p.inv_n;
            const Pair a = pair(-m1, -m1), b = pair(-m2, -m2), r2 = pair(rs[j], rs[j]);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const Pair u = fma2(xh[j][i], b, add2(g[j][i], a));
                if constexpr (DSUM) g[j][i] = fma2(u, r2, d[j][i]);
                else g[j][i] = mul2(u, r2);
            }
            if (row0 + j * kGroups < p.rows)
#pragma unroll
                for (int i = 0; i < P; ++i)
                    store_row_piece(to + static_cast<int64_t>(j * kGroups) * p.N + i * column.kNext, g[j], i, p.N, column);
        }
    }
    if (p.part == nullptr) return;
    start_launch_behind();  // the join, which waits for this grid's end
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* sums = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + which) * p.N;
        float v[2 * E];
#pragma unroll
        for (int i = 0; i < E; ++i) unpair(which ? db[i] : dw[i], v[2 * i], v[2 * i + 1]);
        if constexpr (GROUP == 0) {
#pragma unroll
            for (int e = 0; e < 2 * E; ++e) {
                if (column.has(e / V, e % V, p.N) && column(e / V) + e % V < p.N) sums[column(e / V) + e % V] = v[e];
            }
        } else {
            constexpr int kRow = GROUP * P * V;  // columns kept of a row
            __syncthreads();                     // the sums before have been read
#pragma unroll
            for (int e = 0; e < 2 * E; ++e) joined[group * kRow + (e / V * GROUP + lane) * V + e % V] = v[e];
            __syncthreads();
            for (int c = threadIdx.x; c < p.N; c += kBlock) {
                float s = 0.0f;
#pragma unroll 8
                for (int k = 0; k < kGroups; ++k) s += joined[k * kRow + c];
                sums[c] = s;
            }
        }
    }
}

// The same for rows of more than a piece a lane: registers hold the weights and their sums, the rows to come lie in a ring in
// shared memory, a ring for each warp (GROUP) or block, filled by bulk copies of whole rows.
// us with a row under way in registers (longer rows than 512 in blocks), and so: 153600 rows of 320, fp16, 72 and 59; 60000 of 768 68 and
// 51, with dsum 84 and 61; 100000 of 1024, bf16, 118 and 104 (614 MB, 5.9 TB/s); 20000 of 4096 101 and 87, with dsum 120 and 105
// (6.2 TB/s); 10000 of 4096, fp32, with dsum 134 and 98; 300 of 4096 19 and 10.8; 64 of 1024 3.9 and 4.2.
constexpr int ring_threads(int pieces) { return pieces == 3 ? 384 : 256; }  // of a block of warps, as registers allow
constexpr int ring_blocks(int pieces) { return pieces == 2 ? 2 : 1; }
constexpr int kRingRowThreads = 512;  // of an SM's blocks that hold a row each

template <typename T, int V, int P, int GROUP, bool DSUM>
__global__ void __launch_bounds__(GROUP ? ring_threads(P) : kRingRowThreads, GROUP ? ring_blocks(P) : 1)
    layer_norm_backward_ring_kernel(const __grid_constant__ NormParams p)
{
    constexpr int E = P * V / 2, kTensors = DSUM ? 3 : 2;
    constexpr int kRows = GROUP ? 32 / (GROUP ? GROUP : 1) : 1;  // of a warp side by side
    extern __shared__ __align__(16) uint8_t ring[];
    const int owners = GROUP ? blockDim.x / 32 : 1, owner = GROUP ? threadIdx.x / 32 : 0, S = p.stages;
    const int sub = GROUP ? threadIdx.x % 32 / (GROUP ? GROUP : 1) : 0;
    const bool leader = GROUP ? threadIdx.x % 32 == 0 : threadIdx.x == 0;
    const Columns<V, P, GROUP> column;
    const uint32_t row_bytes = p.N * static_cast<uint32_t>(sizeof(T)), stage = kTensors * kRows * row_bytes;
    float* const red = reinterpret_cast<float*>(ring + static_cast<uint32_t>(owners * S) * (stage + 8));  // [2][64] of a block that holds a row
    uint8_t* const mine = ring + static_cast<uint32_t>(owner * S) * stage;
    const uint32_t to_mine = umma::smem_addr(mine), bars = umma::smem_addr(ring) + static_cast<uint32_t>(owners * S) * stage + owner * S * 8;
    // few rows go to many blocks: an owner of each before the second of any
    const int64_t step = static_cast<int64_t>(gridDim.x) * owners * kRows;
    int64_t row0 = (static_cast<int64_t>(owner) * gridDim.x + blockIdx.x) * kRows;
    // the leader's: rows to come, and where they are
    int64_t ahead = row0;
    const T* xp = static_cast<const T*>(p.x) + row0 * p.xs;
    const T* gp = static_cast<const T*>(p.dy) + row0 * p.gs;
    const T* sp = DSUM ? static_cast<const T*>(p.dsum) + row0 * p.ds : nullptr;
    const int64_t x_step = step * p.xs, g_step = step * p.gs, s_step = step * p.ds;
    const auto rows_in = [&](const T* from, int64_t stride, uint32_t to, int n, uint32_t bar) {
        if (kRows == 1 || stride == p.N) {
            umma::bulk_g2s(to, from, n * row_bytes, bar);
        } else {
            for (int j = 0; j < n; ++j) umma::bulk_g2s(to + j * row_bytes, from + j * stride, row_bytes, bar);
        }
    };
    const auto fill = [&](int s) {
        if (ahead >= p.rows) return;
        const int n = kRows == 1 ? 1 : static_cast<int>(min(static_cast<int64_t>(kRows), p.rows - ahead));
        const uint32_t bar = bars + s * 8, to = to_mine + s * stage;
        umma::mbar_arrive_expect_tx(bar, n * kTensors * row_bytes);
        rows_in(xp, p.xs, to, n, bar);
        rows_in(gp, p.gs, to + kRows * row_bytes, n, bar);
        if constexpr (DSUM) rows_in(sp, p.ds, to + 2 * kRows * row_bytes, n, bar);
        ahead += step;
        xp += x_step;
        gp += g_step;
        if constexpr (DSUM) sp += s_step;
    };
    if (leader) {
        for (int s = 0; s < S; ++s) umma::mbar_init(bars + s * 8, 1);
        umma::mbar_fence_init();
        for (int s = 0; s < S; ++s) fill(s);
    }
    Pair w[E], dw[E], db[E];
    {
        Piece<T, V> raw[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            raw[i].clear();
            if (p.w != nullptr && column(i) < p.N) raw[i].load(static_cast<const T*>(p.w) + column(i));
        }
        values_of<T, V, P>(raw, w);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        dw[i] = db[i] = pair(0.0f, 0.0f);
        if (p.w == nullptr) w[i] = pair(1.0f, 1.0f);
    }
    float mean = 0.0f, rstd = 0.0f;
    const auto stats = [&](int64_t row) {
        mean = row < p.rows ? __ldg(p.mean + row) : 0.0f;
        rstd = row < p.rows ? __ldg(p.rstd + row) : 0.0f;
    };
    stats(row0 + sub);
    __syncthreads();  // the barriers are there
    int s = 0, turn = 0;
    uint32_t parity = 0;
    bool ok = true;
    for (; row0 < p.rows; row0 += step, turn ^= 1) {
        ok = ok && umma::mbar_poll(bars + s * 8, parity);  // once given up, no wait and no copy follows
        const bool real = row0 + sub < p.rows;
        Pair xh[E], g[E];
        const float rs = rstd;
        const T* from = reinterpret_cast<const T*>(mine + s * stage + sub * row_bytes);
        const uint32_t next = kRows * p.N;
        {
            // what lies beyond the row, and rows beyond the last, are zeros, with a mean of 0
            Piece<T, V> x[P], y[P];
#pragma unroll
            for (int i = 0; i < P; ++i) {
                x[i].clear();
                y[i].clear();
                if (real && column(i) < p.N) {
                    x[i].load_shared(from + column(i));
                    y[i].load_shared(from + next + column(i));
                }
            }
            values_of<T, V, P>(x, xh);
            values_of<T, V, P>(y, g);
        }
        const Pair r2 = pair(rs, rs);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float m = column(2 * i / V) < p.N ? -mean : 0.0f;
            xh[i] = mul2(add2(xh[i], pair(m, m)), r2);
        }
        stats(row0 + step + sub);
        if constexpr (GROUP != 0 && !DSUM) {
            __syncwarp();  // the stage has been read
            if (leader && ok) fill(s);
        }
        Pair s1 = pair(0.0f, 0.0f), s2 = s1;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            dw[i] = fma2(g[i], xh[i], dw[i]);
            db[i] = add2(db[i], g[i]);
            g[i] = mul2(g[i], w[i]);
            s1 = add2(s1, g[i]);
            s2 = fma2(g[i], xh[i], s2);
        }
        float v[2] = {both(s1), both(s2)};
        row_sums<GROUP>(v, red + turn * 64);
        if constexpr (GROUP == 0) {  // row_sums' barrier: the stage has been read, or with dsum the one before
            if (!DSUM && leader && ok) fill(s);
            if (DSUM && leader && ok && row0 >= gridDim.x) fill(s == 0 ? S - 1 : s - 1);
        }
        const float m1 = v[0] * p.inv_n, m2 = v[1] * p.inv_n;
        const Pair a = pair(-m1, -m1), b = pair(-m2, -m2);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const Pair u = fma2(xh[i], b, add2(g[i], a));
            if constexpr (DSUM) g[i] = u;
            else g[i] = mul2(u, r2);
        }
        if (real) {
            T* to = static_cast<T*>(p.dx) + (row0 + sub) * p.N;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                if (column(i) >= p.N) continue;
                if constexpr (DSUM) {
                    Piece<T, V> z[1];
                    Pair d[V / 2];
                    z[0].load_shared(from + 2 * next + column(i));
                    values_of<T, V, 1>(z, d);
#pragma unroll
                    for (int e = 0; e < V / 2; ++e) g[i * V / 2 + e] = fma2(g[i * V / 2 + e], r2, d[e]);
                }
                store_piece<T, V>(to + column(i), g, i);
            }
        }
        if constexpr (GROUP != 0 && DSUM) {
            __syncwarp();
            if (leader && ok) fill(s);
        }
        if (++s == S) {
            s = 0;
            parity ^= 1;
        }
    }
    if (!ok) record_device_error(p.err, kErrMbarTimeout | 0x60);
    if (p.part == nullptr) return;
    start_launch_behind();  // the join, which waits for this grid's end
    float* joined = reinterpret_cast<float*>(ring);
    const int lane = threadIdx.x % (GROUP ? GROUP : 1), group = threadIdx.x / (GROUP ? GROUP : 1), groups = blockDim.x / (GROUP ? GROUP : 1);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* sums = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + which) * p.N;
        float v[2 * E];
#pragma unroll
        for (int i = 0; i < E; ++i) unpair(which ? db[i] : dw[i], v[2 * i], v[2 * i + 1]);
        if (GROUP == 0 || groups == 1) {
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (column(i) < p.N)
#pragma unroll
                    for (int e = i * V; e < (i + 1) * V; e += 4)
                        *reinterpret_cast<float4*>(sums + column(i) + e % V) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        } else {
            constexpr int kRow = GROUP * P * V;  // columns kept of a row
            __syncthreads();                     // the rings, or the sums before, have been read
#pragma unroll
            for (int e = 0; e < 2 * E; ++e) joined[group * kRow + (e / V * GROUP + lane) * V + e % V] = v[e];
            __syncthreads();
            for (int c = threadIdx.x; c < p.N; c += blockDim.x) {
                float t = 0.0f;
#pragma unroll 8
                for (int k = 0; k < groups; ++k) t += joined[k * kRow + c];
                sums[c] = t;
            }
        }
    }
}

// Rows of any length: dx by a block for each row, the weight's and bias's sums by columns.
template <typename T>
__global__ void __launch_bounds__(kLongBlock) layer_norm_backward_long_kernel(const __grid_constant__ NormParams p)
{
    __shared__ float red[2][32];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.xs;
    const T* dy = static_cast<const T*>(p.dy) + row * p.gs;
    const T* w = static_cast<const T*>(p.w);
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < p.N; c += kLongBlock) {
        const float g = to_float(dy[c]) * (w == nullptr ? 1.0f : to_float(w[c]));
        s1 += g;
        s2 = fmaf(g, (to_float(x[c]) - mean) * rstd, s2);
    }
    s1 = row_sum<0>(s1, red[0]) * p.inv_n;
    s2 = row_sum<0>(s2, red[1]) * p.inv_n;
    for (int c = threadIdx.x; c < p.N; c += kLongBlock) {
        const float g = to_float(dy[c]) * (w == nullptr ? 1.0f : to_float(w[c]));
        float d = rstd * (g - s1 - (to_float(x[c]) - mean) * rstd * s2);
        if (p.dsum != nullptr) d += to_float(static_cast<const T*>(p.dsum)[row * p.ds + c]);
        static_cast<T*>(p.dx)[row * p.N + c] = from_float<T>(d);
    }
}

template <typename T>
__global__ void __launch_bounds__(kBlock) layer_norm_columns_kernel(const __grid_constant__ NormParams p)
{
    const int c = blockIdx.x * kBlock + threadIdx.x;
    if (c >= p.N) return;
    float dw = 0.0f, db = 0.0f;
#pragma unroll 4
    for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const float g = to_float(static_cast<const T*>(p.dy)[row * p.gs + c]);
        dw = fmaf(g, (to_float(static_cast<const T*>(p.x)[row * p.xs + c]) - __ldg(p.mean + row)) * __ldg(p.rstd + row), dw);
        db += g;
    }
    p.part[static_cast<int64_t>(blockIdx.y) * 2 * p.N + c] = dw;
    p.part[(static_cast<int64_t>(blockIdx.y) * 2 + 1) * p.N + c] = db;
}

// Joins the blocks' sums: 8 columns a block (a sector of each part), 32 threads of each
// over the parts.
constexpr int kJoinColumns = 8;
template <typename T>
__global__ void __launch_bounds__(kJoinColumns * 32) layer_norm_join_kernel(const float* part, int parts, int N, T* dw, T* db)
{
    __shared__ float sums[32][kJoinColumns + 1];
    const int at = threadIdx.x % kJoinColumns, lane = threadIdx.x / kJoinColumns;
    const int64_t all = 2 * static_cast<int64_t>(N), c = static_cast<int64_t>(blockIdx.x) * kJoinColumns + at;
    wait_for_launches_before();
    float s = 0.0f;
    if (c < all)
#pragma unroll 10
        for (int k = lane; k < parts; k += 32) s += part[k * all + c];
    sums[lane][at] = s;
    __syncthreads();
    const int column = threadIdx.x / 32;
    s = sums[threadIdx.x % 32][column];
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    const int64_t to = static_cast<int64_t>(blockIdx.x) * kJoinColumns + column;
    if (threadIdx.x % 32 == 0 && to < all) {
        if (to < N) dw[to] = from_float<T>(s);
        else db[to - N] = from_float<T>(s);
    }
}

bool aligned(const void* p) noexcept { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Rows that can be read and written in pieces of 16 bytes.
bool in_pieces(const ww_layer_norm_t& p, int bytes) noexcept
{
    const int v = 16 / bytes;
    if (p.N % v != 0) return false;
    for (const void* q : {p.x, p.residual, p.weight, p.bias, static_cast<const void*>(p.y), static_cast<const void*>(p.sum), p.dy, p.dsum,
                          static_cast<const void*>(p.dx)})
        if (!aligned(q)) return false;
    for (int64_t s : {p.x_stride, p.residual_stride, p.dy_stride, p.dsum_stride})
        if (s % v != 0) return false;
    return p.y_q == nullptr || (reinterpret_cast<uintptr_t>(p.y_q) % 8 == 0 && p.y_q_stride % v == 0);
}

// Rows of pairs: every tensor's row begins on the grid of two values, or every one off it.  For rows of which a lane
// holds 16 values; us by single values and by pairs: 8000 rows of 5001, fp16, 75 and 64, 4000 in fp32 38 and 30, gradients
// of 6000 198 and 123, of 3000 in fp32 124 and 88; but 40000 of 1337, fp16, 82 and 113, gradients of 401 74 and 78, of 1337 70 and 76.
constexpr int kPairs = 2048;
bool in_pairs(const ww_layer_norm_t& p, int bytes) noexcept
{
    if (p.N <= kPairs) return false;
    const auto off = [&](const void* q) { return reinterpret_cast<uintptr_t>(q) / bytes % 2; };
    for (const void* q : {p.residual, static_cast<const void*>(p.y), static_cast<const void*>(p.sum), p.dy, p.dsum, static_cast<const void*>(p.dx)})
        if (q != nullptr && off(q) != off(p.x)) return false;
    const auto like = [&](const void* q, int64_t stride) { return q == nullptr || p.rows == 1 || (stride - p.N) % 2 == 0; };
    return like(p.x, p.x_stride) && like(p.residual, p.residual_stride) && like(p.dy, p.dy_stride) && like(p.dsum, p.dsum_stride);
}

NormParams params(const ww_layer_norm_t& p, bool norm) noexcept
{
    NormParams f{};
    f.shift = static_cast<int>(reinterpret_cast<uintptr_t>(p.x) / (p.dtype == WW_DTYPE_FLOAT ? 4 : 2) % 2);
    f.odd = p.N % 2;
    f.x = p.x;
    f.r = p.residual;
    f.w = p.weight;
    f.b = p.bias;
    f.y = p.y;
    f.sum = p.sum;
    f.q = p.y_q;
    f.scale = p.y_scale;
    f.mean = p.mean;
    f.rstd = p.rstd;
    f.dy = p.dy;
    f.dsum = p.dsum;
    f.dx = p.dx;
    f.xs = p.x_stride;
    f.rs = p.residual_stride;
    f.qs = p.y_q_stride;
    f.gs = p.dy_stride;
    f.ds = p.dsum_stride;
    f.rows = p.rows;
    f.N = p.N;
    f.norm = norm;
    f.eps = p.eps;
    f.inv_n = 1.0f / static_cast<float>(p.N);
    return f;
}

// Blocks, an even number where each takes rows of pairs one after another.
int even_step(int64_t blocks, int64_t rows, const RowForm& form, bool pairs) noexcept
{
    return static_cast<int>(pairs && form.group == 0 && blocks < rows ? std::max<int64_t>(2, blocks & ~int64_t{1}) : blocks);
}

template <typename T>
bool launch_ring(NormParams& f, int threads, int sms, cudaStream_t stream) noexcept
{
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    const auto kernel = layer_norm_ring_kernel<T, V>;
    static std::atomic<uint64_t> raised{0};
    f.err = device_error_slot();
    if (f.err == nullptr || !allow_shared_memory(reinterpret_cast<const void*>(kernel), raised)) return false;
    const int resident = std::max(1, forward_threads(true) / threads), stage = 2 * f.N * static_cast<int>(sizeof(T)) + 8;
    f.stages = std::min(8, (kMaxShared / resident - 2048) / stage);  // 3 of the longest rows, 2 x 32 KB
    kernel<<<std::min(sms * resident, f.rows), threads, f.stages * stage + 768, stream>>>(f);
    return true;
}

template <typename T>
int forward(const ww_layer_norm_t& p, bool norm, int sms, const char* name, cudaStream_t stream) noexcept
{
    NormParams f = params(p, norm);
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    const bool pieces = in_pieces(p, sizeof(T)), pairs = !pieces && in_pairs(p, sizeof(T));
    const RowForm form = row_form(p.N, pieces ? V : pairs ? 2 : 1, 4, false);
    const auto go = [&](auto kernel, auto with_residual, int r) {
        const int groups = (form.group ? kBlock / form.group : 1) * r;
        const int resident = form.group ? forward_blocks(pieces ? V : 1, form.pieces, p.residual != nullptr) : std::max(1, forward_threads(pieces) / form.threads);
        const unsigned grid = even_step(std::min<int64_t>(i64(sms) * resident, (i64(p.rows) + groups - 1) / groups), i64(p.rows), form, pairs);
        if (p.residual == nullptr) kernel<<<grid, form.threads, 0, stream>>>(f);
        else with_residual<<<grid, form.threads, 0, stream>>>(f);
    };
#define WW_NORM(V, P, GROUP) \
    go(layer_norm_kernel<T, V, P, GROUP, rows_at_once(V, P, GROUP), false>, layer_norm_kernel<T, V, P, GROUP, rows_at_once(V, P, GROUP), true>, \
       rows_at_once(V, P, GROUP))
    const int id = form.group * 100 + form.pieces;
    if (form.threads == 0) layer_norm_long_kernel<T><<<p.rows, kLongBlock, 0, stream>>>(f);
    else if (pairs) WW_NORM(2, 8, 0);
    else if (!pieces)
        switch (id) {
        case 3204: WW_NORM(1, 4, 32); break;
        case 3216: WW_NORM(1, 16, 32); break;
        case 8: WW_NORM(1, 8, 0); break;
        default: WW_NORM(1, 16, 0); break;
        }
    else
        switch (id) {
        case 401: WW_NORM(V, 1, 4); break;
        case 801: WW_NORM(V, 1, 8); break;
        case 1601: WW_NORM(V, 1, 16); break;
        case 1603: WW_NORM(V, 3, 16); break;
        case 3201: WW_NORM(V, 1, 32); break;
        case 3202: WW_NORM(V, 2, 32); break;
        case 3203: WW_NORM(V, 3, 32); break;
        case 3204: WW_NORM(V, 4, 32); break;
        default:
            // rings start later: for rows of several turns
            if (norm && p.residual != nullptr && p.rows > 2 * sms * std::max(1, forward_threads(true) / form.threads)) {
                if (!launch_ring<T>(f, form.threads, sms, stream)) {
                    const int st = launch_status(name);
                    return st != WW_SUCCESS ? st : WW_ERR_DEVICE;
                }
            } else {
                WW_NORM(V, 2, 0);
            }
            break;
        }
#undef WW_NORM
    return launch_status(name);
}

// Blocks of the gradient: one resident round, as far as there are rows for it.
struct BackwardPlan {
    bool pieces, pairs, ring;
    RowForm form;
    int blocks, splits;  // splits: of the rows, for the sums by columns (long rows)
    int stages, shared;  // of a ring, bytes of its block
    int parts() const { return form.threads == 0 ? splits : blocks; }
};

BackwardPlan backward_plan(const ww_layer_norm_t& p, int sms) noexcept
{
    const int bytes = p.dtype == WW_DTYPE_FLOAT ? 4 : 2;
    BackwardPlan r{};
    r.pieces = in_pieces(p, bytes);
    r.pairs = !r.pieces && in_pairs(p, bytes);
    const int v = r.pieces ? 16 / bytes : r.pairs ? 2 : 1;
    r.form = row_form(p.N, v, 4, true);
    r.ring = r.pieces && r.form.pieces > 1;
    if (r.ring) {
        // an owner of rows in each block before the second of any, and as many stages as fit and are needed (2 or more fit: rows
        // of 16 KB of three tensors 4)
        const int resident = r.form.group ? ring_blocks(r.form.pieces) : std::max(1, kRingRowThreads / r.form.threads);
        const int at_once = r.form.group ? 32 / r.form.group : 1;
        const int64_t turns = (i64(p.rows) + at_once - 1) / at_once;
        r.blocks = static_cast<int>(std::min<int64_t>(i64(sms) * resident, turns));
        int owners = 1;
        if (r.form.group) {
            owners = static_cast<int>(std::min<int64_t>(ring_threads(r.form.pieces) / 32, (turns + r.blocks - 1) / r.blocks));
            r.form.threads = 32 * owners;
        }
        const int stage = owners * at_once * p.N * bytes * (p.dsum == nullptr ? 2 : 3) + 8 * owners;
        const int64_t needed = (turns + r.blocks * owners - 1) / (r.blocks * owners);
        r.stages = static_cast<int>(std::min<int64_t>({8, needed, (kMaxShared / resident - 2048) / stage}));
        r.shared = std::max(r.stages * stage + 512, r.form.group ? r.form.threads * r.form.pieces * v * 4 : 0);
        return r;
    }
    const int groups = r.form.group ? kBlock / r.form.group : 1;
    int resident = kBackwardBlocks;
    if (r.form.group == 0 && r.form.threads > 0) resident = std::max(1, backward_threads(r.pairs ? 16 : r.form.pieces) / r.form.threads);
    const int at_once = groups * rows_at_once(v, r.form.pieces, r.form.group);
    r.blocks = even_step(std::min<int64_t>(i64(sms) * resident, (i64(p.rows) + at_once - 1) / at_once), p.rows, r.form, r.pairs);
    const int columns = (p.N + kBlock - 1) / kBlock;
    r.splits = std::max(1, std::min(p.rows, 4 * sms / columns));
    return r;
}

template <typename T, int P, int GROUP>
bool launch_ring(NormParams& f, const BackwardPlan& plan, cudaStream_t stream) noexcept
{
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    const bool sum = f.dsum != nullptr;
    const auto kernel = sum ? layer_norm_backward_ring_kernel<T, V, P, GROUP, true> : layer_norm_backward_ring_kernel<T, V, P, GROUP, false>;
    static std::atomic<uint64_t> raised[2];
    f.stages = plan.stages;
    f.err = device_error_slot();
    if (f.err == nullptr || !allow_shared_memory(reinterpret_cast<const void*>(kernel), raised[sum])) return false;
    kernel<<<plan.blocks, plan.form.threads, plan.shared, stream>>>(f);
    return true;
}

template <typename T>
int backward(const ww_layer_norm_t& p, const BackwardPlan& plan, cudaStream_t stream) noexcept
{
    NormParams f = params(p, true);
    const bool sums = p.dweight != nullptr;
    f.part = sums ? static_cast<float*>(p.workspace) : nullptr;
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    const RowForm& form = plan.form;
    bool ready = true;
    const auto go = [&](auto kernel, auto with_sum) {
        if (p.dsum == nullptr) kernel<<<plan.blocks, form.threads, 0, stream>>>(f);
        else with_sum<<<plan.blocks, form.threads, 0, stream>>>(f);
    };
#define WW_NORM(V, P, GROUP) \
    go(layer_norm_backward_kernel<T, V, P, GROUP, rows_at_once(V, P, GROUP), false>, \
       layer_norm_backward_kernel<T, V, P, GROUP, rows_at_once(V, P, GROUP), true>)
    const int id = form.group * 100 + form.pieces;
    if (form.threads == 0) {
        layer_norm_backward_long_kernel<T><<<p.rows, kLongBlock, 0, stream>>>(f);
        if (sums) layer_norm_columns_kernel<T><<<dim3((p.N + kBlock - 1) / kBlock, plan.splits), kBlock, 0, stream>>>(f);
    } else if (plan.pairs) {
        WW_NORM(2, 8, 0);
    } else if (!plan.pieces) {
        switch (id) {
        case 3204: WW_NORM(1, 4, 32); break;
        case 3216: WW_NORM(1, 16, 32); break;
        case 8: WW_NORM(1, 8, 0); break;
        default: WW_NORM(1, 16, 0); break;
        }
    } else {
        switch (id) {
        case 401: WW_NORM(V, 1, 4); break;
        case 801: WW_NORM(V, 1, 8); break;
        case 1601: WW_NORM(V, 1, 16); break;
        case 3201: WW_NORM(V, 1, 32); break;
        case 1603: ready = launch_ring<T, 3, 16>(f, plan, stream); break;
        case 3202: ready = launch_ring<T, 2, 32>(f, plan, stream); break;
        case 3203: ready = launch_ring<T, 3, 32>(f, plan, stream); break;
        case 3204: ready = launch_ring<T, 4, 32>(f, plan, stream); break;
        default: ready = launch_ring<T, 2, 0>(f, plan, stream); break;
        }
    }
#undef WW_NORM
    const int st = launch_status("layer_norm_backward");
    if (!ready) return st != WW_SUCCESS ? st : WW_ERR_DEVICE;
    if (st != WW_SUCCESS || !sums) return st;
    launch_behind(layer_norm_join_kernel<T>, dim3((2u * p.N + kJoinColumns - 1) / kJoinColumns), dim3(kJoinColumns * 32), 0, stream, f.part, plan.parts(), p.N,
                  static_cast<T*>(p.dweight), static_cast<T*>(p.dbias));
    return launch_status("layer_norm_backward");
}

// What both directions check.
int check(const ww_layer_norm_t& p, bool norm) noexcept
{
    if (p.dtype != WW_DTYPE_HALF && p.dtype != WW_DTYPE_BF16 && p.dtype != WW_DTYPE_FLOAT) return WW_ERR_INVALID_DTYPE;
    if (p.rows < 0 || p.N <= 0) return WW_ERR_INVALID_SHAPE;
    if (norm && !(p.eps >= 0.0f && std::isfinite(p.eps))) return WW_ERR_INVALID_SHAPE;
    if (p.N > (1 << 24)) return WW_ERR_UNSUPPORTED;
    if (p.rows > 0 && p.x == nullptr) return WW_ERR_NULL_POINTER;
    for (int64_t s : {p.x_stride, p.residual_stride, p.dy_stride, p.dsum_stride})
        if (s < 0) return WW_ERR_INVALID_SHAPE;
    const int bytes = p.dtype == WW_DTYPE_FLOAT ? 4 : 2;
    for (const void* q : {p.x, p.residual, p.weight, p.bias, static_cast<const void*>(p.y), static_cast<const void*>(p.sum), p.dy, p.dsum,
                          static_cast<const void*>(p.dx), static_cast<const void*>(p.dweight), static_cast<const void*>(p.dbias)})
        if (reinterpret_cast<uintptr_t>(q) % bytes != 0) return WW_ERR_MISALIGNED;
    for (const void* q : {static_cast<const void*>(p.y_scale), static_cast<const void*>(p.mean), static_cast<const void*>(p.rstd)})
        if (reinterpret_cast<uintptr_t>(q) % 4 != 0) return WW_ERR_MISALIGNED;
    return WW_SUCCESS;
}

int check_forward(const ww_layer_norm_t& p, bool norm) noexcept
{
    const int st = check(p, norm);
    if (st != WW_SUCCESS) return st;
    if (p.y_q != nullptr && p.y_q_stride < p.N) return WW_ERR_INVALID_SHAPE;
    if (p.rows == 0) return WW_SUCCESS;
    if ((p.y == nullptr) == (p.y_q == nullptr) || (p.y_q != nullptr && p.y_scale == nullptr)) return WW_ERR_NULL_POINTER;
    if ((p.bias != nullptr && p.weight == nullptr) || (p.sum != nullptr && p.residual == nullptr)) return WW_ERR_NULL_POINTER;
    return WW_SUCCESS;
}

int run_forward(const ww_layer_norm_t& p, bool norm, const char* name, void* stream) noexcept
{
    DeviceInfo d;
    const int st = current_device_info(&d);
    if (st != WW_SUCCESS) return st;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return p.dtype == WW_DTYPE_HALF ? forward<__half>(p, norm, d.sm_count, name, s)
         : p.dtype == WW_DTYPE_BF16 ? forward<__nv_bfloat16>(p, norm, d.sm_count, name, s) : forward<float>(p, norm, d.sm_count, name, s);
}

int sm_count() noexcept
{
    DeviceInfo d;
    return current_device_info(&d) == WW_SUCCESS ? d.sm_count : 148;
}

}  // namespace

int quantise_rows(const ww_layer_norm_t& p, const char* name, void* stream) noexcept { return run_forward(p, false, name, stream); }

}  // namespace ww

extern "C" {

int ww_layer_norm(const ww_layer_norm_t* p, void* stream)
{
    if (p == nullptr) return WW_ERR_NULL_POINTER;
    const int st = ww::check_forward(*p, true);
    if (st != WW_SUCCESS || p->rows == 0) return st;
    return ww::run_forward(*p, true, "layer_norm", stream);
}

int ww_quantize_tokens(const ww_layer_norm_t* p, void* stream)
{
    if (p == nullptr) return WW_ERR_NULL_POINTER;
    const int st = ww::check_forward(*p, false);
    if (st != WW_SUCCESS) return st;
    if (p->rows == 0) return WW_SUCCESS;
    if (p->y_q == nullptr || p->weight != nullptr || p->residual != nullptr) return WW_ERR_NULL_POINTER;
    return ww::run_forward(*p, false, "quantize_tokens", stream);
}

int64_t ww_layer_norm_backward_workspace(const ww_layer_norm_t* p)
{
    if (p == nullptr || ww::check(*p, true) != WW_SUCCESS || p->rows == 0 || p->dweight == nullptr) return 0;
    return int64_t{8} * p->N * ww::backward_plan(*p, ww::sm_count()).parts();
}

int ww_layer_norm_backward(const ww_layer_norm_t* p, void* stream)
{
    if (p == nullptr) return WW_ERR_NULL_POINTER;
    int st = ww::check(*p, true);
    if (st != WW_SUCCESS) return st;
    if ((p->dweight == nullptr) != (p->dbias == nullptr)) return WW_ERR_NULL_POINTER;
    ww::DeviceInfo d;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (p->rows == 0) {
        if (p->dweight == nullptr) return WW_SUCCESS;
        if ((st = ww::current_device_info(&d)) != WW_SUCCESS) return st;
        const size_t bytes = static_cast<size_t>(p->N) * (p->dtype == WW_DTYPE_FLOAT ? 4 : 2);
        if (cudaMemsetAsync(p->dweight, 0, bytes, s) != cudaSuccess || cudaMemsetAsync(p->dbias, 0, bytes, s) != cudaSuccess)
            return ww::launch_status("layer_norm_backward");
        return WW_SUCCESS;
    }
    if (p->dy == nullptr || p->dx == nullptr || p->mean == nullptr || p->rstd == nullptr) return WW_ERR_NULL_POINTER;
    if ((st = ww::current_device_info(&d)) != WW_SUCCESS) return st;
    const ww::BackwardPlan plan = ww::backward_plan(*p, d.sm_count);
    if (p->dweight != nullptr) {
        if (p->workspace == nullptr) return WW_ERR_NULL_POINTER;
        if (reinterpret_cast<uintptr_t>(p->workspace) % 16 != 0) return WW_ERR_MISALIGNED;
        if (p->workspace_bytes < int64_t{8} * p->N * plan.parts()) return WW_ERR_UNSUPPORTED;
    }
    return p->dtype == WW_DTYPE_HALF ? ww::backward<__half>(*p, plan, s)
         : p->dtype == WW_DTYPE_BF16 ? ww::backward<__nv_bfloat16>(*p, plan, s) : ww::backward<float>(*p, plan, s);
}

}  // extern "C"
