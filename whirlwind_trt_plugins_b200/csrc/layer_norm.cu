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
// variance from the deviations, so that a large mean costs nothing), held by a
// group of 4 to 32 lanes or, where a warp's registers do not hold it, by a block;
// loads are 16 bytes a lane where rows start on 16 bytes, else single values.
// The gradient runs one resident round of blocks: a lane owns the same columns of
// all its rows, so the weight's and bias's sums stay in registers; the next row's
// loads are under way while a row is computed.  Sums are joined per block in shared
// memory and over blocks by a second kernel, both in a fixed order.
// Rows beyond a block's registers are read again from L2 for each step.
#include "rows.cuh"

#include <algorithm>
#include <cmath>

namespace ww {
namespace {

constexpr int kBlock = 256;
constexpr int kLongBlock = 1024;
constexpr int kForwardThreads = 1024;  // of a block that holds a row
__host__ __device__ constexpr int backward_threads(int v) { return v > 1 ? 512 : 640; }

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
};

template <typename T, int V, int P, int GROUP>
__global__ void __launch_bounds__(GROUP ? kBlock : kForwardThreads) layer_norm_kernel(const __grid_constant__ NormParams p)
{
    __shared__ float red[3][32];
    constexpr int E = P * V / 2;
    const int lanes = GROUP ? GROUP : static_cast<int>(blockDim.x), lane = GROUP ? threadIdx.x % GROUP : threadIdx.x;
    const int64_t row = GROUP ? static_cast<int64_t>(blockIdx.x) * (kBlock / (GROUP ? GROUP : 1)) + threadIdx.x / (GROUP ? GROUP : 1) : blockIdx.x;
    const int64_t known = min(row, static_cast<int64_t>(p.rows) - 1);
    const T* x = static_cast<const T*>(p.x) + known * p.xs;
    Piece<T, V> raw[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int c = (i * lanes + lane) * V;
        if (c < p.N) raw[i].load(x + c);
        else raw[i].clear();
    }
    Pair f[E];
    values_of<T, V, P>(raw, f);
    if (p.r != nullptr) {
        const T* r = static_cast<const T*>(p.r) + known * p.rs;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c = (i * lanes + lane) * V;
            if (c < p.N) raw[i].load(r + c);
        }
        Pair g[E];
        values_of<T, V, P>(raw, g);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            float a, b;
            unpair(add2(f[i], g[i]), a, b);
            f[i] = pair(to_float(from_float<T>(a)), to_float(from_float<T>(b)));
        }
        if (p.sum != nullptr && row < p.rows) {
            T* to = static_cast<T*>(p.sum) + row * p.N;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int c = (i * lanes + lane) * V;
                if (c < p.N) store_piece<T, V>(to + c, f, i);
            }
        }
#pragma unroll
        for (int i = 0; i < P; ++i)  // beyond the row: zeros again
            if ((i * lanes + lane) * V >= p.N)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float a, b;
                    unpair(f[(i * V + e) / 2], a, b);
                    f[(i * V + e) / 2] = (i * V + e) % 2 ? pair(a, 0.0f) : pair(0.0f, b);
                }
    }
    if (p.norm) {
        Pair s = f[0];
#pragma unroll
        for (int i = 1; i < E; ++i) s = add2(s, f[i]);
        const float mean = row_sum<GROUP>(both(s), red[0]) * p.inv_n;
        const Pair nm = pair(-mean, -mean);
        s = pair(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = add2(f[i], nm);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if ((i * lanes + lane) * V >= p.N) continue;
            if constexpr (V == 1) {
                float a, b;
                unpair(f[i / 2], a, b);
                const float d = i % 2 ? b : a;
                s = fma2(pair(d, 0.0f), pair(d, 0.0f), s);
            } else {
#pragma unroll
                for (int j = i * V / 2; j < (i + 1) * V / 2; ++j) s = fma2(f[j], f[j], s);
            }
        }
        const float rstd = rsqrtf(fmaf(row_sum<GROUP>(both(s), red[1]), p.inv_n, p.eps));
        if (lane == 0 && row < p.rows) {
            if (p.mean != nullptr) p.mean[row] = mean;
            if (p.rstd != nullptr) p.rstd[row] = rstd;
        }
        const Pair r2 = pair(rstd, rstd);
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = mul2(f[i], r2);
        if (p.w != nullptr) {
            Piece<T, V> wr[P], br[P];
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int c = (i * lanes + lane) * V;
                wr[i].clear();
                br[i].clear();
                if (c < p.N) {
                    wr[i].load(static_cast<const T*>(p.w) + c);
                    if (p.b != nullptr) br[i].load(static_cast<const T*>(p.b) + c);
                }
            }
            Pair w[E], b[E];
            values_of<T, V, P>(wr, w);
            values_of<T, V, P>(br, b);
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = fma2(f[i], w[i], b[i]);
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i)  // without weights what lies beyond the row is not 0 yet
                if ((i * lanes + lane) * V >= p.N)
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        float a, b;
                        unpair(f[(i * V + e) / 2], a, b);
                        f[(i * V + e) / 2] = (i * V + e) % 2 ? pair(a, 0.0f) : pair(0.0f, b);
                    }
        }
    }
    if (p.q != nullptr) {
        const RowScale k = row_scale(row_max<GROUP>(largest(f), red[2]));
        if (row >= p.rows) return;
        if (lane == 0) p.scale[row] = k.scale;
        int8_t* to = p.q + row * p.qs;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c = (i * lanes + lane) * V;
            if (c < p.N) store_piece_int8<V>(to + c, f, k.inv, i);
        }
        return;
    }
    if (row >= p.rows) return;
    T* to = static_cast<T*>(p.y) + row * p.N;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int c = (i * lanes + lane) * V;
        if (c < p.N) store_piece<T, V>(to + c, f, i);
    }
}

// Rows of any length: a block each, read again for each step.
template <typename T>
__global__ void __launch_bounds__(kLongBlock) layer_norm_long_kernel(const __grid_constant__ NormParams p)
{
    __shared__ float red[3][32];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.xs;
    const T* r = p.r == nullptr ? nullptr : static_cast<const T*>(p.r) + row * p.rs;
    const auto at = [&](int c) { return r == nullptr ? to_float(x[c]) : to_float(from_float<T>(to_float(x[c]) + to_float(r[c]))); };
    float mean = 0.0f, rstd = 1.0f;
    if (p.norm) {
        float s = 0.0f;
        for (int c = threadIdx.x; c < p.N; c += kLongBlock) s += at(c);
        mean = row_sum<0>(s, red[0]) * p.inv_n;
        s = 0.0f;
        for (int c = threadIdx.x; c < p.N; c += kLongBlock) {
            const float d = at(c) - mean;
            s = fmaf(d, d, s);
        }
        rstd = rsqrtf(fmaf(row_sum<0>(s, red[1]), p.inv_n, p.eps));
        if (threadIdx.x == 0) {
            if (p.mean != nullptr) p.mean[row] = mean;
            if (p.rstd != nullptr) p.rstd[row] = rstd;
        }
    }
    if (p.sum != nullptr)
        for (int c = threadIdx.x; c < p.N; c += kLongBlock) static_cast<T*>(p.sum)[row * p.N + c] = from_float<T>(at(c));
    const auto value = [&](int c) {
        float v = at(c);
        if (!p.norm) return v;
        v = (v - mean) * rstd;
        if (p.w == nullptr) return v;
        return fmaf(v, to_float(static_cast<const T*>(p.w)[c]), p.b == nullptr ? 0.0f : to_float(static_cast<const T*>(p.b)[c]));
    };
    if (p.q == nullptr) {
        for (int c = threadIdx.x; c < p.N; c += kLongBlock) static_cast<T*>(p.y)[row * p.N + c] = from_float<T>(value(c));
        return;
    }
    float top = 0.0f;
    for (int c = threadIdx.x; c < p.N; c += kLongBlock) top = max_nan(top, fabsf(value(c)));
    const RowScale k = row_scale(row_max<0>(top, red[2]));
    if (threadIdx.x == 0) p.scale[row] = k.scale;
    for (int c = threadIdx.x; c < p.N; c += kLongBlock)
        p.q[row * p.qs + c] = quantise(value(c), k.inv);
}

template <typename T, int V, int P, int GROUP>
__global__ void __launch_bounds__(GROUP ? kBlock : backward_threads(V)) layer_norm_backward_kernel(const __grid_constant__ NormParams p)
{
    constexpr int E = P * V / 2;
    constexpr int kGroups = GROUP ? kBlock / (GROUP ? GROUP : 1) : 1;  // rows of a block at a time
    constexpr int kJoin = GROUP ? kBlock * P * V : 1;                  // values of a block's rows
    __shared__ float joined[kJoin];
    __shared__ float red[2][2][32];
    const int lanes = GROUP ? GROUP : static_cast<int>(blockDim.x), lane = GROUP ? threadIdx.x % GROUP : threadIdx.x;
    const int group = GROUP ? threadIdx.x / (GROUP ? GROUP : 1) : 0;
    Pair w[E], dw[E], db[E];
    {
        Piece<T, V> raw[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c = (i * lanes + lane) * V;
            raw[i].clear();
            if (p.w != nullptr && c < p.N) raw[i].load(static_cast<const T*>(p.w) + c);
        }
        values_of<T, V, P>(raw, w);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        dw[i] = db[i] = pair(0.0f, 0.0f);
        if (p.w == nullptr) w[i] = pair(1.0f, 1.0f);
    }
    // what lies beyond the row stays 0 in x and dy, and with it in every sum but xh (-mean rstd), which only meets zeros
    Piece<T, V> xr[P], gr[P];
    float mean = 0.0f, rstd = 0.0f;
    const auto load = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int c = (i * lanes + lane) * V;
            if (c < p.N) {
                xr[i].load(static_cast<const T*>(p.x) + row * p.xs + c);
                gr[i].load(static_cast<const T*>(p.dy) + row * p.gs + c);
            } else {
                xr[i].clear();
                gr[i].clear();
            }
        }
        mean = __ldg(p.mean + row);
        rstd = __ldg(p.rstd + row);
    };
    const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups, last = p.rows - 1;
    load(min(static_cast<int64_t>(blockIdx.x) * kGroups + group, last));
    int turn = 0;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups; base < p.rows; base += step, turn ^= 1) {
        const int64_t row = base + group;
        Pair xh[E], g[E];
        values_of<T, V, P>(xr, xh);
        values_of<T, V, P>(gr, g);
        const float rs = rstd;
        const Pair nm = pair(-mean, -mean), r2 = pair(rs, rs);
        if (base + step < p.rows) load(min(row + step, last));
        const bool real = row < p.rows;
        Pair s1 = pair(0.0f, 0.0f), s2 = s1;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            xh[i] = mul2(add2(xh[i], nm), r2);
            if (GROUP == 0 || real) {
                dw[i] = fma2(g[i], xh[i], dw[i]);
                db[i] = add2(db[i], g[i]);
            }
            g[i] = mul2(g[i], w[i]);
            s1 = add2(s1, g[i]);
            s2 = fma2(g[i], xh[i], s2);
        }
        const float m1 = row_sum<GROUP>(both(s1), red[turn][0]) * p.inv_n, m2 = row_sum<GROUP>(both(s2), red[turn][1]) * p.inv_n;
        const Pair a = pair(-m1, -m1), b = pair(-m2, -m2);
#pragma unroll
        for (int i = 0; i < E; ++i) g[i] = mul2(fma2(xh[i], b, add2(g[i], a)), r2);
        if (p.dsum != nullptr) {
            Piece<T, V> raw[P];
            Pair d[E];
            const T* from = static_cast<const T*>(p.dsum) + min(row, last) * p.ds;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int c = (i * lanes + lane) * V;
                raw[i].clear();
                if (c < p.N) raw[i].load(from + c);
            }
            values_of<T, V, P>(raw, d);
#pragma unroll
            for (int i = 0; i < E; ++i) g[i] = add2(g[i], d[i]);
        }
        if (real) {
            T* to = static_cast<T*>(p.dx) + row * p.N;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int c = (i * lanes + lane) * V;
                if (c < p.N) store_piece<T, V>(to + c, g, i);
            }
        }
    }
    if (p.part == nullptr) return;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* to = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + which) * p.N;
        float v[2 * E];
#pragma unroll
        for (int i = 0; i < E; ++i) unpair(which ? db[i] : dw[i], v[2 * i], v[2 * i + 1]);
        if constexpr (GROUP == 0) {
#pragma unroll
            for (int e = 0; e < 2 * E; ++e) {
                const int c = (e / V * lanes + lane) * V + e % V;
                if (c < p.N) to[c] = v[e];
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
                to[c] = s;
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

// Joins the blocks' sums: 32 columns a block, 32 warps over the parts.
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_join_kernel(const float* part, int parts, int N, T* dw, T* db)
{
    __shared__ float sums[32][33];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;  // of the 2 N
    wait_for_launches_before();
    float s = 0.0f;
    if (c < 2 * static_cast<int64_t>(N))
#pragma unroll 4
        for (int k = warp; k < parts; k += 32) s += part[static_cast<int64_t>(k) * 2 * N + c];
    sums[warp][lane] = s;
    __syncthreads();
    s = sums[lane][warp];
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    const int64_t to = static_cast<int64_t>(blockIdx.x) * 32 + warp;
    if (lane == 0 && to < 2 * static_cast<int64_t>(N)) {
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

NormParams params(const ww_layer_norm_t& p, bool norm) noexcept
{
    NormParams f{};
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

template <typename T>
int forward(const ww_layer_norm_t& p, bool norm, const char* name, cudaStream_t stream) noexcept
{
    const NormParams f = params(p, norm);
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    const bool pieces = in_pieces(p, sizeof(T));
    const RowForm form = row_form(p.N, pieces ? V : 1, 16, kForwardThreads);
    const unsigned groups = form.group ? kBlock / form.group : 1;
    const unsigned grid = static_cast<unsigned>((i64(p.rows) + groups - 1) / groups);
    const auto go = [&](auto kernel) { kernel<<<grid, form.threads, 0, stream>>>(f); };
    const int id = form.group * 100 + form.pieces;
    if (form.threads == 0) layer_norm_long_kernel<T><<<p.rows, kLongBlock, 0, stream>>>(f);
    else if (!pieces)
        switch (id) {
        case 3204: go(layer_norm_kernel<T, 1, 4, 32>); break;
        case 3216: go(layer_norm_kernel<T, 1, 16, 32>); break;
        case 4: go(layer_norm_kernel<T, 1, 4, 0>); break;
        default: go(layer_norm_kernel<T, 1, 16, 0>); break;
        }
    else
        switch (id) {
        case 401: go(layer_norm_kernel<T, V, 1, 4>); break;
        case 801: go(layer_norm_kernel<T, V, 1, 8>); break;
        case 1601: go(layer_norm_kernel<T, V, 1, 16>); break;
        case 1603: go(layer_norm_kernel<T, V, 3, 16>); break;
        case 3201: go(layer_norm_kernel<T, V, 1, 32>); break;
        case 3202: go(layer_norm_kernel<T, V, 2, 32>); break;
        case 3203: go(layer_norm_kernel<T, V, 3, 32>); break;
        case 3204: go(layer_norm_kernel<T, V, 4, 32>); break;
        case 2: go(layer_norm_kernel<T, V, 2, 0>); break;
        default: go(layer_norm_kernel<T, V, 4, 0>); break;
        }
    return launch_status(name);
}

// Blocks of the gradient: one resident round, as far as there are rows for it.
struct BackwardPlan {
    bool pieces;
    RowForm form;
    int blocks, splits;  // splits: of the rows, for the sums by columns (long rows)
    int parts() const { return form.threads == 0 ? splits : blocks; }
};

BackwardPlan backward_plan(const ww_layer_norm_t& p, int sms) noexcept
{
    const int bytes = p.dtype == WW_DTYPE_FLOAT ? 4 : 2;
    BackwardPlan r;
    r.pieces = in_pieces(p, bytes);
    const int v = r.pieces ? 16 / bytes : 1;
    r.form = row_form(p.N, v, r.pieces ? 3 : 16, backward_threads(v));
    const int groups = r.form.group ? kBlock / r.form.group : 1;
    const int resident = r.form.threads == 0 ? 1 : std::max(1, (r.form.pieces > 4 ? 768 : 1024) / r.form.threads);
    r.blocks = static_cast<int>(std::min<int64_t>(i64(sms) * resident, (i64(p.rows) + groups - 1) / groups));
    const int columns = (p.N + kBlock - 1) / kBlock;
    r.splits = std::max(1, std::min(p.rows, 4 * sms / columns));
    return r;
}

template <typename T>
int backward(const ww_layer_norm_t& p, const BackwardPlan& plan, cudaStream_t stream) noexcept
{
    NormParams f = params(p, true);
    const bool sums = p.dweight != nullptr;
    f.part = sums ? static_cast<float*>(p.workspace) : nullptr;
    constexpr int V = 16 / static_cast<int>(sizeof(T));
    const RowForm& form = plan.form;
    const auto go = [&](auto kernel) { kernel<<<plan.blocks, form.threads, 0, stream>>>(f); };
    const int id = form.group * 100 + form.pieces;
    if (form.threads == 0) {
        layer_norm_backward_long_kernel<T><<<p.rows, kLongBlock, 0, stream>>>(f);
        if (sums) layer_norm_columns_kernel<T><<<dim3((p.N + kBlock - 1) / kBlock, plan.splits), kBlock, 0, stream>>>(f);
    } else if (!plan.pieces) {
        switch (id) {
        case 3204: go(layer_norm_backward_kernel<T, 1, 4, 32>); break;
        case 3216: go(layer_norm_backward_kernel<T, 1, 16, 32>); break;
        case 4: go(layer_norm_backward_kernel<T, 1, 4, 0>); break;
        default: go(layer_norm_backward_kernel<T, 1, 16, 0>); break;
        }
    } else {
        switch (id) {
        case 401: go(layer_norm_backward_kernel<T, V, 1, 4>); break;
        case 801: go(layer_norm_backward_kernel<T, V, 1, 8>); break;
        case 1601: go(layer_norm_backward_kernel<T, V, 1, 16>); break;
        case 1603: go(layer_norm_backward_kernel<T, V, 3, 16>); break;
        case 3201: go(layer_norm_backward_kernel<T, V, 1, 32>); break;
        case 3202: go(layer_norm_backward_kernel<T, V, 2, 32>); break;
        case 3203: go(layer_norm_backward_kernel<T, V, 3, 32>); break;
        default: go(layer_norm_backward_kernel<T, V, 2, 0>); break;
        }
    }
    const int st = launch_status("layer_norm_backward");
    if (st != WW_SUCCESS || !sums) return st;
    launch_behind(layer_norm_join_kernel<T>, dim3((2u * p.N + 31) / 32), dim3(1024), 0, stream, f.part, plan.parts(), p.N,
                  static_cast<T*>(p.dweight), static_cast<T*>(p.dbias));
    return launch_status("layer_norm_backward");
}

// What both directions check; *go = false: nothing to do.
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
    return p.dtype == WW_DTYPE_HALF ? forward<__half>(p, norm, name, s)
         : p.dtype == WW_DTYPE_BF16 ? forward<__nv_bfloat16>(p, norm, name, s) : forward<float>(p, norm, name, s);
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
