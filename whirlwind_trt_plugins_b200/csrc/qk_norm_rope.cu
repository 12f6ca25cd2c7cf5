// qk_norm_rope.cu -- per-head RMS norm of queries and keys and the position
// rotation in the same pass, with its gradient.
//
//   r = rsqrt(mean_d x^2 + eps),  xh = x r,  y = xh w
//   (y1, y2) -> (y1 c - y2 s, y2 c + y1 s)        first R of D dims
//
// and backwards, with g the incoming gradient turned by the opposite angle:
//
//   dw = sum over rows of g xh,   u = g w,   dx = r (u - xh mean_d(u xh)).
//
// Bound: HBM (forward 2 values per element moved, backward 3; ~10 flops).
// That leaves about 16 instructions per value and lane, so the layout saves them:
// all (token, head) rows are one sequence, a row is a group of lanes, and a lane
// holds two pieces of V values that are each other's rotation partners (piece a of
// the first half, piece b of the second; for interleaved pairs each its own
// pairs): the rotation needs no exchange and both pieces share their angles.
// Neighbouring groups hold neighbouring rows, so that a warp's loads lie side by
// side; divisions by H and L are multiplies;
// arithmetic is two values an instruction.  cos and sin come from L1 (a token's
// heads are neighbours).  Queries and keys are one grid: one launch.
// The weight gradients stay in registers over all rows of a lane, are joined per
// block through shared memory and over blocks by a second small kernel, both in a
// fixed order: the same inputs give the same bits.
//
// Measured: rows of 16 pairs 94 x 312, 8 heads of 32, fp16, 961 MB: 158 us, 6.1
// TB/s; gradient of 8 x 1200 queries, 16 heads of 128, and 1777 keys, 4 heads, bf16,
// 162 MB: 38 + 4.5 us; of 120 rows of 160, 5 heads of 64, fp32, 147 MB: 23 + 4 us.
#include "attention.cuh"

#include <algorithm>
#include <cmath>

namespace ww {
namespace {

constexpr int kBlock = 256;
// Resident blocks asked of the compiler, one row of a lane in flight: more rows
// per lane cost registers and with them warps (rows of 16 pairs 94 x 312, fp16,
// 961 MB: 158 us; two rows and 4 blocks 180 us, four and 3 207 us, one and 8,
// which spills, 304 us).
constexpr int kForwardBlocks = 6;
constexpr int backward_blocks(int V) { return V == 8 ? 3 : 4; }
constexpr int kSms = 148;

struct Side {
    const void* x;
    const void* w;
    const int32_t* pos;
    const void* dout;  // backward
    void* y;           // forward: output; backward: dx
    void* dw;
    float* part;  // backward: [blocks][D] partial weight gradients
    int64_t sb, sl, sh, gb, gl, gh;
    Divisor L, H;
    int32_t x_linear, g_linear;  // rows follow one another without a gap
    int32_t pos_stride;
    int32_t rows;    // B * L * H
    int32_t blocks;  // grid blocks of this side
};

struct RopeParams {
    Side side[2];
    const float* cos;
    const float* sin;
    int32_t D, R, P;
    int32_t lanes;  // lanes of a group with pieces
    float eps, inv_d;
};

// V values of T as V / 2 pairs of fp32.
template <typename T, int V>
__device__ __forceinline__ void load(const T* p, Pair (&f)[V / 2])
{
    constexpr int kN = V * static_cast<int>(sizeof(T)) / 4;
    uint32_t w[kN];
    if constexpr (kN == 4) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = u.x;
        w[1] = u.y;
        w[2] = u.z;
        w[3] = u.w;
    } else {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
        w[0] = u.x;
        w[1] = u.y;
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        if constexpr (sizeof(T) == 4) {
            f[i] = pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[i] = pair(v.x, v.y);
        } else {
            f[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const Pair (&f)[V / 2])
{
    float v[V];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) unpair(f[i], v[2 * i], v[2 * i + 1]);
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else if constexpr (V == 8)
        *reinterpret_cast<uint4*>(p) =
            make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    else
        *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
}

// The two pieces of a lane: dims [a, a + V) and [b, b + V), and whether they
// rotate.  Lanes beyond the row hold its last pieces.
struct Pieces {
    int a, b;
    bool rotates;
};

template <int V>
__device__ __forceinline__ Pieces pieces_of(int lane, const RopeParams& p)
{
    Pieces r;
    const int l = min(lane, p.lanes - 1), n = p.R / (2 * V);
    r.rotates = l < n;
    r.a = r.rotates ? l * V : p.R + (l - n) * V;
    r.b = r.a + (r.rotates ? p.R / 2 : (p.D - p.R) / 2);
    return r;
}

// cos and sin of the two pieces: V angles that both share, or (interleaved) V / 2
// for each, a's first; as pairs (INTER: as values).
template <int V, bool INTER>
struct Angles {
    float c[V], s[V];
    __device__ __forceinline__ void get(const RopeParams& p, int pos, const Pieces& x)
    {
        if (!x.rotates) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                c[i] = 1.0f;
                s[i] = 0.0f;
            }
            return;
        }
        const int64_t row = static_cast<int64_t>(pos) * (p.R / 2);
        if (INTER) {
            part(p, row + x.a / 2, 0);
            part(p, row + x.b / 2, V / 2);
        } else {
            part(p, row + x.a, 0);
            part(p, row + x.a + V / 2, V / 2);
        }
    }
    // V / 2 angles from `at` to place i
    __device__ __forceinline__ void part(const RopeParams& p, int64_t at, int i)
    {
        if constexpr (V == 8) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p.cos + at)), b = __ldg(reinterpret_cast<const float4*>(p.sin + at));
            c[i] = a.x;
            c[i + 1] = a.y;
            c[i + 2] = a.z;
            c[i + 3] = a.w;
            s[i] = b.x;
            s[i + 1] = b.y;
            s[i + 2] = b.z;
            s[i + 3] = b.w;
        } else {
            const float2 a = __ldg(reinterpret_cast<const float2*>(p.cos + at)), b = __ldg(reinterpret_cast<const float2*>(p.sin + at));
            c[i] = a.x;
            c[i + 1] = a.y;
            s[i] = b.x;
            s[i + 1] = b.y;
        }
    }
    // both pieces turned by the angle (DIR 1) or back (-1)
    template <int DIR>
    __device__ __forceinline__ void turn(Pair (&x)[V / 2], Pair (&y)[V / 2]) const
    {
        if (INTER) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                float u, v;
                unpair(x[i], u, v);
                x[i] = pair(u * c[i] - v * (DIR * s[i]), v * c[i] + u * (DIR * s[i]));
                unpair(y[i], u, v);
                y[i] = pair(u * c[V / 2 + i] - v * (DIR * s[V / 2 + i]), v * c[V / 2 + i] + u * (DIR * s[V / 2 + i]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const Pair cc = pair(c[2 * i], c[2 * i + 1]), ss = pair(DIR * s[2 * i], DIR * s[2 * i + 1]),
                           ns = pair(-DIR * s[2 * i], -DIR * s[2 * i + 1]);
                const Pair u = x[i];
                x[i] = fma2(y[i], ns, mul2(u, cc));
                y[i] = fma2(u, ss, mul2(y[i], cc));
            }
        }
    }
};

template <int GROUP>
__device__ __forceinline__ float group_sum(float v)
{
#pragma unroll
    for (int o = GROUP / 2; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

__device__ __forceinline__ float both(Pair p)
{
    float a, b;
    unpair(p, a, b);
    return a + b;
}

// Batch item, token and head of a row.
struct RowAt {
    int b, l, h;
    __device__ __forceinline__ RowAt(const Side& s, int row)
    {
        const int token = s.H.div(row);
        h = row - token * s.H.d;
        b = s.L.div(token);
        l = token - b * s.L.d;
    }
};

__device__ __forceinline__ int position(const RopeParams& p, const Side& s, const RowAt& at)
{
    const int pos = s.pos != nullptr ? __ldg(s.pos + static_cast<int64_t>(at.b) * s.pos_stride + at.l) : at.l;
    return min(max(pos, 0), p.P - 1);
}

__device__ __forceinline__ int64_t offset(bool linear, int D, int row, const RowAt& at, int64_t sb, int64_t sl, int64_t sh)
{
    return linear ? static_cast<int64_t>(row) * D : at.b * sb + at.l * sl + at.h * sh;
}

template <typename T, int V, int GROUP, bool INTER>
__global__ void __launch_bounds__(kBlock, kForwardBlocks) qk_norm_rope_kernel(const __grid_constant__ RopeParams p)
{
    const bool second = static_cast<int>(blockIdx.x) >= p.side[0].blocks;
    const Side& s = p.side[second ? 1 : 0];
    const int block = blockIdx.x - (second ? p.side[0].blocks : 0);
    const int lane = threadIdx.x % GROUP;
    constexpr int kStep = kBlock / GROUP;  // rows of a block at a time
    const int row = block * kStep + threadIdx.x / GROUP;
    const Pieces pc = pieces_of<V>(lane, p);
    const int known = min(row, s.rows - 1);
    const RowAt at(s, known);
    const T* x = static_cast<const T*>(s.x) + offset(s.x_linear, p.D, known, at, s.sb, s.sl, s.sh);
    Pair xa[V / 2], xb[V / 2], wa[V / 2], wb[V / 2];
    load<T, V>(x + pc.a, xa);
    load<T, V>(x + pc.b, xb);
    load<T, V>(static_cast<const T*>(s.w) + pc.a, wa);
    load<T, V>(static_cast<const T*>(s.w) + pc.b, wb);
    Pair sq = mul2(xa[0], xa[0]);
#pragma unroll
    for (int i = 1; i < V / 2; ++i) sq = fma2(xa[i], xa[i], sq);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) sq = fma2(xb[i], xb[i], sq);
    const float r = rsqrtf(fmaf(group_sum<GROUP>(lane < p.lanes ? both(sq) : 0.0f), p.inv_d, p.eps));
    const Pair r2 = pair(r, r);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        xa[i] = mul2(xa[i], mul2(r2, wa[i]));
        xb[i] = mul2(xb[i], mul2(r2, wb[i]));
    }
    Angles<V, INTER> ang;
    ang.get(p, p.R > 0 ? position(p, s, at) : 0, pc);
    ang.template turn<1>(xa, xb);
    if (row < s.rows && lane < p.lanes) {
        T* y = static_cast<T*>(s.y) + static_cast<int64_t>(row) * p.D;
        store<T, V>(y + pc.a, xa);
        store<T, V>(y + pc.b, xb);
    }
}

template <typename T, int V, int GROUP, bool INTER>
__global__ void __launch_bounds__(kBlock, backward_blocks(V)) qk_norm_rope_backward_kernel(const __grid_constant__ RopeParams p)
{
    __shared__ float joined[kBlock * 2 * V];
    const bool second = static_cast<int>(blockIdx.x) >= p.side[0].blocks;
    const Side& s = p.side[second ? 1 : 0];
    const int block = blockIdx.x - (second ? p.side[0].blocks : 0);
    const int lane = threadIdx.x % GROUP;
    constexpr int kStep = kBlock / GROUP;
    const Pieces pc = pieces_of<V>(lane, p);
    Pair wa[V / 2], wb[V / 2], da[V / 2], db[V / 2];
    load<T, V>(static_cast<const T*>(s.w) + pc.a, wa);
    load<T, V>(static_cast<const T*>(s.w) + pc.b, wb);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) da[i] = db[i] = pair(0.0f, 0.0f);
    // every lane makes the same number of rounds (the sums are warp-wide shuffles)
    const int stride = s.blocks * kStep;
    for (int base = 0; base < s.rows; base += stride) {
        const int row = base + block * kStep + threadIdx.x / GROUP, known = min(row, s.rows - 1);
        const RowAt at(s, known);
        const T* x = static_cast<const T*>(s.x) + offset(s.x_linear, p.D, known, at, s.sb, s.sl, s.sh);
        const T* g = static_cast<const T*>(s.dout) + offset(s.g_linear, p.D, known, at, s.gb, s.gl, s.gh);
        Pair xa[V / 2], xb[V / 2], ga[V / 2], gb[V / 2];
        load<T, V>(x + pc.a, xa);
        load<T, V>(x + pc.b, xb);
        load<T, V>(g + pc.a, ga);
        load<T, V>(g + pc.b, gb);
        Angles<V, INTER> ang;
        ang.get(p, p.R > 0 ? position(p, s, at) : 0, pc);
        ang.template turn<-1>(ga, gb);
        Pair sq = mul2(xa[0], xa[0]), dot = mul2(mul2(ga[0], wa[0]), xa[0]);
#pragma unroll
        for (int i = 1; i < V / 2; ++i) {
            sq = fma2(xa[i], xa[i], sq);
            dot = fma2(mul2(ga[i], wa[i]), xa[i], dot);
        }
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            sq = fma2(xb[i], xb[i], sq);
            dot = fma2(mul2(gb[i], wb[i]), xb[i], dot);
        }
        const float r = rsqrtf(fmaf(group_sum<GROUP>(lane < p.lanes ? both(sq) : 0.0f), p.inv_d, p.eps));
        const float m = group_sum<GROUP>(lane < p.lanes ? both(dot) : 0.0f) * r * r * p.inv_d;  // mean(u xh) r, applied to x
        if (row < s.rows && lane < p.lanes) {
            const Pair r2 = pair(r, r), nm = pair(-m, -m);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                da[i] = fma2(ga[i], mul2(xa[i], r2), da[i]);
                db[i] = fma2(gb[i], mul2(xb[i], r2), db[i]);
                ga[i] = mul2(r2, fma2(xa[i], nm, mul2(ga[i], wa[i])));
                gb[i] = mul2(r2, fma2(xb[i], nm, mul2(gb[i], wb[i])));
            }
            T* y = static_cast<T*>(s.y) + static_cast<int64_t>(row) * p.D;
            store<T, V>(y + pc.a, ga);
            store<T, V>(y + pc.b, gb);
        }
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        unpair(da[i], joined[threadIdx.x * 2 * V + 2 * i], joined[threadIdx.x * 2 * V + 2 * i + 1]);
        unpair(db[i], joined[threadIdx.x * 2 * V + V + 2 * i], joined[threadIdx.x * 2 * V + V + 2 * i + 1]);
    }
    __syncthreads();
    // one thread per value of the lanes: the groups' sums in order
    for (int t = threadIdx.x; t < p.lanes * 2 * V; t += kBlock) {
        const int ln = t / (2 * V), i = t - ln * 2 * V;
        float sum = 0.0f;
        for (int n = 0; n < kStep; ++n) sum += joined[(n * GROUP + ln) * 2 * V + i];
        const Pieces x = pieces_of<V>(ln, p);
        s.part[static_cast<int64_t>(block) * p.D + (i < V ? x.a + i : x.b + i - V)] = sum;
    }
}

// Joins the blocks' weight gradients: 32 dims per CTA, each of 32 warps takes
// every 32nd block's row (eight loads in flight), then the warps' sums in order.
template <typename T>
__global__ void __launch_bounds__(1024) weight_gradient_kernel(const __grid_constant__ RopeParams p)
{
    __shared__ float sums[32][33];
    const Side& s = p.side[blockIdx.y];
    const int d = blockIdx.x * 32 + threadIdx.x % 32, w = threadIdx.x / 32;
    wait_for_launches_before();
    float sum = 0.0f;
    if (d < p.D) {
#pragma unroll 8
        for (int n = w; n < s.blocks; n += 32) sum += s.part[static_cast<int64_t>(n) * p.D + d];
    }
    sums[w][threadIdx.x % 32] = sum;
    __syncthreads();
    if (w == 0 && d < p.D) {
        sum = 0.0f;
#pragma unroll
        for (int n = 0; n < 32; ++n) sum += sums[n][threadIdx.x];
        static_cast<T*>(s.dw)[d] = from_float<T>(sum);
    }
}

int elem_size(int dtype) { return dtype == WW_DTYPE_FLOAT ? 4 : 2; }

int check(const ww_qk_norm_rope_t& p, bool backward) noexcept
{
    if (p.dtype != WW_DTYPE_HALF && p.dtype != WW_DTYPE_BF16 && p.dtype != WW_DTYPE_FLOAT) return WW_ERR_INVALID_DTYPE;
    if (p.B < 0 || p.Lq < 0 || p.Lk < 0 || p.Hq <= 0 || p.Hk <= 0 || p.D <= 0) return WW_ERR_INVALID_SHAPE;
    if (p.R < 0 || p.R > p.D || p.R % 2 != 0 || p.P < 0 || !(p.eps >= 0.0f)) return WW_ERR_INVALID_SHAPE;
    if (p.q_pos_stride < 0 || p.k_pos_stride < 0) return WW_ERR_INVALID_SHAPE;
    if (p.D % 8 != 0 || p.R % 8 != 0 || p.D > 256) return WW_ERR_UNSUPPORTED;
    const int64_t lim = int64_t{1} << 30;  // rows and one grid step beyond them in 32 bits
    const int64_t nq = i64(p.B) * p.Lq, nk = i64(p.B) * p.Lk;
    if (nq > lim || nk > lim || nq * (p.Hq) > lim || nk * (p.Hk) > lim)
        return WW_ERR_UNSUPPORTED;
    const bool any = nq > 0 || nk > 0;
    if (p.R > 0 && any && (p.P == 0 || p.cos == nullptr || p.sin == nullptr))
        return p.P == 0 ? WW_ERR_INVALID_SHAPE : WW_ERR_NULL_POINTER;
    const int es = elem_size(p.dtype);
    const auto off = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 != 0; };
    if (any && (off(p.cos) || off(p.sin))) return WW_ERR_MISALIGNED;
    if (nq > 0) {
        if (p.q == nullptr || p.q_weight == nullptr || (backward ? p.dq == nullptr || p.dq_out == nullptr : p.q_out == nullptr))
            return WW_ERR_NULL_POINTER;
        if (!vectors_ok(p.q, p.q_strides, p.B, p.Lq, p.Hq, es) || off(p.q_weight) || off(backward ? p.dq : p.q_out) ||
            (backward && !vectors_ok(p.dq_out, p.dq_out_strides, p.B, p.Lq, p.Hq, es)))
            return WW_ERR_MISALIGNED;
    }
    if (nk > 0) {
        if (p.k == nullptr || p.k_weight == nullptr || (backward ? p.dk == nullptr || p.dk_out == nullptr : p.k_out == nullptr))
            return WW_ERR_NULL_POINTER;
        if (!vectors_ok(p.k, p.k_strides, p.B, p.Lk, p.Hk, es) || off(p.k_weight) || off(backward ? p.dk : p.k_out) ||
            (backward && !vectors_ok(p.dk_out, p.dk_out_strides, p.B, p.Lk, p.Hk, es)))
            return WW_ERR_MISALIGNED;
    }
    if (backward && (p.dq_weight == nullptr || p.dk_weight == nullptr)) return WW_ERR_NULL_POINTER;
    return WW_SUCCESS;
}

// Values of a lane's piece: 8 of 16 bits where both halves split into them, else 4.
int piece_values(const ww_qk_norm_rope_t& p)
{
    if (p.dtype == WW_DTYPE_FLOAT) return 4;
    return p.R % 16 == 0 && p.D % 16 == 0 ? 8 : 4;
}

// Lanes of a row: the power of two that holds its pieces, two a lane.
int group_lanes(const ww_qk_norm_rope_t& p)
{
    const int lanes = p.D / (2 * piece_values(p));
    int g = 1;
    while (g < lanes) g *= 2;
    return g;
}

void fill(const ww_qk_norm_rope_t& p, bool backward, RopeParams* out) noexcept
{
    RopeParams& r = *out;
    r.cos = p.cos;
    r.sin = p.sin;
    r.D = p.D;
    r.R = p.R;
    r.P = p.P;
    r.eps = p.eps;
    r.inv_d = 1.0f / p.D;
    r.lanes = p.D / (2 * piece_values(p));
    const int per_block = kBlock / group_lanes(p);
    for (int i = 0; i < 2; ++i) {
        Side& s = r.side[i];
        const int64_t* st = i ? p.k_strides : p.q_strides;
        const int64_t* gs = i ? p.dk_out_strides : p.dq_out_strides;
        s.x = i ? p.k : p.q;
        s.w = i ? p.k_weight : p.q_weight;
        s.pos = i ? p.k_pos : p.q_pos;
        s.dout = i ? p.dk_out : p.dq_out;
        s.y = backward ? (i ? p.dk : p.dq) : (i ? p.k_out : p.q_out);
        s.dw = i ? p.dk_weight : p.dq_weight;
        s.sb = st[0]; s.sl = st[1]; s.sh = st[2];
        s.gb = gs[0]; s.gl = gs[1]; s.gh = gs[2];
        s.pos_stride = i ? p.k_pos_stride : p.q_pos_stride;
        const int L = i ? p.Lk : p.Lq, H = i ? p.Hk : p.Hq;
        s.L = make_divisor(L > 0 ? L : 1);
        s.H = make_divisor(H);
        // strides of dims with one element do not matter
        const auto linear = [&](int64_t sb, int64_t sl, int64_t sh) {
            return (H == 1 || sh == p.D) && (L == 1 || sl == i64(H) * p.D) && (p.B == 1 || sb == i64(L) * H * p.D);
        };
        s.x_linear = linear(s.sb, s.sl, s.sh);
        s.g_linear = linear(s.gb, s.gl, s.gh);
        s.rows = static_cast<int32_t>(i64(p.B) * L * H);
        s.blocks = (s.rows + per_block - 1) / per_block;
    }
    if (backward) {
        // one round of resident blocks, shared between the sides by their rows
        const int all = kSms * backward_blocks(piece_values(p));
        const int64_t total = i64(r.side[0].rows) + r.side[1].rows;
        for (Side& s : r.side)
            if (s.rows > 0)
                s.blocks = static_cast<int>(std::min<int64_t>(s.blocks, std::max<int64_t>(1, all * i64(s.rows) / total)));
    }
    r.side[0].part = static_cast<float*>(p.workspace);
    r.side[1].part = r.side[0].part + static_cast<int64_t>(r.side[0].blocks) * p.D;
}

template <typename T, int V, int GROUP>
int launch(const RopeParams& r, bool inter, bool backward, cudaStream_t stream) noexcept
{
    const int blocks = r.side[0].blocks + r.side[1].blocks;
    if (blocks > 0) {
        if (!backward) {
            if (inter) qk_norm_rope_kernel<T, V, GROUP, true><<<blocks, kBlock, 0, stream>>>(r);
            else qk_norm_rope_kernel<T, V, GROUP, false><<<blocks, kBlock, 0, stream>>>(r);
        } else {
            if (inter) qk_norm_rope_backward_kernel<T, V, GROUP, true><<<blocks, kBlock, 0, stream>>>(r);
            else qk_norm_rope_backward_kernel<T, V, GROUP, false><<<blocks, kBlock, 0, stream>>>(r);
        }
    }
    if (backward) launch_behind(weight_gradient_kernel<T>, dim3((r.D + 31) / 32, 2), dim3(1024), 0, stream, r);
    return launch_status(backward ? "qk_norm_rope_backward" : "qk_norm_rope");
}

template <typename T, int V>
int launch_group(const RopeParams& r, int group, bool inter, bool backward, cudaStream_t stream) noexcept
{
    switch (group) {
        case 1: return launch<T, V, 1>(r, inter, backward, stream);
        case 2: return launch<T, V, 2>(r, inter, backward, stream);
        case 4: return launch<T, V, 4>(r, inter, backward, stream);
        case 8: return launch<T, V, 8>(r, inter, backward, stream);
        case 16: return launch<T, V, 16>(r, inter, backward, stream);
        default: return launch<T, V, 32>(r, inter, backward, stream);
    }
}

template <typename T>
int launch_type(const ww_qk_norm_rope_t& p, bool backward, cudaStream_t stream) noexcept
{
    RopeParams r;
    fill(p, backward, &r);
    const int group = group_lanes(p);
    if constexpr (sizeof(T) == 2)
        if (piece_values(p) == 8) return launch_group<T, 8>(r, group, p.interleaved != 0, backward, stream);
    return launch_group<T, 4>(r, group, p.interleaved != 0, backward, stream);
}

int64_t workspace(const ww_qk_norm_rope_t& p) noexcept
{
    RopeParams r;
    fill(p, true, &r);
    return static_cast<int64_t>(r.side[0].blocks + r.side[1].blocks) * p.D * 4;
}

int entry(const ww_qk_norm_rope_t* p, bool backward, void* stream) noexcept
{
    if (p == nullptr) return WW_ERR_NULL_POINTER;
    int st = check(*p, backward);
    if (st != WW_SUCCESS) return st;
    if (!backward && (p->B == 0 || (p->Lq == 0 && p->Lk == 0))) return WW_SUCCESS;
    if (backward) {
        const int64_t need = workspace(*p);
        if (need > 0 && p->workspace == nullptr) return WW_ERR_NULL_POINTER;
        if (need > p->workspace_bytes) return WW_ERR_UNSUPPORTED;
        if (reinterpret_cast<uintptr_t>(p->workspace) % 16 != 0) return WW_ERR_MISALIGNED;
    }
    DeviceInfo d;
    if ((st = current_device_info(&d)) != WW_SUCCESS) return st;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (p->dtype == WW_DTYPE_HALF) return launch_type<__half>(*p, backward, s);
    if (p->dtype == WW_DTYPE_BF16) return launch_type<__nv_bfloat16>(*p, backward, s);
    return launch_type<float>(*p, backward, s);
}

}  // namespace
}  // namespace ww

extern "C" {

int ww_qk_norm_rope(const ww_qk_norm_rope_t* p, void* stream) { return ww::entry(p, false, stream); }

int ww_qk_norm_rope_backward(const ww_qk_norm_rope_t* p, void* stream) { return ww::entry(p, true, stream); }

int64_t ww_qk_norm_rope_backward_workspace(const ww_qk_norm_rope_t* p)
{
    if (p == nullptr || ww::check(*p, true) != WW_SUCCESS) return 0;
    return ww::workspace(*p);
}

}  // extern "C"
