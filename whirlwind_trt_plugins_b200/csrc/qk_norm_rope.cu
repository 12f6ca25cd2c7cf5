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
// Layout: a group of lanes owns a token's head; each lane holds two chunks of
// V consecutive dims whose members are rotation partners of one another
// (chunk a of the first half, chunk b of the second; for interleaved pairs
// each chunk holds its own pairs), so the rotation needs no exchange and the
// only shuffles are the group's sums.  A group takes kHeads heads of one token
// at once: their loads are in flight together and the token's cos and sin are
// read once.  Queries and keys are one grid: one launch.
// The weight gradients stay in registers over all tokens of a group, are
// joined per block through shared memory and over blocks by a second small
// kernel, both in a fixed order: the same inputs give the same bits.
#include "attention.cuh"

#include <cmath>

namespace ww {
namespace {

constexpr int kBlock = 256;
constexpr int kHeads = 4;
constexpr int kMaxPartBlocks = 296;  // backward: two blocks of each of 148 SMs per side

struct Side {
    const void* x;
    const void* w;
    const int32_t* pos;
    const void* dout;  // backward
    void* y;           // forward: output; backward: dx
    void* dw;
    float* part;  // backward: [blocks][D] partial weight gradients
    int64_t sb, sl, sh, gb, gl, gh;
    int32_t pos_stride;
    int32_t L, H;
    int32_t chunks;   // head chunks of kHeads per token
    int32_t items;    // B * L * chunks
    int32_t blocks;   // grid blocks of this side
};

struct RopeParams {
    Side side[2];
    const float* cos;
    const float* sin;
    int32_t D, R, P;
    int32_t lanes;  // lanes with work in a group
    float eps;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&f)[V])
{
    const Vec<T, V> u = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_float(u.v[i]);
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&f)[V])
{
    Vec<T, V> u;
#pragma unroll
    for (int i = 0; i < V; ++i) u.v[i] = from_float<T>(f[i]);
    *reinterpret_cast<Vec<T, V>*>(p) = u;
}

// The two chunks of lane l: dims [a, a + V) and [b, b + V), and whether they rotate.
template <int V>
__device__ __forceinline__ void chunk_dims(int l, int D, int R, int& a, int& b, bool& rot)
{
    const int nr = R / (2 * V);
    rot = l < nr;
    if (rot) {
        a = l * V;
        b = R / 2 + a;
    } else {
        a = R + (l - nr) * V;
        b = a + (D - R) / 2;
    }
}

// Angles of one lane: V per chunk.  Pairs (i, i + R/2): both chunks share the
// V angles from a; interleaved: V/2 angles for each chunk.
template <int V, bool INTER>
struct Angles {
    float ca[V], sa[V];  // INTER: first V/2 for chunk a, the others for chunk b
    __device__ __forceinline__ void get(const float* cos, const float* sin, int64_t row, int a, int b)
    {
        if (INTER) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                ca[i] = __ldg(cos + row + a / 2 + i);
                sa[i] = __ldg(sin + row + a / 2 + i);
                ca[V / 2 + i] = __ldg(cos + row + b / 2 + i);
                sa[V / 2 + i] = __ldg(sin + row + b / 2 + i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                ca[i] = __ldg(cos + row + a + i);
                sa[i] = __ldg(sin + row + a + i);
            }
        }
    }
    __device__ __forceinline__ void none()
    {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            ca[i] = 1.0f;
            sa[i] = 0.0f;
        }
    }
    // turn by the angle (dir = 1) or back (dir = -1)
    template <int DIR>
    __device__ __forceinline__ void turn(float (&x)[V], float (&y)[V]) const
    {
        if (INTER) {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float s0 = DIR * sa[i], s1 = DIR * sa[V / 2 + i];
                const float p = x[2 * i], q = x[2 * i + 1];
                x[2 * i] = p * ca[i] - q * s0;
                x[2 * i + 1] = q * ca[i] + p * s0;
                const float u = y[2 * i], v = y[2 * i + 1];
                y[2 * i] = u * ca[V / 2 + i] - v * s1;
                y[2 * i + 1] = v * ca[V / 2 + i] + u * s1;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float p = x[i], q = y[i], s = DIR * sa[i];
                x[i] = p * ca[i] - q * s;
                y[i] = q * ca[i] + p * s;
            }
        }
    }
};

template <int GROUP>
__device__ __forceinline__ float group_sum(float v)
{
#pragma unroll
    for (int o = GROUP / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ int position(const RopeParams& p, const Side& s, int b, int l)
{
    const int at = s.pos != nullptr ? __ldg(s.pos + static_cast<int64_t>(b) * s.pos_stride + l) : l;
    return min(max(at, 0), p.P - 1);
}

template <typename T, int V, int GROUP, bool INTER>
__global__ void __launch_bounds__(kBlock) qk_norm_rope_kernel(const __grid_constant__ RopeParams p)
{
    const bool second = static_cast<int>(blockIdx.x) >= p.side[0].blocks;
    const Side& s = p.side[second ? 1 : 0];
    const int block = blockIdx.x - (second ? p.side[0].blocks : 0);
    const int item = block * (kBlock / GROUP) + threadIdx.x / GROUP;
    const int lane = threadIdx.x % GROUP;
    const bool live = item < s.items && lane < p.lanes;
    const int it = min(item, s.items - 1);
    const int token = it / s.chunks;
    const int h0 = (it - token * s.chunks) * kHeads;
    const int b = token / s.L, l = token - b * s.L;
    int a, c;
    bool rot;
    chunk_dims<V>(min(lane, p.lanes - 1), p.D, p.R, a, c, rot);

    const T* x = static_cast<const T*>(s.x) + b * s.sb + l * s.sl;
    T* y = static_cast<T*>(s.y) + (static_cast<int64_t>(token) * s.H) * p.D;
    float xa[kHeads][V], xc[kHeads][V];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
        const int h = min(h0 + j, s.H - 1);
        load<T, V>(x + h * s.sh + a, xa[j]);
        load<T, V>(x + h * s.sh + c, xc[j]);
    }
    Angles<V, INTER> ang;
    if (rot) ang.get(p.cos, p.sin, static_cast<int64_t>(position(p, s, b, l)) * (p.R / 2), a, c);
    else ang.none();
    float wa[V], wc[V];
    load<T, V>(static_cast<const T*>(s.w) + a, wa);
    load<T, V>(static_cast<const T*>(s.w) + c, wc);
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) sq += xa[j][i] * xa[j][i] + xc[j][i] * xc[j][i];
        sq = group_sum<GROUP>(lane < p.lanes ? sq : 0.0f);
        const float r = rsqrtf(sq / p.D + p.eps);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            xa[j][i] *= r * wa[i];
            xc[j][i] *= r * wc[i];
        }
        ang.template turn<1>(xa[j], xc[j]);
        if (live && h0 + j < s.H) {
            store<T, V>(y + static_cast<int64_t>(h0 + j) * p.D + a, xa[j]);
            store<T, V>(y + static_cast<int64_t>(h0 + j) * p.D + c, xc[j]);
        }
    }
}

template <typename T, int V, int GROUP, bool INTER>
__global__ void __launch_bounds__(kBlock) qk_norm_rope_backward_kernel(const __grid_constant__ RopeParams p)
{
    __shared__ float joined[kBlock * 2 * V];
    const bool second = static_cast<int>(blockIdx.x) >= p.side[0].blocks;
    const Side& s = p.side[second ? 1 : 0];
    const int block = blockIdx.x - (second ? p.side[0].blocks : 0);
    const int lane = threadIdx.x % GROUP;
    int a, c;
    bool rot;
    chunk_dims<V>(min(lane, p.lanes - 1), p.D, p.R, a, c, rot);
    float wa[V], wc[V], da[V], dc[V];
    load<T, V>(static_cast<const T*>(s.w) + a, wa);
    load<T, V>(static_cast<const T*>(s.w) + c, wc);
#pragma unroll
    for (int i = 0; i < V; ++i) da[i] = dc[i] = 0.0f;

    const int step = s.blocks * (kBlock / GROUP);
    // every group of a warp makes the same number of rounds (the sums are warp-wide shuffles)
    const int first = block * (kBlock / GROUP) + threadIdx.x / GROUP;
    const int rounds = (s.items + step - 1) / step;
    for (int n = 0; n < rounds; ++n) {
        const int item = first + n * step;
        const int it = min(item, s.items - 1);
        const int token = it / s.chunks;
        const int h0 = (it - token * s.chunks) * kHeads;
        const int b = token / s.L, l = token - b * s.L;
        const T* x = static_cast<const T*>(s.x) + b * s.sb + l * s.sl;
        const T* g = static_cast<const T*>(s.dout) + b * s.gb + l * s.gl;
        T* y = static_cast<T*>(s.y) + (static_cast<int64_t>(token) * s.H) * p.D;
        Angles<V, INTER> ang;
        if (rot) ang.get(p.cos, p.sin, static_cast<int64_t>(position(p, s, b, l)) * (p.R / 2), a, c);
        else ang.none();
        constexpr int kPair = 2;  // heads in flight
        for (int j0 = 0; j0 < kHeads; j0 += kPair) {
            float xa[kPair][V], xc[kPair][V], ga[kPair][V], gc[kPair][V];
#pragma unroll
            for (int j = 0; j < kPair; ++j) {
                const int h = min(h0 + j0 + j, s.H - 1);
                load<T, V>(x + h * s.sh + a, xa[j]);
                load<T, V>(x + h * s.sh + c, xc[j]);
                load<T, V>(g + h * s.gh + a, ga[j]);
                load<T, V>(g + h * s.gh + c, gc[j]);
            }
#pragma unroll
            for (int j = 0; j < kPair; ++j) {
                const bool live = item < s.items && lane < p.lanes && h0 + j0 + j < s.H;
                ang.template turn<-1>(ga[j], gc[j]);
                float sq = 0.0f, dot = 0.0f;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    sq += xa[j][i] * xa[j][i] + xc[j][i] * xc[j][i];
                    dot += ga[j][i] * wa[i] * xa[j][i] + gc[j][i] * wc[i] * xc[j][i];
                }
                sq = group_sum<GROUP>(lane < p.lanes ? sq : 0.0f);
                dot = group_sum<GROUP>(lane < p.lanes ? dot : 0.0f);
                const float r = rsqrtf(sq / p.D + p.eps);
                const float m = dot * r * r / p.D;  // mean(u xh) r, applied to x
                if (live) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        da[i] += ga[j][i] * (xa[j][i] * r);
                        dc[i] += gc[j][i] * (xc[j][i] * r);
                        ga[j][i] = r * (ga[j][i] * wa[i] - xa[j][i] * m);
                        gc[j][i] = r * (gc[j][i] * wc[i] - xc[j][i] * m);
                    }
                    store<T, V>(y + static_cast<int64_t>(h0 + j0 + j) * p.D + a, ga[j]);
                    store<T, V>(y + static_cast<int64_t>(h0 + j0 + j) * p.D + c, gc[j]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        joined[threadIdx.x * 2 * V + i] = da[i];
        joined[threadIdx.x * 2 * V + V + i] = dc[i];
    }
    __syncthreads();
    // one thread per (lane, value): the groups' partials in order
    for (int t = threadIdx.x; t < p.lanes * 2 * V; t += kBlock) {
        const int ln = t / (2 * V), i = t - ln * 2 * V;
        float sum = 0.0f;
        for (int gidx = 0; gidx < kBlock / GROUP; ++gidx) sum += joined[(gidx * GROUP + ln) * 2 * V + i];
        int la, lc;
        bool lrot;
        chunk_dims<V>(ln, p.D, p.R, la, lc, lrot);
        s.part[static_cast<int64_t>(block) * p.D + (i < V ? la + i : lc + i - V)] = sum;
    }
}

// Joins the blocks' weight gradients: one block per side, kBlock / 32 warps
// each take every 8th block's row, then the warps' sums in order.
template <typename T>
__global__ void __launch_bounds__(kBlock) weight_gradient_kernel(const __grid_constant__ RopeParams p)
{
    __shared__ float sums[kBlock / 32][32];
    const Side& s = p.side[blockIdx.y];
    const int d = blockIdx.x * 32 + threadIdx.x % 32, w = threadIdx.x / 32;
    wait_for_launches_before();
    float sum = 0.0f;
    if (d < p.D)
        for (int n = w; n < s.blocks; n += kBlock / 32) sum += s.part[static_cast<int64_t>(n) * p.D + d];
    sums[w][threadIdx.x % 32] = sum;
    __syncthreads();
    if (w == 0 && d < p.D) {
        sum = 0.0f;
#pragma unroll
        for (int n = 0; n < kBlock / 32; ++n) sum += sums[n][threadIdx.x];
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
    const int64_t lim = int64_t{1} << 30;  // items and one grid step beyond them in 32 bits
    const int64_t nq = i64(p.B) * p.Lq, nk = i64(p.B) * p.Lk;
    if (nq > lim || nk > lim || nq * ((p.Hq + kHeads - 1) / kHeads) > lim || nk * ((p.Hk + kHeads - 1) / kHeads) > lim)
        return WW_ERR_UNSUPPORTED;
    const bool any = nq > 0 || nk > 0;
    if (p.R > 0 && any && (p.P == 0 || p.cos == nullptr || p.sin == nullptr))
        return p.P == 0 ? WW_ERR_INVALID_SHAPE : WW_ERR_NULL_POINTER;
    const int es = elem_size(p.dtype);
    const auto off = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 != 0; };
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

// Dims per lane and chunk: 16-byte loads where both halves split into them,
// else 4 values.  Lanes per head are then D / (2 V).
int chunk_values(const ww_qk_norm_rope_t& p)
{
    if (p.dtype == WW_DTYPE_FLOAT) return 4;
    return p.R % 16 == 0 && p.D % 16 == 0 ? 8 : 4;
}

int group_lanes(const ww_qk_norm_rope_t& p)
{
    const int lanes = p.D / (2 * chunk_values(p));
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
    r.lanes = p.D / (2 * chunk_values(p));
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
        s.L = i ? p.Lk : p.Lq;
        s.H = i ? p.Hk : p.Hq;
        s.chunks = (s.H + kHeads - 1) / kHeads;
        s.items = static_cast<int32_t>(i64(p.B) * s.L * s.chunks);
        const int need = (s.items + per_block - 1) / per_block;
        s.blocks = backward ? (need < kMaxPartBlocks ? need : kMaxPartBlocks) : need;
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
    if (backward) launch_behind(weight_gradient_kernel<T>, dim3((r.D + 31) / 32, 2), dim3(kBlock), 0, stream, r);
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
        if (chunk_values(p) == 8) return launch_group<T, 8>(r, group, p.interleaved != 0, backward, stream);
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
