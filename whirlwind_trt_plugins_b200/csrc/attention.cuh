// attention.cuh -- what the attention kernels share: 16-bit type helpers, the
// relative-position buckets and the argument checks.
#pragma once

#include "ww_common.cuh"

#include <cuda_bf16.h>

#include <atomic>
#include <cstdint>

namespace ww {

constexpr float kLog2eF = 1.4426950408889634f;
constexpr float kLn2F = 0.6931471805599453f;
constexpr int kMaxBuckets = 128;

__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Division of n < 2^31 by d, prepared on the host.
struct Divisor {
    uint32_t mul = 1;
    int32_t shift = 0;
    int32_t d = 1;
    __device__ __forceinline__ int div(int n) const
    {
        return static_cast<int>((__umulhi(static_cast<uint32_t>(n), mul) + static_cast<uint32_t>(n)) >> shift);
    }
};

inline Divisor make_divisor(int d)
{
    Divisor r;
    r.d = d;
    while ((int64_t{1} << r.shift) < d) ++r.shift;
    r.mul = static_cast<uint32_t>(((((uint64_t{1} << r.shift) - d) << 32) / d) + 1);
    return r;
}

// ---- pairs of floats: one instruction for two values ----

struct Pair {
    uint64_t v;
};

__device__ __forceinline__ Pair pair(float lo, float hi)
{
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
    return r;
}

__device__ __forceinline__ void unpair(Pair p, float& lo, float& hi)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p.v));
}

__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c)
{
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

__device__ __forceinline__ Pair add2(Pair a, Pair b)
{
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

__device__ __forceinline__ Pair mul2(Pair a, Pair b)
{
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The largest; NaN if one is (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 2^x of two values on the FMA pipe, for x <= 127: x = n + f with n the nearest
// whole number (read off the low bits after adding 1.5 * 2^23), 2^f on
// [-1/2, 1/2] by a polynomial of degree 4 fitted to its relative error (2.6e-6,
// a hundredth of what rounding P to 16 bits costs), times 2^n.  The exponential unit
// does 16 values per clock and SM against 128 here, so a share of a tile's
// exponentials is done this way.
// SPECIALS: 2^n is a factor, formed as a float.  Below 2^-126.5 the result is 0, so -inf
// gives 0 as in the exponential unit; NaN and +inf give NaN: the clamp keeps a NaN,
// inf - inf makes one, the product carries it.
// Else n is added to the exponent field, an instruction less (8192 to 8192, 8 heads of
// 128: 335 us and 347): below 2^-126 and for NaN 2^-126, nothing for +inf; for callers
// that look at their arguments' maximum.
template <bool SPECIALS>
__device__ __forceinline__ Pair exp2_poly(Pair x)
{
    float a, b;
    unpair(x, a, b);
    x = SPECIALS ? pair(max_nan(a, -127.0f), max_nan(b, -127.0f)) : pair(fmaxf(a, -126.0f), fmaxf(b, -126.0f));
    constexpr float kMagic = 12582912.0f;
    const Pair t = add2(x, pair(kMagic, kMagic));
    const Pair n = add2(t, pair(-kMagic, -kMagic));
    const Pair f = fma2(n, pair(-1.0f, -1.0f), x);
    Pair p = pair(0.009570102f, 0.009570102f);
    p = fma2(p, f, pair(0.05591786f, 0.05591786f));
    p = fma2(p, f, pair(0.24024744f, 0.24024744f));
    p = fma2(p, f, pair(0.6931218f, 0.6931218f));
    p = fma2(p, f, pair(0.9999993f, 0.9999993f));
    float ta, tb;
    unpair(t, ta, tb);
    const uint32_t na = __float_as_uint(ta) << 23, nb = __float_as_uint(tb) << 23;
    if constexpr (SPECIALS) {  // (n + 127) << 23; n = -127 is 0
        return mul2(p, pair(__uint_as_float(na + 0x3f800000u), __uint_as_float(nb + 0x3f800000u)));
    } else {
        unpair(p, a, b);
        return pair(__uint_as_float(__float_as_uint(a) + na), __uint_as_float(__float_as_uint(b) + nb));
    }
}

// Relative-position buckets.  Distance d >= exact is in bucket
// exact + #{t : least[t] <= d}: least[t] is the smallest whole distance of
// logarithmic bucket t + 1, found once per call on the host, so that the
// kernels compare whole numbers and no logarithm is rounded at an edge.
struct RelBuckets {
    int32_t per_side = 0;  // buckets of one direction; 0: no bias
    int32_t exact = 0;
    int32_t bidirectional = 0;
    int32_t q_offset = 0;
    int32_t total = 0;
    int32_t max_distance = 0;  // |rel| >= this: last bucket of its side
    int32_t n_least = 0;
    int32_t least[kMaxBuckets / 2];
};

__host__ __device__ __forceinline__ int rel_bucket(const RelBuckets& r, int rel)
{
    int first = 0, d;
    if (r.bidirectional) {
        d = rel < 0 ? -rel : rel;
        if (rel > 0) first = r.per_side;
    } else {
        d = rel < 0 ? -rel : 0;
    }
    if (d < r.exact) return first + d;
    // counted, not searched: every thread reads the same edges in the same
    // order (a search's constant-memory reads differ by thread and serialise)
    int n = 0;
#ifdef __CUDA_ARCH__
#pragma unroll 8
#endif
    for (int t = 0; t < r.n_least; ++t) n += r.least[t] <= d;
    return first + r.exact + n;
}

// A bias at the type's lowest finite value forbids the pair like -inf: a row
// of such biases alone is empty instead of a softmax of rounding errors.
template <typename T>
__device__ __forceinline__ float bias_value(T b);
template <>
__device__ __forceinline__ float bias_value<__half>(__half b)
{
    const float f = __half2float(b);
    return f <= -65504.0f ? -INFINITY : f;
}
template <>
__device__ __forceinline__ float bias_value<__nv_bfloat16>(__nv_bfloat16 b)
{
    const float f = __bfloat162float(b);
    return f <= -0x1.fep127f ? -INFINITY : f;
}

// What one CTA needs of a head's bias: buckets of the relative positions
// [lo, hi] of its tiles, of which those further than max_distance + kRelMargin
// are left out -- a tile that reaches beyond holds one bucket only (a tile
// spans fewer than kRelMargin positions).  Built once per CTA into shared
// memory; entry e stands for rel = lo + e.
constexpr int kRelMargin = 256;
constexpr int kMaxDistance = 1024;  // what fits beside the operands of the widest heads
// positions that a CTA keeps at most
__host__ __device__ constexpr int rel_positions(int max_distance) { return 2 * (max_distance + kRelMargin) + 1; }
constexpr int kMaxPositions = rel_positions(kMaxDistance);
constexpr int kMaxShared = 232448;  // dynamic shared memory of a CTA, bytes

struct RelRange {
    int lo = 0, hi = -1;
    __host__ __device__ int count() const { return hi - lo + 1; }
};

__host__ __device__ __forceinline__ RelRange rel_range(const RelBuckets& r, int lo, int hi)
{
    const int far = r.max_distance + kRelMargin;
    RelRange g;
    g.lo = lo < -far ? -far : lo > far ? far : lo;
    g.hi = hi > far ? far : hi < -far ? -far : hi;
    return g;
}

// One head's table, spread over the lanes of a warp in log2 units: loaded early,
// looked up by shuffles (all lanes together) instead of dependent loads.
template <typename T>
struct TableRow {
    float v[kMaxBuckets / 32];
    __device__ __forceinline__ void load(const RelBuckets& r, const void* table, int h, int lane)
    {
        const T* row = static_cast<const T*>(table) + static_cast<int64_t>(h) * r.total;
#pragma unroll
        for (int k = 0; k < kMaxBuckets / 32; ++k)
            v[k] = lane + 32 * k < r.total ? bias_value<T>(row[lane + 32 * k]) * kLog2eF : 0.0f;
    }
    __device__ __forceinline__ float get(const RelBuckets& r, int bucket) const
    {
        float x = __shfl_sync(~0u, v[0], bucket & 31);
#pragma unroll
        for (int k = 1; k < kMaxBuckets / 32; ++k) {
            if (32 * k >= r.total) break;  // the same for all
            const float y = __shfl_sync(~0u, v[k], bucket & 31);
            if (bucket >> 5 == k) x = y;
        }
        return x;
    }
};

// Positions [lo, hi] of bucket t (empty where two edges coincide).
__device__ __forceinline__ RelRange bucket_positions(const RelBuckets& r, int t)
{
    constexpr int kFar = 1 << 30;
    const bool right = r.bidirectional && t >= r.per_side;
    const int i = right ? t - r.per_side : t;
    // distances [d0, d1]
    const int d0 = i <= r.exact ? i : r.least[i - r.exact - 1];
    const int d1 = i < r.exact ? i : i - r.exact < r.n_least ? r.least[i - r.exact] - 1 : kFar;
    RelRange x;
    x.lo = right ? max(d0, 1) : -d1;  // position 0 is on the left
    x.hi = right ? d1 : !r.bidirectional && i == 0 ? kFar : -d0;
    return x;
}

// Buckets of a range.  Ends without a barrier.
__device__ __forceinline__ void build_buckets(const RelBuckets& r, const RelRange& g, uint8_t* to, int thread, int threads)
{
    for (int e = thread; e < g.count(); e += threads) to[e] = static_cast<uint8_t>(rel_bucket(r, g.lo + e));
}

__device__ __forceinline__ int bucket_at(const RelRange& g, const uint8_t* buckets, int rel)
{
    return buckets[min(max(rel, g.lo), g.hi) - g.lo];
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ float f32(uint32_t u) { return __uint_as_float(u); }

// Barrier of the 128 threads of warpgroup w < 4.
__device__ __forceinline__ void warpgroup_sync(int w)
{
    if (w == 0) asm volatile("bar.sync 1, 128;" : : : "memory");
    else if (w == 1) asm volatile("bar.sync 2, 128;" : : : "memory");
    else if (w == 2) asm volatile("bar.sync 3, 128;" : : : "memory");
    else asm volatile("bar.sync 4, 128;" : : : "memory");
}

// Lets a kernel be launched with any dynamic shared memory that the current device has.
// The limit belongs to the kernel, not to a call: set to every call's own size, one host
// thread could lower it between another's setting and its launch.  So it is raised once,
// to the most; `raised` is the kernel's, a bit per device.
inline bool allow_shared_memory(const void* kernel, std::atomic<uint64_t>& raised) noexcept
{
    int dev = 0;
    DeviceInfo d;
    if (cudaGetDevice(&dev) != cudaSuccess || current_device_info(&d) != WW_SUCCESS) return false;
    const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
    if ((raised.load(std::memory_order_acquire) & bit) != 0) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, d.smem_optin) != cudaSuccess) return false;
    raised.fetch_or(bit, std::memory_order_release);
    return true;
}

// Launch of a kernel that follows another one of the same call, and waits for it
// (wait_for_launches_before) before it reads what that one writes, at the latest
// before it ends itself.  Where that one calls start_launch_behind (the gradient's pass
// over keys does), this kernel runs beside its last CTAs; else it starts when they have
// ended, without the gap of a launch that waits for their writes first.
template <typename... P, typename... A>
inline cudaError_t launch_behind(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A... args) noexcept
{
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

__device__ __forceinline__ void wait_for_launches_before()
{
    asm volatile("griddepcontrol.wait;" : : : "memory");
}

// Lets the kernel launched behind this one start on what SMs have left, once every
// CTA of this grid has called this or ended.
__device__ __forceinline__ void start_launch_behind()
{
    asm volatile("griddepcontrol.launch_dependents;" : : : "memory");
}

__device__ __forceinline__ void store_release(uint32_t* to, uint32_t v)
{
    asm volatile("st.release.gpu.global.u32 [%0], %1;" : : "l"(to), "r"(v) : "memory");
}

// Waits until *from is v: what the thread that released it had seen, this one sees too.
// Bounded (about half a second); false if it ran out.
__device__ __forceinline__ bool wait_acquire(const uint32_t* from, uint32_t v)
{
    for (int i = 0; i < 1 << 20; ++i) {
        uint32_t x;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(x) : "l"(from) : "memory");
        if (x == v) return true;
    }
    return false;
}

// Share [first, first + n) of part `split` of `splits` in `all` steps (a 64-bit
// division is worth avoiding where there is one part).
__device__ __forceinline__ void part_of(int all, int split, int splits, int& first, int& n)
{
    first = 0;
    n = all;
    if (splits > 1) {
        first = static_cast<int>(static_cast<int64_t>(all) * split / splits);
        n = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / splits) - first;
    }
}

// Fills `out`; WW_SUCCESS or the status of rejected arguments (attention_host.cu).
int make_buckets(int num_buckets, int max_distance, int bidirectional, int q_offset, RelBuckets* out) noexcept;

// Parts for each of `rest` items that do not fill a round of `slots` CTAs, of
// `tiles` steps each: the count whose rounds end soonest.
int tail_splits(int rest, int slots, int64_t tiles) noexcept;

// Checks the arguments that both directions of ww_cross_attention share.
int check_attention(const ww_attention_t& p) noexcept;
// What only the gradient needs: its pointers and `need` bytes of workspace.
int check_attention_backward(const ww_attention_t& p, int64_t need) noexcept;
bool vectors_ok(const void* ptr, const int64_t (&strides)[3], int B, int L, int H, int elem_bytes) noexcept;

}  // namespace ww
