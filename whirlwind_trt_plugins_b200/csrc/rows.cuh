// rows.cuh -- what the kernels over rows of values share: pieces of a row in
// registers as pairs of fp32, sums over the lanes of a row, and the 8-bit form
// of a row.
#pragma once

#include "attention.cuh"

#include <climits>

namespace ww {

// ---- a row in 8 bits ----
//
// a = max |x|,  scale = a / 127,  q = rint(x * (127 * (1 / a))), every operation rounded in
// fp32, so that tensor operations give the same numbers: whole ones in [-127, 127], x = scale q
// within half a step and 2^-15 of one (one of 10^5 fp32 values goes to the other side of a middle).  A row with a NaN or an infinity
// has scale NaN, so that what is computed from it is NaN; one whose largest
// magnitude is below 2^-119 (the scale would leave fp32's normal range) has
// scale 0 and zeros.
struct RowScale {
    float inv, scale;
};

__device__ __forceinline__ RowScale row_scale(float top)  // top: max_nan over |x|
{
    RowScale r{0.0f, 0.0f};
    if (!(top < INFINITY)) r.scale = __int_as_float(0x7fffffff);
    else if (top >= 0x1p-119f) {
        r.inv = __fmul_rn(__fdiv_rn(1.0f, top), 127.0f);
        r.scale = __fdiv_rn(top, 127.0f);
    }
    return r;
}

// rint of a product in [-127, 127] in the low byte: adding 1.5 * 2^23 leaves the whole
// number, ties to even, in the low bits.  The product is rounded before, as the formula says, so
// that most values of few bits that lie half way between two steps are met as ties (packed
// forms of the two would be fused by the compiler).
constexpr float kRintMagic = 12582912.0f;

__device__ __forceinline__ int8_t quantise(float x, float inv)
{
    return static_cast<int8_t>(__float_as_uint(__fadd_rn(__fmul_rn(x, inv), kRintMagic)));
}

__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)  // low bytes
{
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Two values to whole numbers in the low bytes.
__device__ __forceinline__ void quantise2(Pair x, Pair inv, uint32_t& lo, uint32_t& hi)
{
    float a, b;
    unpair(mul2(x, inv), a, b);
    lo = __float_as_uint(__fadd_rn(a, kRintMagic));
    hi = __float_as_uint(__fadd_rn(b, kRintMagic));
}

// ---- pieces of V values of T, as they are loaded ----

template <typename T, int V>
struct Piece {
    static constexpr int kBytes = V * static_cast<int>(sizeof(T));
    static constexpr int kWords = kBytes >= 4 ? kBytes / 4 : 1;
    alignas(kBytes >= 4 ? kBytes : 4) uint32_t w[kWords];

    __device__ __forceinline__ void load(const T* p)
    {
        if constexpr (kBytes == 16) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
            w[0] = u.x;
            w[1] = u.y;
            w[2] = u.z;
            w[3] = u.w;
        } else if constexpr (kBytes == 8) {
            const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
            w[0] = u.x;
            w[1] = u.y;
        } else if constexpr (kBytes == 4) {
            w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
        } else {
            static_assert(kBytes == 2, "16, 8, 4 or 2 bytes");
            w[0] = __ldg(reinterpret_cast<const unsigned short*>(p));
        }
    }
    // Values 0 and 1 of a pair of which one may lie outside the row; outside becomes 0.
    __device__ __forceinline__ void set_pair(const T* first, bool has0, bool has1)
    {
        static_assert(V == 2, "pairs");
        Piece<T, 1> a, b;
        a.clear();
        b.clear();
        if (has0) a.load(first);
        if (has1) b.load(first + 1);
        if constexpr (sizeof(T) == 4) {
            w[0] = a.w[0];
            w[1] = b.w[0];
        } else {
            w[0] = a.w[0] | b.w[0] << 16;
        }
    }
    // Of a pair at an edge of a row, read whole (its word lies in the row's memory), what lies outside becomes 0.
    __device__ __forceinline__ void keep(bool has0, bool has1)
    {
        static_assert(V == 2, "pairs");
        if constexpr (sizeof(T) == 4) {
            w[0] = has0 ? w[0] : 0;
            w[1] = has1 ? w[1] : 0;
        } else {
            w[0] &= (has0 ? 0xffffu : 0u) | (has1 ? 0xffff0000u : 0u);
        }
    }
    __device__ __forceinline__ void load_shared(const T* p)
    {
        static_assert(kBytes == 16, "16 bytes");
        *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
    }
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    __device__ __forceinline__ float get(int i) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        const uint32_t u = i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu;
        if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(static_cast<unsigned short>(u)));
        return i % 2 ? __uint_as_float(w[i / 2] & 0xffff0000u) : __uint_as_float(w[i / 2] << 16);
    }
};

// E values of a row as E / 2 pairs; value e of the lane is value e % V of its piece e / V.
template <typename T, int V, int P>
__device__ __forceinline__ void values_of(const Piece<T, V> (&raw)[P], Pair (&f)[P * V / 2])
{
#pragma unroll
    for (int i = 0; i < P * V / 2; ++i) {
        const int e = 2 * i;
        if constexpr (std::is_same<T, __half>::value && V > 1) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&raw[e / V].w[e % V / 2]));
            f[i] = pair(v.x, v.y);
        } else {
            f[i] = pair(raw[e / V].get(e % V), raw[(e + 1) / V].get((e + 1) % V));
        }
    }
}

// Columns of a lane's pieces: piece i begins at `first` + i kNext, side by side over the lanes
// of a group or, where a block holds the row, of a warp (whose pieces follow one another).
// Pairs (V == 2) of a row that begins off their grid are shifted by one: the first begins at -1.
template <int V, int P, int GROUP>
struct Columns {
    static constexpr int kNext = (GROUP ? GROUP : 32) * V;
    int first;
    __device__ __forceinline__ explicit Columns(int shift = 0)
        : first((GROUP ? threadIdx.x % (GROUP ? GROUP : 1) * V : threadIdx.x / 32 * (P * kNext) + threadIdx.x % 32 * V) - shift) {}
    __device__ __forceinline__ int operator()(int i) const { return first + i * kNext; }
    // All of piece i lies within a row of n values; value j of it does.
    __device__ __forceinline__ bool whole(int i, int n) const
    {
        return V == 2 ? static_cast<uint32_t>((*this)(i)) < static_cast<uint32_t>(n - 1) : (*this)(i) < n;
    }
    __device__ __forceinline__ bool has(int i, int j, int n) const
    {
        return V == 2 ? static_cast<uint32_t>((*this)(i) + j) < static_cast<uint32_t>(n) : (*this)(i) < n;
    }
};

// Piece i of a row of n values, from `at`, zeros where it lies outside.  Pairs at an edge: EDGES value by value, else their
// word or two words, which lie in the memory of the row's edge, with what is outside cleared.
template <bool EDGES, typename T, int V, int P, int GROUP>
__device__ __forceinline__ void load_piece(Piece<T, V>& to, const T* at, int i, int n, bool real, const Columns<V, P, GROUP>& column)
{
    if constexpr (V == 2 && EDGES) {
        if (real && column.whole(i, n)) {
            to.load(at);
        } else {
            to.clear();
            if (real && column(i) < n) to.set_pair(at, column.has(i, 0, n), column.has(i, 1, n));
        }
    } else {
        to.clear();
        if (real && column(i) < n) to.load(at);
        if constexpr (V == 2) to.keep(column(i) >= 0, column(i) + 1 < n);
    }
}

// Weights of a lane's columns, which may begin anywhere.
template <typename T, int V, int P, int GROUP>
__device__ __forceinline__ void load_weights(Piece<T, V> (&to)[P], const T* w, int n, const Columns<V, P, GROUP>& column)
{
#pragma unroll
    for (int i = 0; i < P; ++i) {
        to[i].clear();
        if (w == nullptr) continue;
        if constexpr (V == 2) to[i].set_pair(w + column(i), column.has(i, 0, n), column.has(i, 1, n));
        else if (column(i) < n) to[i].load(w + column(i));
    }
}

// What a lane holds beyond the n values of its row becomes 0.
template <int V, int P, int GROUP>
__device__ __forceinline__ void clear_beyond(Pair (&f)[P * V / 2], int n, const Columns<V, P, GROUP>& column)
{
#pragma unroll
    for (int i = 0; i < P; ++i)
        if (!column.whole(i, n))
#pragma unroll
            for (int e = i * V; e < (i + 1) * V; ++e) {
                if (column.has(i, e % V, n)) continue;
                float a, b;
                unpair(f[e / 2], a, b);
                f[e / 2] = e % 2 ? pair(a, 0.0f) : pair(0.0f, b);
            }
}

// Piece i of a lane's values to memory.
template <typename T, int V, int E>
__device__ __forceinline__ void store_piece(T* p, const Pair (&f)[E], int i)
{
    if constexpr (V == 1) {
        float v[2];
        unpair(f[i / 2], v[0], v[1]);
        *p = from_float<T>(i % 2 ? v[1] : v[0]);
    } else if constexpr (V == 2) {
        float v[2];
        unpair(f[i], v[0], v[1]);
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
        else *reinterpret_cast<uint32_t*>(p) = pack2<T>(v[0], v[1]);
    } else {
        float v[V];
#pragma unroll
        for (int j = 0; j < V / 2; ++j) unpair(f[i * V / 2 + j], v[2 * j], v[2 * j + 1]);
        if constexpr (sizeof(T) == 4)
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else
            *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
}

// Piece i of a row of n values, as far as it lies within.
template <typename T, int V, int P, int GROUP, int E>
__device__ __forceinline__ void store_row_piece(T* p, const Pair (&f)[E], int i, int n, const Columns<V, P, GROUP>& column)
{
    if (column.whole(i, n)) {
        store_piece<T, V>(p, f, i);
    } else if constexpr (V == 2) {
        float v[2];
        unpair(f[i], v[0], v[1]);
        if (column.has(i, 0, n)) p[0] = from_float<T>(v[0]);
        if (column.has(i, 1, n)) p[1] = from_float<T>(v[1]);
    }
}

// Piece i in 8 bits to memory.
template <int V, int E>
__device__ __forceinline__ void store_piece_int8(int8_t* p, const Pair (&f)[E], float inv, int i, bool has0 = true, bool has1 = true)
{
    const Pair k = pair(inv, inv);
    if constexpr (V == 1) {
        uint32_t q[2];
        quantise2(f[i / 2], k, q[0], q[1]);
        *p = static_cast<int8_t>(i % 2 ? q[1] : q[0]);
    } else if constexpr (V == 2) {
        uint32_t q[2];
        quantise2(f[i], k, q[0], q[1]);
        if (has0) p[0] = static_cast<int8_t>(q[0]);
        if (has1) p[1] = static_cast<int8_t>(q[1]);
    } else {
        uint32_t q[V];
#pragma unroll
        for (int j = 0; j < V / 2; ++j) quantise2(f[i * V / 2 + j], k, q[2 * j], q[2 * j + 1]);
        if constexpr (V == 4)
            *reinterpret_cast<uint32_t*>(p) = pack4(q[0], q[1], q[2], q[3]);
        else
            *reinterpret_cast<uint2*>(p) = make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
    }
}

__device__ __forceinline__ float both(Pair p)
{
    float a, b;
    unpair(p, a, b);
    return a + b;
}

// K sums, or largest values (NaN above all), over the GROUP lanes of a row; GROUP 0: over
// the block, in a fixed order (`red`: 32 K floats of shared memory that no other call
// under way uses; one barrier).
template <int GROUP, bool MAX, int K>
__device__ __forceinline__ void row_joins(float (&v)[K], float* red)
{
    const auto join = [](float a, float b) { return MAX ? max_nan(a, b) : a + b; };
#pragma unroll
    for (int o = (GROUP ? GROUP : 32) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = join(v[k], __shfl_xor_sync(~0u, v[k], o));
    if constexpr (GROUP == 0) {
        if (threadIdx.x % 32 == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) red[k * 32 + threadIdx.x / 32] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = threadIdx.x % 32 < blockDim.x / 32 ? red[k * 32 + threadIdx.x % 32] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] = join(v[k], __shfl_xor_sync(~0u, v[k], o));
    }
}

template <int GROUP, int K>
__device__ __forceinline__ void row_sums(float (&v)[K], float* red)
{
    row_joins<GROUP, false, K>(v, red);
}

template <int GROUP, int K>
__device__ __forceinline__ void row_maxima(float (&v)[K], float* red)
{
    row_joins<GROUP, true, K>(v, red);
}

template <int GROUP>
__device__ __forceinline__ float row_sum(float v, float* red)
{
    float x[1] = {v};
    row_sums<GROUP>(x, red);
    return x[0];
}

template <int GROUP>
__device__ __forceinline__ float row_max(float v, float* red)
{
    float x[1] = {v};
    row_maxima<GROUP>(x, red);
    return x[0];
}

// Scales of the K <= GROUP rows that a group of lanes holds (GROUP 0: of a block's warp), whose
// largest magnitudes every lane has: lane k divides for row k (a division costs as much as
// bringing several values to 8 bits), the others get its quotients.
template <int GROUP, int K>
__device__ __forceinline__ void row_scales(const float (&top)[K], RowScale (&r)[K])
{
    if constexpr (K == 1) {
        r[0] = row_scale(top[0]);
    } else {
        constexpr int kLanes = GROUP ? GROUP : 32;
        static_assert(K <= kLanes, "a lane for each row");
        const int lane = threadIdx.x % kLanes;
        float mine = top[0];
#pragma unroll
        for (int k = 1; k < K; ++k) mine = lane == k ? top[k] : mine;
        const RowScale own = row_scale(mine);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            r[k].inv = __shfl_sync(~0u, own.inv, k, kLanes);
            r[k].scale = __shfl_sync(~0u, own.scale, k, kLanes);
        }
    }
}

template <int E>
__device__ __forceinline__ float largest(const Pair (&f)[E])
{
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        float a, b;
        unpair(f[i], a, b);
        top = max3_nan(top, fabsf(a), fabsf(b));
    }
    return top;
}

// How a row of n values lies on lanes: `group` lanes a row (0: `threads` of a block),
// `pieces` pieces of V values each; group and pieces both 0: too long for registers.
struct RowForm {
    int group, pieces, threads;
};

// Most threads of a block that holds a row, P pieces of V values a lane.
__host__ __device__ constexpr int row_threads(int v, int p, bool backward) { return v > 2 ? (backward ? 512 : 1024) : v == 1 && p == 8 ? 256 : 640; }

// Pieces of 16 bytes (v > 1): the form with the fewest idle lanes, and of those the one
// with the fewest pieces a lane (at most `most` in a warp).  Pairs or single values (v <= 2, rows that
// do not start on 16 bytes): 4, 8 or 16 values a lane, pairs only where a block's lanes hold 16.  Rows that
// a warp does not hold: a block.
inline RowForm row_form(int n, int v, int most, bool backward)
{
    const int all = v == 2 ? n / 2 + 1 : (n + v - 1) / v;  // pairs may be shifted by one
    const auto fits = [&](int p) { return all <= row_threads(v, p, backward) * p; };
    const auto block = [&](int p) { return RowForm{0, p, ((all + p - 1) / p + 31) / 32 * 32}; };
    if (v > 2) {
        constexpr int kForms[][2] = {{4, 1}, {8, 1}, {16, 1}, {32, 1}, {16, 3}, {32, 2}, {32, 3}, {32, 4}};
        for (const auto& f : kForms)  // ascending lanes x pieces
            if (f[0] * f[1] >= all && f[1] <= most) return {f[0], f[1], 256};
        if (fits(2)) return block(2);
    } else if (v == 2) {
        if (fits(8)) return block(8);
    } else {
        if (n <= 128) return {32, 4, 256};
        if (n <= 512) return {32, 16, 256};
        for (int p : {8, 16})
            if (fits(p)) return block(p);
    }
    return {0, 0, 0};
}

}  // namespace ww
