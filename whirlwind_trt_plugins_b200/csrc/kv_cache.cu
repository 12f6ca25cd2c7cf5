// kv_cache.cu -- keys and values kept in 8 bits: rows (token, head) written with
// a scale each, and read back.
//
// Bound: HBM (writing: 2 bytes a value read, 1 written, and 4 a row; reading the
// reverse).  A row is held by a group of lanes with 16 bytes each of the 16-bit side,
// so that both sides of a warp lie side by side; the row's largest magnitude takes
// log2(lanes) shuffles, and a lane divides for each row of the group.  Where rows come
// from and go is worked out by a thread each and kept in shared memory.  Scales stand
// by head, so that attention reads those of a head's keys as a run.
//
// Measured, 2 x 40001 tokens of 8 heads of 128, fp16, keys and values: written (492 MB) in
// 88 us, read back (492 MB) in 83: 5.6 and 5.9 TB/s.
#include "rows.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace ww {
namespace {

constexpr int kBlock = 256;
// Rows of a group under way, reading and writing (2 x 40001 x 8 rows of 128 written and read
// back: 4 rows written at a time 171 us, 2 185).
constexpr int kRows = 2, kWriteRows = 4;

struct CacheSide {
    const void* x;
    int8_t* q;
    float* scale;
    void* out;
    int64_t xb, xl, xh, qb, ql, qh, sb, sh;
};

struct CacheParams {
    CacheSide side[2];  // keys, values
    const int32_t *start, *lens;
    Divisor L, H;  // tokens (reading: places) of an item, heads
    int32_t rows, places, D, keep;  // keep: what lies behind the lens is not written (reading)
    const uint8_t* mask;            // [B][places] of the keys that count, or
    float2* powers;                 // [B][H] of keys and values that are read back divided by powers of two
};

struct CacheRow {
    int b, l, h;
    __device__ __forceinline__ CacheRow(const CacheParams& p, int row)
    {
        const int token = p.H.div(row);
        h = row - token * p.H.d;
        b = p.L.div(token);
        l = token - b * p.L.d;
    }
};

template <typename T, int GROUP>
__global__ void __launch_bounds__(kBlock) quantize_kv_kernel(const __grid_constant__ CacheParams p)
{
    constexpr int R = kWriteRows, kStep = kBlock / GROUP;
    // where the block's rows come from and go, worked out by a thread each
    __shared__ int64_t from[kStep * R], to[kStep * R], scale_to[kStep * R];  // from < 0: not written
    const CacheSide& s = p.side[blockIdx.y];
    const int lane = threadIdx.x % GROUP, d = lane * 8, first = threadIdx.x / GROUP;
    for (int i = threadIdx.x; i < kStep * R; i += kBlock) {
        const int64_t row = static_cast<int64_t>(blockIdx.x) * (kStep * R) + i;
        from[i] = -1;
        if (row >= p.rows) continue;
        const CacheRow at(p, static_cast<int>(row));
        const int64_t place = (p.start == nullptr ? int64_t{0} : static_cast<int64_t>(__ldg(p.start + at.b))) + at.l;
        if (place < 0 || place >= p.places || (p.lens != nullptr && at.l >= __ldg(p.lens + at.b))) continue;
        from[i] = at.b * s.xb + at.l * s.xl + at.h * s.xh;
        to[i] = at.b * s.qb + place * s.ql + at.h * s.qh;
        scale_to[i] = at.b * s.sb + at.h * s.sh + place;
    }
    __syncthreads();
    Piece<T, 8> raw[R][1];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        raw[i][0].clear();
        const int64_t at = from[first + i * kStep];
        if (at >= 0 && d < p.D) raw[i][0].load(static_cast<const T*>(s.x) + at + d);
    }
    Pair f[R][4];
    float top[R];
    RowScale k[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        values_of<T, 8, 1>(raw[i], f[i]);
        top[i] = largest(f[i]);
    }
    row_maxima<GROUP>(top, nullptr);
    row_scales<GROUP>(top, k);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = first + i * kStep;
        if (from[r] < 0) continue;
        if (d < p.D) store_piece_int8<8>(s.q + to[r] + d, f[i], k[i].inv, 0);
        if (lane == 0) s.scale[scale_to[r]] = k[i].scale;
    }
}

// The power of two by which a head's keys or values are divided in fp16, whose range is narrower than the scales': the largest
// comes to [2^8, 2^9) 127, or stays what it is where fp16 holds it with 5 bits to spare above its subnormal numbers.
__device__ __forceinline__ float power_of(float top)
{
    if (top == 0.0f || (top >= 0x1p-17f && top < 0x1p9f)) return 1.0f;
    const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127 - 8;
    return __uint_as_float(static_cast<uint32_t>(127 + min(max(e, -100), 113)) << 23);
}

// Those of all heads, keys and values in turn (rows [B][H][2]): a warp for each, or where places are many a cluster of blocks.
// Bound: latency, a few loads after one another: 8 heads of 40001 places 7 us, 12032 of 312 10.5.
constexpr int kWarpPlaces = 1024, kMostBlocks = 8;

template <bool MANY>
__global__ void __launch_bounds__(MANY ? 1024 : kBlock) kv_powers_kernel(const __grid_constant__ CacheParams p, int rows)
{
    __shared__ float red[32], joined;
    start_launch_behind();  // reading back waits for this grid's end
    const auto cluster = cooperative_groups::this_cluster();
    const int blocks = MANY ? static_cast<int>(cluster.num_blocks()) : 1, rank = MANY ? static_cast<int>(cluster.block_rank()) : 0;
    const int row = MANY ? blockIdx.x / blocks : blockIdx.x * (kBlock / 32) + threadIdx.x / 32;
    float top = 0.0f;
    if (row < rows) {
        const int b = p.H.div(row / 2), h = row / 2 - b * p.H.d;
        const CacheSide& s = p.side[row % 2];
        const float* scale = s.scale + b * s.sb + h * s.sh;
        const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + static_cast<int64_t>(b) * p.places;
        const int len = p.lens == nullptr ? p.places : min(__ldg(p.lens + b), p.places);
#pragma unroll 8
        for (int at = MANY ? rank * 1024 + threadIdx.x : threadIdx.x % 32; at < len; at += MANY ? blocks * 1024 : 32) {
            const float x = fabsf(__ldg(scale + at));
            const bool counts = mask == nullptr || __ldg(mask + at) != 0;
            top = counts && x < INFINITY ? fmaxf(top, x) : top;
        }
    }
    top = row_max<MANY ? 0 : 32>(top, red);
    if constexpr (MANY) {
        if (threadIdx.x == 0) joined = top;
        cluster.sync();
        if (rank == 0 && threadIdx.x == 0)
            for (int i = 1; i < blocks; ++i) top = fmaxf(top, *cluster.map_shared_rank(&joined, i));
        cluster.sync();  // until it has been read
    }
    if (row < rows && rank == 0 && (MANY ? threadIdx.x : threadIdx.x % 32) == 0) reinterpret_cast<float*>(p.powers)[row] = power_of(top);
}

int launch_powers(const CacheParams& f, const char* name, cudaStream_t stream) noexcept
{
    const int rows = f.rows / f.places * 2;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(std::min(kMostBlocks, (f.places + 4095) / 4096));
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.stream = stream;
    if (f.places > kWarpPlaces) {
        cfg.gridDim = dim3(static_cast<unsigned>(rows) * attr.val.clusterDim.x);
        cfg.blockDim = dim3(1024);
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        cudaLaunchKernelEx(&cfg, kv_powers_kernel<true>, f, rows);
    } else {
        cfg.gridDim = dim3((rows + kBlock / 32 - 1) / (kBlock / 32));
        cfg.blockDim = dim3(kBlock);
        cudaLaunchKernelEx(&cfg, kv_powers_kernel<false>, f, rows);
    }
    return launch_status(name);
}

template <typename T, int GROUP>
__global__ void __launch_bounds__(kBlock) dequantize_kv_kernel(const __grid_constant__ CacheParams p)
{
    const CacheSide& s = p.side[blockIdx.y];
    const int lane = threadIdx.x % GROUP, d = lane * 8;
    constexpr int kStep = kBlock / GROUP;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kStep * kRows + threadIdx.x / GROUP;
    if (d >= p.D) return;
    uint2 q[kRows];
    float scale[kRows];
    int head[kRows];
    bool put[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int64_t row = first + i * kStep;
        put[i] = row < p.rows;
        q[i] = make_uint2(0, 0);
        scale[i] = 0.0f;
        head[i] = 0;
        if (!put[i]) continue;
        const CacheRow at(p, static_cast<int>(row));
        head[i] = at.b * p.H.d + at.h;
        if (p.lens == nullptr || at.l < __ldg(p.lens + at.b)) {
            q[i] = __ldg(reinterpret_cast<const uint2*>(s.q + at.b * s.qb + at.l * s.ql + at.h * s.qh + d));
            scale[i] = __ldg(s.scale + at.b * s.sb + at.h * s.sh + at.l);
        } else if (p.keep) {
            put[i] = false;
        }
    }
    if (p.powers != nullptr) {
        wait_for_launches_before();
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const float power = reinterpret_cast<const float*>(p.powers + head[i])[blockIdx.y];
            scale[i] *= __uint_as_float((254u << 23) - __float_as_uint(power));  // 1 / power
        }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if (!put[i]) continue;
        uint32_t r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t w = j < 2 ? q[i].x : q[i].y;
            const float a = static_cast<float>(static_cast<int8_t>(w >> (j % 2 * 16))), b = static_cast<float>(static_cast<int8_t>(w >> (j % 2 * 16 + 8)));
            r[j] = pack2<T>(a * scale[i], b * scale[i]);
        }
        *reinterpret_cast<uint4*>(static_cast<T*>(s.out) + (first + i * kStep) * p.D + d) = make_uint4(r[0], r[1], r[2], r[3]);
    }
}

CacheParams params(const ww_kv_cache_t& p, int tokens) noexcept
{
    CacheParams f{};
    const auto side = [&](CacheSide& s, const void* x, int8_t* q, float* scale, void* out, const int64_t (&xs)[3], const int64_t (&qs)[3],
                          const int64_t (&ss)[2]) {
        s = {x, q, scale, out, xs[0], xs[1], xs[2], qs[0], qs[1], qs[2], ss[0], ss[1]};
    };
    side(f.side[0], p.k, p.k_cache, p.k_scale, p.k_out, p.k_strides, p.k_cache_strides, p.k_scale_strides);
    side(f.side[1], p.v, p.v_cache, p.v_scale, p.v_out, p.v_strides, p.v_cache_strides, p.v_scale_strides);
    f.start = p.start;
    f.lens = p.lens;
    f.L = make_divisor(std::max(tokens, 1));
    f.H = make_divisor(p.H);
    f.rows = p.B * tokens * p.H;
    f.places = p.places;
    f.D = p.D;
    return f;
}

template <bool WRITE, typename T>
int launch(const CacheParams& f, const char* name, cudaStream_t stream) noexcept
{
    const int group = f.D <= 32 ? 4 : f.D <= 64 ? 8 : 16, step = kBlock / group * (WRITE ? kWriteRows : kRows);
    const dim3 grid(static_cast<unsigned>((i64(f.rows) + step - 1) / step), 2);
    if (f.powers != nullptr) {
        if (const int st = launch_powers(f, name, stream); st != WW_SUCCESS) return st;
    }
    const auto go = [&](auto kernel) {
        if (f.powers != nullptr) launch_behind(kernel, grid, dim3(kBlock), 0, stream, f);
        else kernel<<<grid, kBlock, 0, stream>>>(f);
    };
    if constexpr (WRITE) {
        if (group == 4) go(quantize_kv_kernel<T, 4>);
        else if (group == 8) go(quantize_kv_kernel<T, 8>);
        else go(quantize_kv_kernel<T, 16>);
    } else {
        if (group == 4) go(dequantize_kv_kernel<T, 4>);
        else if (group == 8) go(dequantize_kv_kernel<T, 8>);
        else go(dequantize_kv_kernel<T, 16>);
    }
    return launch_status(name);
}

int check(const ww_kv_cache_t& p, bool write) noexcept
{
    if (p.dtype != WW_DTYPE_HALF && p.dtype != WW_DTYPE_BF16) return WW_ERR_INVALID_DTYPE;
    const int tokens = write ? p.L : p.places;
    if (p.B < 0 || p.L < 0 || p.places < 0 || p.H <= 0 || p.D <= 0) return WW_ERR_INVALID_SHAPE;
    if (p.D % 16 != 0 || p.D > 128) return WW_ERR_UNSUPPORTED;
    if (i64(p.B) * tokens >= INT32_MAX || i64(p.B) * tokens * p.H >= INT32_MAX) return WW_ERR_UNSUPPORTED;
    if (p.B == 0 || tokens == 0 || p.places == 0) return WW_SUCCESS;
    if (p.k_cache == nullptr || p.v_cache == nullptr || p.k_scale == nullptr || p.v_scale == nullptr) return WW_ERR_NULL_POINTER;
    if (write ? p.k == nullptr || p.v == nullptr : p.k_out == nullptr || p.v_out == nullptr) return WW_ERR_NULL_POINTER;
    for (const int64_t(*s)[3] : {&p.k_cache_strides, &p.v_cache_strides}) {
        const int n[3] = {p.B, p.places, p.H};
        for (int i = 0; i < 3; ++i) {
            if (n[i] <= 1) continue;
            if (write && (*s)[i] == 0) return WW_ERR_INVALID_SHAPE;  // two places in one
            if ((*s)[i] < 0 || (*s)[i] % 16 != 0) return WW_ERR_MISALIGNED;
        }
    }
    for (const int64_t(*s)[2] : {&p.k_scale_strides, &p.v_scale_strides})
        for (int i = 0; i < 2; ++i)
            if ((i ? p.H : p.B) > 1 && ((*s)[i] < 0 || (write && (*s)[i] < p.places))) return WW_ERR_INVALID_SHAPE;  // two in one
    const auto off = [](const void* q, int by) { return reinterpret_cast<uintptr_t>(q) % by != 0; };
    if (off(p.k_cache, 16) || off(p.v_cache, 16) || off(p.k_scale, 4) || off(p.v_scale, 4) || off(p.start, 4) || off(p.lens, 4))
        return WW_ERR_MISALIGNED;
    if (write ? !vectors_ok(p.k, p.k_strides, p.B, p.L, p.H, 2) || !vectors_ok(p.v, p.v_strides, p.B, p.L, p.H, 2)
              : off(p.k_out, 16) || off(p.v_out, 16))
        return WW_ERR_MISALIGNED;
    return WW_SUCCESS;
}

// What reading back for an attention call adds: see dequantise_valid.
struct Valid {
    bool keep = false;
    const uint8_t* mask = nullptr;
    float2* powers = nullptr;
};

template <bool WRITE>
int run(const ww_kv_cache_t* p, const Valid& valid, const char* name, void* stream) noexcept
{
    if (p == nullptr) return WW_ERR_NULL_POINTER;
    int st = check(*p, WRITE);
    const int tokens = WRITE ? p->L : p->places;
    if (st != WW_SUCCESS || p->B == 0 || tokens == 0 || p->places == 0) return st;
    DeviceInfo d;
    if ((st = current_device_info(&d)) != WW_SUCCESS) return st;
    CacheParams f = params(*p, tokens);
    f.keep = valid.keep;
    f.mask = valid.mask;
    f.powers = valid.powers;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return p->dtype == WW_DTYPE_HALF ? launch<WRITE, __half>(f, name, s) : launch<WRITE, __nv_bfloat16>(f, name, s);
}

}  // namespace

// ww_dequantize_kv that leaves what lies behind the lens unwritten.  With `powers` [B][H] it divides the keys and values of each
// item's head by powers of two, of the scales in valid places (mask [B][places], nullptr for all), and leaves those there.
int dequantise_valid(const ww_kv_cache_t& p, const uint8_t* mask, float2* powers, const char* name, void* stream) noexcept
{
    return run<false>(&p, {true, mask, powers}, name, stream);
}

}  // namespace ww

extern "C" {

int ww_quantize_kv(const ww_kv_cache_t* p, void* stream) { return ww::run<true>(p, {}, "quantize_kv", stream); }
int ww_dequantize_kv(const ww_kv_cache_t* p, void* stream) { return ww::run<false>(p, {}, "dequantize_kv", stream); }

}  // extern "C"
