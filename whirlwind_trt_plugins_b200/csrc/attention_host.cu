// attention_host.cu -- host side that the attention entry points share:
// argument checks and the relative-position bucket edges; the test hook of their
// device waits.
#include "attention.cuh"
#include "umma.cuh"

#include <cmath>

namespace ww {

int make_buckets(int num_buckets, int max_distance, int bidirectional, int q_offset, RelBuckets* out) noexcept
{
    if (num_buckets < 2 || (bidirectional && num_buckets % 2 != 0)) return WW_ERR_INVALID_SHAPE;
    if (num_buckets > kMaxBuckets) return WW_ERR_UNSUPPORTED;
    const int n = bidirectional ? num_buckets / 2 : num_buckets;
    const int e = n / 2;
    if (e < 1 || max_distance <= e || max_distance > (1 << 24)) return WW_ERR_INVALID_SHAPE;
    if (q_offset < -(1 << 30) || q_offset > (1 << 30)) return WW_ERR_INVALID_SHAPE;
    out->per_side = n;
    out->exact = e;
    out->bidirectional = bidirectional ? 1 : 0;
    out->q_offset = q_offset;
    out->total = num_buckets;
    out->max_distance = max_distance;
    out->n_least = n - e - 1;
    for (int t = 1; t < n - e; ++t) {
        // smallest whole d with ln(d / e) / ln(max / e) * (n - e) >= t.  The
        // edge is a whole number itself only where the power is exact; a
        // double is within 1e-14 of it there, and an irrational edge is not.
        const double edge = e * std::pow(static_cast<double>(max_distance) / e, static_cast<double>(t) / (n - e));
        const double whole = std::nearbyint(edge);
        out->least[t - 1] = static_cast<int32_t>(std::fabs(edge - whole) <= 1e-14 * edge ? whole : std::ceil(edge));
    }
    return WW_SUCCESS;
}

int tail_splits(int rest, int slots, int64_t tiles) noexcept
{
    if (rest == 0) return 1;
    // a CTA's start and end cost about 8 steps, joining parts about 6
    constexpr double kStart = 8.0, kJoin = 6.0;
    int best = 1;
    double least = tiles + kStart;
    for (int s = 2; s <= 64 && s * 4 <= tiles; ++s) {
        const double time = static_cast<double>((i64(rest) * s + slots - 1) / slots) * (static_cast<double>(tiles) / s + kStart) + kJoin;
        if (time < least) {
            least = time;
            best = s;
        }
    }
    return best;
}

bool vectors_ok(const void* ptr, const int64_t (&strides)[3], int B, int L, int H, int elem_bytes) noexcept
{
    if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0) return false;
    const int n[3] = {B, L, H};
    for (int i = 0; i < 3; ++i)
        if (n[i] > 1 && (strides[i] < 0 || (strides[i] * elem_bytes) % 16 != 0)) return false;
    return L <= 1 || strides[1] != 0;  // broadcast along b and h only
}

int check_attention(const ww_attention_t& p) noexcept
{
    if (p.dtype != WW_DTYPE_HALF && p.dtype != WW_DTYPE_BF16) return WW_ERR_INVALID_DTYPE;
    if (p.B < 0 || p.Lq < 0 || p.Lk < 0 || p.Hq <= 0 || p.Hk <= 0 || p.D <= 0) return WW_ERR_INVALID_SHAPE;
    if (p.Hq % p.Hk != 0) return WW_ERR_INVALID_SHAPE;
    if (!(std::isfinite(p.scale))) return WW_ERR_INVALID_SHAPE;
    if (p.D % 8 != 0 || p.D > 128) return WW_ERR_UNSUPPORTED;
    if (p.Lq > (1 << 28) || p.Lk > (1 << 28)) return WW_ERR_UNSUPPORTED;
    const bool has_q = p.B > 0 && p.Lq > 0, has_k = p.B > 0 && p.Lk > 0;
    if (has_q && (p.q == nullptr || p.out == nullptr)) return WW_ERR_NULL_POINTER;
    if (has_k && (p.k == nullptr || p.v == nullptr)) return WW_ERR_NULL_POINTER;
    if (p.bias_table != nullptr) {
        RelBuckets r;
        const int st = make_buckets(p.num_buckets, p.max_distance, p.bidirectional, p.q_offset, &r);
        if (st != WW_SUCCESS) return st;
        if (p.max_distance > kMaxDistance) return WW_ERR_UNSUPPORTED;
    }
    if (has_q && (!vectors_ok(p.q, p.q_strides, p.B, p.Lq, p.Hq, 2) || reinterpret_cast<uintptr_t>(p.out) % 16 != 0))
        return WW_ERR_MISALIGNED;
    if (has_k && (!vectors_ok(p.k, p.k_strides, p.B, p.Lk, p.Hk, 2) || !vectors_ok(p.v, p.v_strides, p.B, p.Lk, p.Hk, 2)))
        return WW_ERR_MISALIGNED;
    if (p.workspace != nullptr && reinterpret_cast<uintptr_t>(p.workspace) % 16 != 0) return WW_ERR_MISALIGNED;
    return WW_SUCCESS;
}

int check_attention_backward(const ww_attention_t& p, int64_t need) noexcept
{
    const bool has_q = p.B > 0 && p.Lq > 0, has_k = p.B > 0 && p.Lk > 0;
    if (has_q && (p.lse == nullptr || p.dout == nullptr || p.dq == nullptr)) return WW_ERR_NULL_POINTER;
    if (has_k && (p.dk == nullptr || p.dv == nullptr)) return WW_ERR_NULL_POINTER;
    if (p.bias_table != nullptr && p.dbias_table == nullptr) return WW_ERR_NULL_POINTER;
    if (need > 0 && p.workspace == nullptr) return WW_ERR_NULL_POINTER;
    if (need > p.workspace_bytes) return WW_ERR_UNSUPPORTED;
    if (has_q && (!vectors_ok(p.dout, p.dout_strides, p.B, p.Lq, p.Hq, 2) || reinterpret_cast<uintptr_t>(p.dq) % 16 != 0))
        return WW_ERR_MISALIGNED;
    if (has_k && (reinterpret_cast<uintptr_t>(p.dk) % 16 != 0 || reinterpret_cast<uintptr_t>(p.dv) % 16 != 0))
        return WW_ERR_MISALIGNED;
    return WW_SUCCESS;
}

namespace {

// Time until the wait for a barrier that nothing completes gave up; 0 if it did not.
__device__ unsigned long long g_bounded_wait_ns;

__global__ void bounded_wait_kernel()
{
    __shared__ uint64_t bar;
    const auto now = [] {
        unsigned long long t;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
        return t;
    };
    umma::mbar_init(umma::smem_addr(&bar), 1);
    umma::mbar_fence_init();
    const unsigned long long start = now();
    const bool done = umma::mbar_poll(umma::smem_addr(&bar), 0);
    g_bounded_wait_ns = done ? 0 : now() - start;
}

}  // namespace
}  // namespace ww

extern "C" int ww_selftest_bounded_wait(unsigned long long* ns)
{
    if (ns == nullptr) return WW_ERR_NULL_POINTER;
    ww::DeviceInfo d;
    const int st = ww::current_device_info(&d);
    if (st != WW_SUCCESS) return st;
    ww::bounded_wait_kernel<<<1, 1>>>();
    if (cudaMemcpyFromSymbol(ns, ww::g_bounded_wait_ns, sizeof(*ns)) != cudaSuccess)
        return ww::launch_status("ww_selftest_bounded_wait");
    return *ns != 0 ? WW_SUCCESS : WW_ERR_LAUNCH;
}

extern "C" int ww_relative_position_bucket(int rel, int num_buckets, int max_distance, int bidirectional)
{
    ww::RelBuckets r;
    const int st = ww::make_buckets(num_buckets, max_distance, bidirectional, 0, &r);
    if (st != WW_SUCCESS) return -st;
    if (rel == INT32_MIN) rel = -INT32_MAX;
    return ww::rel_bucket(r, rel);
}
