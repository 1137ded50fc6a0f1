// Paged key-value cache: the append of new keys and values (with the rotary position embedding applied on the way) and the
// attention of new tokens' query rows over the pages.
#include <hip/hip_runtime.h>

#include <cmath>

#include "ops_kernels.hpp"

namespace t3k {
namespace {

// fp32 -> bf16, to the nearest, ties to even; NaN stays NaN
__device__ __forceinline__ uint16_t to_bf16(float f) {
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ float from_bf16(uint16_t h) { return __uint_as_float((uint32_t)h << 16); }

template <typename T> __device__ __forceinline__ float load1(const void* p, long long i) {
    if constexpr (sizeof(T) == 2) return from_bf16(static_cast<const uint16_t*>(p)[i]);
    else return static_cast<const float*>(p)[i];
}
template <typename T> __device__ __forceinline__ void store1(void* p, long long i, float v) {
    if constexpr (sizeof(T) == 2) static_cast<uint16_t*>(p)[i] = to_bf16(v);
    else static_cast<float*>(p)[i] = v;
}

// page of key j of sequence s, or -1: outside the table, or an entry that names no page of the pool
__device__ __forceinline__ int page_of(const PagedCache& c, int s, int j) {
    const int e = j >> c.page_shift;
    if (e >= c.max_pages) return -1;
    const int p = c.table[(long long)s * c.table_stride + e];
    return p >= 0 && p < c.n_pages ? p : -1;
}

// one thread per element pair (i, i + head_dim / 2) of a head of q, k or v:  (a, b) -> (a cos - b sin, b cos + a sin)
template <typename IN, typename KV>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
    const int half = a.c.head_dim >> 1;
    const int heads = (a.q ? a.q_heads : 0) + 2 * a.c.kv_heads;
    const long long per_row = (long long)heads * half, total = per_row * a.rows;
    const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
    if (idx >= total) return;
    const int row = (int)(idx / per_row), rem = (int)(idx % per_row);
    int head = rem / half;
    const int i = rem % half;
    const int pos = a.positions[row], s = a.seq ? a.seq[row] : row;
    if (pos < 0 || s < 0 || s >= a.c.n_seqs || (a.cos && pos >= a.rope_len)) return;
    const int page = page_of(a.c, s, pos);
    if (page < 0) return;
    const int slot = pos & ((1 << a.c.page_shift) - 1);
    const bool is_v = head >= heads - a.c.kv_heads;
    float c = 1.f, sn = 0.f;
    if (a.cos && !is_v) {
        c = a.cos[pos * a.rope_stride + i];
        sn = a.sin[pos * a.rope_stride + i];
    }
    const int qn = a.q ? a.q_heads : 0;
    if (head < qn) {
        const long long o = row * a.qr + head * a.qh + i, w = row * a.qor + head * a.qoh + i;
        const float x = load1<IN>(a.q, o), y = load1<IN>(a.q, o + half);
        store1<IN>(a.q_out, w, x * c - y * sn);
        store1<IN>(a.q_out, w + half, y * c + x * sn);
    } else if (!is_v) {
        head -= qn;
        const long long o = row * a.kr + head * a.kh + i, w = page * a.c.kp + slot * a.c.ks + head * a.c.kh + i;
        const float x = load1<IN>(a.k, o), y = load1<IN>(a.k, o + half);
        store1<KV>(a.c.k, w, x * c - y * sn);
        store1<KV>(a.c.k, w + half, y * c + x * sn);
    } else {
        head -= qn + a.c.kv_heads;
        const long long o = row * a.vr + head * a.vh + i, w = page * a.c.vp + slot * a.c.vs + head * a.c.vh + i;
        store1<KV>(a.c.v, w, load1<IN>(a.v, o));
        store1<KV>(a.c.v, w + half, load1<IN>(a.v, o + half));
    }
}

// one wave per (row, query head): keys one after the other, a running maximum and sum (the softmax in one pass)
template <typename QT, typename KV, typename OT>
__global__ __launch_bounds__(64) void paged_attention_kernel(PagedAttnArgs a) {
    const int row = blockIdx.x / a.q_heads, h = blockIdx.x % a.q_heads, lane = threadIdx.x;
    const int hk = h / (a.q_heads / a.c.kv_heads), per = a.c.head_dim >> 6;
    int n = a.lengths[row];
    if (n < 0) return;
    n += a.length_add;
    const long long most = (long long)a.c.max_pages << a.c.page_shift;
    if (n > most) n = (int)most;
    const int s = a.seq ? a.seq[row] : row;
    if (s < 0 || s >= a.c.n_seqs) n = 0;
    const int first = a.starts ? max(a.starts[row], 0) : 0;
    float q[2] = {0.f, 0.f}, acc[2] = {0.f, 0.f}, m = -INFINITY, l = 0.f;
    for (int e = 0; e < per; ++e) q[e] = load1<QT>(a.q, row * a.qr + h * a.qh + e * 64 + lane);
    for (int j = first; j < n; ++j) {
        const int page = page_of(a.c, s, j);
        if (page < 0) continue;
        const int slot = j & ((1 << a.c.page_shift) - 1);
        float dot = 0.f;
        for (int e = 0; e < per; ++e) dot += q[e] * load1<KV>(a.c.k, page * a.c.kp + slot * a.c.ks + hk * a.c.kh + e * 64 + lane);
        for (int o = 32; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
        dot *= a.scale;
        const float mn = fmaxf(m, dot), ref = mn > -INFINITY ? mn : 0.f, keep = expf(m - ref), p = expf(dot - ref);
        l = l * keep + p;
        for (int e = 0; e < per; ++e) acc[e] = acc[e] * keep + p * load1<KV>(a.c.v, page * a.c.vp + slot * a.c.vs + hk * a.c.vh + e * 64 + lane);
        m = mn;
    }
    for (int e = 0; e < per; ++e) store1<OT>(a.out, row * a.outr + h * a.outh + e * 64 + lane, l > 0.f ? acc[e] / l : 0.f);
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s) {
    const long long total = (long long)a.rows * ((a.q ? a.q_heads : 0) + 2 * a.c.kv_heads) * (a.c.head_dim / 2);
    if (a.rows <= 0 || (total + 255) / 256 > 0x7FFFFFFFLL) return hipErrorInvalidValue;
    const dim3 grid((unsigned)((total + 255) / 256)), block(256);
    if (a.in_bf16 && a.c.bf16) hipLaunchKernelGGL((paged_append_kernel<uint16_t, uint16_t>), grid, block, 0, s, a);
    else if (a.in_bf16) hipLaunchKernelGGL((paged_append_kernel<uint16_t, float>), grid, block, 0, s, a);
    else if (a.c.bf16) hipLaunchKernelGGL((paged_append_kernel<float, uint16_t>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((paged_append_kernel<float, float>), grid, block, 0, s, a);
    return hipGetLastError();
}

template <typename QT, typename KV>
static void launch_attention_o(const PagedAttnArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)(a.rows * a.q_heads)), block(64);
    if (a.out_bf16) hipLaunchKernelGGL((paged_attention_kernel<QT, KV, uint16_t>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((paged_attention_kernel<QT, KV, float>), grid, block, 0, s, a);
}

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t s) {
    if (a.rows <= 0 || (long long)a.rows * a.q_heads > 0x7FFFFFFFLL) return hipErrorInvalidValue;
    if (a.q_bf16) launch_attention_o<uint16_t, uint16_t>(a, s);
    else if (a.c.bf16) launch_attention_o<float, uint16_t>(a, s);
    else launch_attention_o<float, float>(a, s);
    return hipGetLastError();
}

}  // namespace t3k
