// The rules a logits row goes through before it is sampled: guidance, biases, penalties for repeated tokens, allowed tokens.
#include <hip/hip_runtime.h>

#include <cmath>

#include "ops_kernels.hpp"

namespace t3k {
namespace {

__device__ __forceinline__ float bf16_value(uint16_t h) { return __uint_as_float((uint32_t)h << 16); }
__device__ __forceinline__ uint16_t bf16_bits(float f) {   // to the nearest, ties to even; NaN stays NaN
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

constexpr int kChunk = 4096;        // vocabulary entries of a block
constexpr int kThreads = 256;
constexpr int kBiasShift = 20;      // note word of an entry: occurrences in the low 20 bits, 1 + index of its bias above

// A block owns kChunk entries of one row.  It notes, in LDS, how often each of them occurs among the row's tokens and which bias names
// it (integer atomics: the result does not depend on their order; of two biases with one id the later counts), then makes one pass
// over the entries.
template <typename T>
__global__ __launch_bounds__(kThreads) void process_logits_kernel(LogitsArgs a) {
    __shared__ uint32_t note[kChunk];
    const int row = blockIdx.y, v0 = blockIdx.x * kChunk, tid = threadIdx.x;
    const int nv = min(kChunk, a.vocab - v0);
    for (int i = tid; i < kChunk; i += kThreads) note[i] = 0u;
    __syncthreads();
    for (int j = tid; j < a.n_bias; j += kThreads) {
        const int v = a.bias_ids[row * a.br + j] - v0;
        if (v >= 0 && v < nv) atomicMax(&note[v], (uint32_t)(j + 1) << kBiasShift);
    }
    __syncthreads();
    if (a.tokens) {
        const int n = min(max(a.n_tokens[row], 0), a.cap);
        for (int j = tid; j < n; j += kThreads) {
            const int v = a.tokens[row * a.tr + j] - v0;
            if (v >= 0 && v < nv) atomicAdd(&note[v], 1u);
        }
    }
    __syncthreads();
    const float rep = a.repetition ? a.repetition[row] : a.repetition_s;
    const float fre = a.frequency ? a.frequency[row] : a.frequency_s;
    const float pre = a.presence ? a.presence[row] : a.presence_s;
    for (int i = tid; i < nv; i += kThreads) {
        const int v = v0 + i;
        float z, u = 0.f;
        if constexpr (sizeof(T) == 2) {
            z = bf16_value(static_cast<const uint16_t*>(a.logits)[row * a.lr + v]);
            if (a.uncond) u = bf16_value(static_cast<const uint16_t*>(a.uncond)[row * a.ur + v]);
        } else {
            z = static_cast<const float*>(a.logits)[row * a.lr + v];
            if (a.uncond) u = static_cast<const float*>(a.uncond)[row * a.ur + v];
        }
        if (a.uncond) z = z + a.cfg_weight * (z - u);
        const uint32_t w = note[i], bias = w >> kBiasShift, count = w & ((1u << kBiasShift) - 1);
        if (bias) z += a.bias_values[row * a.bvr + bias - 1];
        if (count) {
            z = z > 0.f ? z / rep : z * rep;
            z = z - fre * (float)count - pre;
        }
        if (a.allowed && !((a.allowed[row * a.ar + (v >> 5)] >> (v & 31)) & 1u)) z = -INFINITY;
        if constexpr (sizeof(T) == 2) static_cast<uint16_t*>(a.out)[row * a.outr + v] = bf16_bits(z);
        else static_cast<float*>(a.out)[row * a.outr + v] = z;
    }
}

}  // namespace

hipError_t launch_process_logits(const LogitsArgs& a, hipStream_t s) {
    if (a.rows <= 0 || a.rows > 65535 || a.vocab <= 0) return hipErrorInvalidValue;
    const dim3 grid((unsigned)((a.vocab + kChunk - 1) / kChunk), (unsigned)a.rows);
    if (a.bf16) hipLaunchKernelGGL(process_logits_kernel<uint16_t>, grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL(process_logits_kernel<float>, grid, dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace t3k
