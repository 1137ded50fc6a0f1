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

constexpr int kListed = 16384;      // tokens of a row that are sorted by chunk (longer lists are walked whole for every chunk)
constexpr int kMaxRun = 64;         // chunks of a block
constexpr int kBiasShift = 20;      // note of an entry: occurrences in the low 20 bits, 1 + index of its bias above

// sixteen bytes at any element address (the memory unit needs no more than the element's alignment)
template <typename T> struct Piece;
template <> struct Piece<float> {
    static constexpr int N = 4;
    typedef float V __attribute__((ext_vector_type(4), aligned(4)));
    __device__ static __forceinline__ V load(const void* p, long long i) { return *reinterpret_cast<const V*>(static_cast<const float*>(p) + i); }
    __device__ static __forceinline__ float value(const V& v, int k) { return v[k]; }
    __device__ static __forceinline__ void put1(V& v, int k, const void* p, long long i) { v[k] = static_cast<const float*>(p)[i]; }
    __device__ static __forceinline__ void store(void* p, long long i, const float (&o)[4]) {
        *reinterpret_cast<V*>(static_cast<float*>(p) + i) = V{o[0], o[1], o[2], o[3]};
    }
    __device__ static __forceinline__ void store1(void* p, long long i, float v) { static_cast<float*>(p)[i] = v; }
};
template <> struct Piece<uint16_t> {
    static constexpr int N = 8;
    typedef unsigned V __attribute__((ext_vector_type(4), aligned(2)));
    __device__ static __forceinline__ V load(const void* p, long long i) { return *reinterpret_cast<const V*>(static_cast<const uint16_t*>(p) + i); }
    __device__ static __forceinline__ float value(const V& v, int k) { return __uint_as_float(k & 1 ? v[k >> 1] & 0xFFFF0000u : v[k >> 1] << 16); }
    __device__ static __forceinline__ void put1(V& v, int k, const void* p, long long i) {
        const unsigned h = static_cast<const uint16_t*>(p)[i];
        v[k >> 1] = k & 1 ? (v[k >> 1] & 0xFFFFu) | h << 16 : h;
    }
    __device__ static __forceinline__ void store(void* p, long long i, const float (&o)[8]) {
        V v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (unsigned)bf16_bits(o[2 * k]) | (unsigned)bf16_bits(o[2 * k + 1]) << 16;
        *reinterpret_cast<V*>(static_cast<uint16_t*>(p) + i) = v;
    }
    __device__ static __forceinline__ void store1(void* p, long long i, float v) { static_cast<uint16_t*>(p)[i] = bf16_bits(v); }
};

// a barrier for what the block shares in LDS: loads from memory stay in flight across it
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// n ids dealt to the TH threads of a block, 16 of a thread asked for at a time (one walk over a few thousand is one memory latency);
// HOLD: the first 16 are kept for the next walk
template <int TH, bool HOLD> struct IdList {
    int held[16];
    const int* ids;
    int n;
    __device__ __forceinline__ void load(int at, int (&x)[16]) const {
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int j = at + k * TH + (int)threadIdx.x;
            x[k] = -1;
            if (at + k * TH < n) {                       // (block-uniform)
                const int v = ids[min(j, n - 1)];
                x[k] = j < n ? v : -1;
            }
        }
    }
    __device__ __forceinline__ void take(const int* p, int count) {
        ids = p;
        n = count;
        if (HOLD) load(0, held);
    }
    template <typename F> __device__ __forceinline__ void each(F f) const {
        for (int at = 0; at < n; at += TH * 16) {
            int x[16];
            if (HOLD && at == 0) {
#pragma unroll
                for (int k = 0; k < 16; ++k) x[k] = held[k];
            } else {
                load(at, x);
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                if (at + k * TH >= n) break;
                f(x[k]);
            }
        }
    }
};

// Chunks [c0, c1) of CH entries of one row, one after the other, TH threads.  Bound: the logits are read and written once (256 rows of 131072
// fp32 entries with 2000 tokens, 300 biases and a mask each: 54.7 us in the kernel, 5.0 TB/s); everything else is kept off that stream.  The entries go to LDS as they arrive, the next
// chunk's already asked for.  How often each entry occurs among the row's tokens and which bias names it is noted in LDS (integer atomics: the
// result does not depend on their order; of two biases with one id the later counts).  Few entries have a note: a second walk over the
// tokens and biases lets the first thread that comes to one take the note (which leaves it clear for the next chunk) and change the
// entry in place, so that the division and the bias are paid for those alone; then the entries leave, masked, in whole pieces.
struct LogitsLds {
    float* val;
    uint32_t* note;
    uint16_t* listed;       // the row's tokens by chunk, as places in it
    int *from, *fill;
};
template <typename T, int CH, int TH, bool MANY, bool TAIL>
__device__ __forceinline__ void process_chunks(const LogitsArgs& a, const LogitsLds& sm, int c0, int c1) {
    using P = Piece<T>;
    constexpr int N = P::N, PER = CH / (TH * N);
    static_assert(PER * TH * N == CH && CH % (TH * 4) == 0, "whole pieces");
    float* const val = sm.val;
    uint32_t* const note = sm.note;
    uint16_t* const listed = sm.listed;
    int *const from = sm.from, *const fill = sm.fill;
    const long long row = blockIdx.y;
    const int tid = threadIdx.x;
    // a piece of the row as it comes from memory; what lies past the row's end is not read
    typename P::V x[PER], u[PER];
    uint32_t bits[PER];
    const auto ask = [&](int c) {
        if constexpr (!TAIL) {
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const int i = c * CH + (k * TH + tid) * N;
                x[k] = P::load(a.logits, row * a.lr + i);
                if (a.uncond) u[k] = P::load(a.uncond, row * a.ur + i);
                if (a.allowed) bits[k] = a.allowed[row * a.ar + (i >> 5)];   // N divides 32: a piece's bits are in one word
            }
        } else {                                         // the row ends in this chunk: past its end its last entry is read instead
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const int i = c * CH + (k * TH + tid) * N;
                x[k] = u[k] = typename P::V{};
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const int e = min(i + q, a.vocab - 1);
                    P::put1(x[k], q, a.logits, row * a.lr + e);
                    if (a.uncond) P::put1(u[k], q, a.uncond, row * a.ur + e);
                }
                if (a.allowed) bits[k] = a.allowed[row * a.ar + (min(i, a.vocab - 1) >> 5)];
            }
        }
        __builtin_amdgcn_sched_barrier(0);               // asked for here, not where it is used
    };
    ask(c0);
    const int n_tok = a.tokens ? min(max(a.n_tokens[row], 0), a.cap) : 0;
    const bool notes = n_tok > 0 || a.n_bias > 0;   // (block-uniform)
    int bid = -1;                                    // the first TH biases are held, a longer list is read again for every chunk
    float bval = 0.f;
    IdList<TH, true> tok;
    float rep = 1.f, fre = 0.f, pre = 0.f;
    if (notes) {
        tok.take(a.tokens + row * a.tr, n_tok);
        rep = a.repetition ? a.repetition[row] : a.repetition_s;
        fre = a.frequency ? a.frequency[row] : a.frequency_s;
        pre = a.presence ? a.presence[row] : a.presence_s;
        if (tid < a.n_bias) {
            bid = a.bias_ids[row * a.br + tid];
            bval = a.bias_values[row * a.bvr + tid];
        }
#pragma unroll
        for (int i = 0; i < CH / (TH * 4); ++i) *reinterpret_cast<uint4*>(&note[(i * TH + tid) * 4]) = uint4{0u, 0u, 0u, 0u};
    }
    // a block of several chunks sorts the tokens by chunk first: each chunk then walks its own few, not the whole list (the call in
    // launch_logits: 79 us without it, 53 with)
    const bool sorted = MANY && n_tok > 0 && n_tok <= kListed;
    if (sorted) {
        if (tid < kMaxRun) fill[tid] = 0;
        lds_barrier();
        tok.each([&](int t) {
            const unsigned v = (unsigned)t - (unsigned)(c0 * CH);
            if (v / CH < (unsigned)(c1 - c0) && t < a.vocab) atomicAdd(&fill[v / CH], 1);
        });
        lds_barrier();
        if (tid < 64) {                              // kMaxRun = 64: a lane each; where each chunk's tokens begin
            const int count = fill[tid];
            int at = count;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int left = __shfl_up(at, d, 64);
                if (tid >= d) at += left;
            }
            if (tid == 0) from[0] = 0;
            from[tid + 1] = at;
            fill[tid] = at - count;
        }
        lds_barrier();
        tok.each([&](int t) {
            const unsigned v = (unsigned)t - (unsigned)(c0 * CH);
            if (v / CH < (unsigned)(c1 - c0) && t < a.vocab) listed[atomicAdd(&fill[v / CH], 1)] = (uint16_t)(v % CH);
        });
    }
    for (int c = c0; c < c1; ++c) {              // (one turn without MANY)
        const int v0 = c * CH;
        const unsigned nv = (unsigned)min(CH, a.vocab - v0);
        float z[PER][N];
        uint32_t allow[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            allow[k] = a.allowed ? bits[k] >> (((k * TH + tid) * N) & 31) : 0u;
#pragma unroll
            for (int q = 0; q < N; ++q) {
                z[k][q] = P::value(x[k], q);
                if (a.uncond) z[k][q] = z[k][q] + a.cfg_weight * (z[k][q] - P::value(u[k], q));
            }
        }
        if (MANY) ask(min(c + 1, c1 - 1));           // (the last chunk once more, not used: no branch around the loads, or the loop would wait for them)
        if (notes) {
            if (c == c0) lds_barrier();          // the notes are clear, the tokens sorted (later chunks: since the last barrier)
            if (a.n_bias > 0) {
                const auto mark = [&](int j, int id) {
                    const unsigned v = (unsigned)id - (unsigned)v0;
                    if (v < nv) atomicMax(&note[v], (uint32_t)(j + 1) << kBiasShift);
                };
                mark(tid, bid);
                for (int j = tid + TH; j < a.n_bias; j += TH) mark(j, a.bias_ids[row * a.br + j]);
                lds_barrier();
            }
            // f of the place of every token in this chunk
            const auto each_here = [&](auto f) {
                if (sorted) {
                    for (int j = from[c - c0] + tid; j < from[c - c0 + 1]; j += TH) f((unsigned)listed[j]);
                } else {
                    tok.each([&](int t) {
                        const unsigned v = (unsigned)t - (unsigned)v0;
                        if (v < nv) f(v);
                    });
                }
            };
            each_here([&](unsigned v) { atomicAdd(&note[v], 1u); });
#pragma unroll
            for (int k = 0; k < PER; ++k)
#pragma unroll
                for (int q = 0; q < N; q += 4) *reinterpret_cast<float4*>(&val[(k * TH + tid) * N + q]) = float4{z[k][q], z[k][q + 1], z[k][q + 2], z[k][q + 3]};
            lds_barrier();
            // an entry with a bias is changed by the thread that holds that bias, any other by the first that comes to it
            const auto penalise = [&](float y, uint32_t count) {
                if (count) {
                    y = y > 0.f ? y / rep : y * rep;
                    y = y - fre * (float)count - pre;
                }
                return y;
            };
            each_here([&](unsigned v) {
                if ((note[v] >> kBiasShift) != 0u) return;
                const uint32_t w = atomicExch(&note[v], 0u);
                if (w != 0u) val[v] = penalise(val[v], w);
            });
            if (a.n_bias > 0) {
                // (the value of a bias beyond the first TH is read where it is used: the common path then waits for no load)
                const auto add = [&](int j, int id, auto value) {
                    const unsigned v = (unsigned)id - (unsigned)v0;
                    if (v >= nv) return;
                    const uint32_t w = note[v];
                    if ((w >> kBiasShift) != (uint32_t)(j + 1)) return;
                    val[v] = penalise(val[v] + value(), w & ((1u << kBiasShift) - 1));
                    note[v] = 0u;
                };
                add(tid, bid, [&] { return bval; });
                for (int j = tid + TH; j < a.n_bias; j += TH) add(j, a.bias_ids[row * a.br + j], [&] { return a.bias_values[row * a.bvr + j]; });
            }
            lds_barrier();
#pragma unroll
            for (int k = 0; k < PER; ++k)
#pragma unroll
                for (int q = 0; q < N; q += 4) {
                    const float4 y = *reinterpret_cast<const float4*>(&val[(k * TH + tid) * N + q]);
                    z[k][q] = y.x; z[k][q + 1] = y.y; z[k][q + 2] = y.z; z[k][q + 3] = y.w;
                }
        }
        if (a.allowed) {
#pragma unroll
            for (int k = 0; k < PER; ++k)
#pragma unroll
                for (int q = 0; q < N; ++q) z[k][q] = (allow[k] >> q) & 1u ? z[k][q] : -INFINITY;
        }
        if constexpr (!TAIL) {
#pragma unroll
            for (int k = 0; k < PER; ++k) P::store(a.out, row * a.outr + v0 + (k * TH + tid) * N, z[k]);
        } else {
#pragma unroll
            for (int k = 0; k < PER; ++k)
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const int i = v0 + (k * TH + tid) * N + q;
                    if (i < a.vocab) P::store1(a.out, row * a.outr + i, z[k][q]);
                }
        }
    }
}

// blocks of the row's whole chunks, `run` each (MANY) or one, and one more for the chunk in which the row ends
template <typename T, int CH, int TH, bool MANY>
__global__ __launch_bounds__(TH) void process_logits_kernel(LogitsArgs a, int run) {
    __shared__ __attribute__((aligned(16))) float val[CH];
    __shared__ __attribute__((aligned(16))) uint32_t note[CH];
    __shared__ uint16_t listed[MANY ? kListed : 1];
    __shared__ int from[kMaxRun + 1], fill[kMaxRun];
    const LogitsLds sm = {val, note, listed, from, fill};
    const int whole = a.vocab / CH, c0 = blockIdx.x * (MANY ? run : 1);
    if (c0 < whole) process_chunks<T, CH, TH, MANY, false>(a, sm, c0, MANY ? min(c0 + run, whole) : c0 + 1);
    else process_chunks<T, CH, TH, false, true>(a, sm, whole, whole + 1);
}

template <typename T> void launch_logits(const LogitsArgs& a, hipStream_t s) {
    constexpr int CH = 4096, TH = 512;
    // Blocks of a row: two blocks fit a CU at a time (LDS), 512 the chip; the time goes as the rounds they make times the chunks of one,
    // and a block starts for about three chunks' time (it sorts the row's tokens).  256 rows of 131072 fp32 entries with 2000 tokens,
    // 300 biases and a mask each, 20 calls in a row over four inputs, 1 / 2 / 3 / 4 blocks a row: 75 / 53 / 64 / 64 us; a block for every chunk, unsorted: 79.
    const int whole = a.vocab / CH;
    int run = 1;
    if ((long long)whole * a.rows > 512) {
        long long best = -1;
        for (int nb = 1; nb <= whole && nb <= 64; ++nb) {
            const int r = (whole + nb - 1) / nb;
            if (r > kMaxRun) continue;
            const long long time = ((long long)a.rows * nb + 511) / 512 * (r + 3);
            if (best < 0 || time < best) { best = time; run = r; }
        }
        if (best < 0) run = kMaxRun;
    }
    const dim3 grid((unsigned)((whole + run - 1) / run) + (a.vocab % CH ? 1u : 0u), (unsigned)a.rows);
    if (run > 1) hipLaunchKernelGGL((process_logits_kernel<T, CH, TH, true>), grid, dim3(TH), 0, s, a, run);
    else hipLaunchKernelGGL((process_logits_kernel<T, CH, TH, false>), grid, dim3(TH), 0, s, a, 1);
}

}  // namespace

hipError_t launch_process_logits(const LogitsArgs& a, hipStream_t s) {
    if (a.rows <= 0 || a.rows > 65535 || a.vocab <= 0) return hipErrorInvalidValue;
    if (a.bf16) launch_logits<uint16_t>(a, s);
    else launch_logits<float>(a, s);
    return hipGetLastError();
}

}  // namespace t3k
