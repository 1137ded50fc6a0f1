// Paged key-value cache: the append of new keys and values (with the rotary position embedding applied on the way) and the
// attention of new tokens' query rows over the pages.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

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

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // sixteen bytes at a float's address
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// N neighbouring values as floats: 16 bytes of the type that comes in (N = 4 floats or 8 bf16), any type going out
template <typename T, int N> __device__ __forceinline__ void load_row(const void* p, long long at, float (&x)[N]) {
    if constexpr (sizeof(T) == 2) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
    } else {
        const f32x4 w = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = w[i];
    }
}
template <typename T, int N> __device__ __forceinline__ void store_row(void* p, long long at, const float (&x)[N]) {
    if constexpr (sizeof(T) == 2) {
        unsigned w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = (unsigned)to_bf16(x[2 * i]) | (unsigned)to_bf16(x[2 * i + 1]) << 16;
        uint16_t* o = static_cast<uint16_t*>(p) + at;
        if constexpr (N == 8) *reinterpret_cast<u32x4*>(o) = u32x4{w[0], w[1], w[2], w[3]};
        else *reinterpret_cast<u32x2*>(o) = u32x2{w[0], w[1]};
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) *reinterpret_cast<f32x4*>(static_cast<float*>(p) + at + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
    }
}

// page of key j of sequence s, or -1: outside the table, or an entry that names no page of the pool
__device__ __forceinline__ int page_of(const PagedCache& c, int s, int j) {
    const int e = j >> c.page_shift;
    if (e >= c.max_pages) return -1;
    const int p = c.table[(long long)s * c.table_stride + e];
    return p >= 0 && p < c.n_pages ? p : -1;
}

// A thread takes 16 bytes of the first half of a head of q, k or v and the 16 bytes that turn with them in the second half:
// (a, b) -> (a cos - b sin, b cos + a sin) in fp32, rounded once.  Bound: every value is read and written once; the angles come from
// L2 (the heads of a row share them), so the kernel is a copy with a permutation of rows.
template <typename IN, typename KV, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
    constexpr int N = 16 / sizeof(IN), H = D / 2, UN = H / N;   // values of a piece, of a half, pieces of a half
    const unsigned heads = (unsigned)(a.q_heads + 2 * a.c.kv_heads);
    const unsigned idx = blockIdx.x * 256u + threadIdx.x;
    const unsigned hr = idx / UN;
    const int i = (int)(idx % UN) * N;
    const unsigned row = hr / heads;
    if (row >= (unsigned)a.rows) return;
    int head = (int)(hr - row * heads);
    const int pos = a.positions[row], s = a.seq ? a.seq[row] : (int)row;
    if (pos < 0 || s < 0 || s >= a.c.n_seqs || (a.cos && pos >= a.rope_len)) return;
    const int page = page_of(a.c, s, pos);
    if (page < 0) return;
    const int slot = pos & ((1 << a.c.page_shift) - 1);
    float x[N], y[N];
    if (head >= a.q_heads + a.c.kv_heads) {
        head -= a.q_heads + a.c.kv_heads;
        const long long o = row * a.vr + head * a.vh + i, w = page * a.c.vp + slot * a.c.vs + head * a.c.vh + i;
        load_row<IN, N>(a.v, o, x);
        load_row<IN, N>(a.v, o + H, y);
        store_row<KV, N>(a.c.v, w, x);
        store_row<KV, N>(a.c.v, w + H, y);
        return;
    }
    const bool is_q = head < a.q_heads;
    if (!is_q) head -= a.q_heads;
    const long long o = is_q ? row * a.qr + head * a.qh + i : row * a.kr + head * a.kh + i;
    load_row<IN, N>(is_q ? a.q : a.k, o, x);
    load_row<IN, N>(is_q ? a.q : a.k, o + H, y);
    if (a.cos) {
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            const f32x4 c = *reinterpret_cast<const f32x4u*>(a.cos + pos * a.rope_stride + i + e), sn = *reinterpret_cast<const f32x4u*>(a.sin + pos * a.rope_stride + i + e);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float p = x[e + k], r = y[e + k];
                x[e + k] = p * c[k] - r * sn[k];
                y[e + k] = r * c[k] + p * sn[k];
            }
        }
    }
    if (is_q) {
        const long long w = row * a.qor + head * a.qoh + i;
        store_row<IN, N>(a.q_out, w, x);
        store_row<IN, N>(a.q_out, w + H, y);
    } else {
        const long long w = page * a.c.kp + slot * a.c.ks + head * a.c.kh + i;
        store_row<KV, N>(a.c.k, w, x);
        store_row<KV, N>(a.c.k, w + H, y);
    }
}

// four neighbouring results of a head: the weighted sum over the sum of weights, zero where no key was seen
__device__ __forceinline__ void store_out(const PagedAttnArgs& a, int row, int h, int d, f32x4 o, float sum) {
    const long long at = (long long)row * a.outr + (long long)h * a.outh + d;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = sum == 0.f ? 0.f : o[i] / sum;
    if (a.out_bf16) {
        const uint2 w = {(unsigned)to_bf16(o[0]) | (unsigned)to_bf16(o[1]) << 16, (unsigned)to_bf16(o[2]) | (unsigned)to_bf16(o[3]) << 16};
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = w;
    } else {
        *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + at) = o;
    }
}

// ---- attention -----------------------------------------------------------------------------------------------------------------
// o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(x_j - max x),  x_j = scale log2(e) q . k_j.  Bound: every live key and value is read once from
// HBM (4 G flop for each pair of elements, G query heads to a key head: far below the matrix rate), so the kernel is built around loads.
// A wave takes 32 keys at a time of one key head for up to 16 of its query heads:
//   S^T = K Q^T   (A: 16 keys x head_dim, straight from memory to the registers the matrix instruction takes; B: the queries, resident)
//   O^T += V^T P  (B: the 8 weights a lane holds after the softmax are already its operand: lane (query n, group g) has keys 4 g + i of both
//                  16-key tiles, and the sum over keys may run in any order; A: a lane loads D / 16 neighbouring values of each of
//                  these 8 keys -- whole rows of the cache to an instruction -- and turns the 8 x D/16 block in its registers)
// so neither K nor V passes through LDS.  The next 32 keys are requested as soon as their registers are free: keys after the first
// product, values after the second, one tile in flight per wave all the time.  Waves of a block take every nw-th tile and meet in LDS;
// blocks of a row (split) leave (max, sum, weighted sum) in the workspace for paged_join_kernel.
// Types: bf16 operands go to the bf16 matrix instruction.  An fp32 query over a bf16 cache is cut into three bf16 parts of 8 significant
// bits each, which hold it exactly, and so are the weights when the result is fp32.  Under a bf16 result a weight is two rounded parts, 2^-16 of it off
// at most: a 256th of what the result's own rounding may be off.  (One part would be off by as much as the result: its error against 64 bits 1.77e-3
// instead of 1.68e-3 over 3 rows of 100003 to 131071 keys.)  An fp32 cache uses the exact fp32 matrix instruction.  Sums, maxima and products: fp32.
// Parts and infinities: a part of an ordinary number may be 0, and 0 times an infinite key or value is NaN where the number itself gives an infinity.  A wave
// whose sums end as NaN goes through its keys a second time (whole_pass) and takes the columns concerned from products of whole numbers: NaN that the
// formula has comes out again, anything else as it should be.  Nothing is looked for on the way: finite keys and values pay for one test at the end.

// over the four 16-lane groups of a wave (lanes n, n + 16, n + 32, n + 48), by register swaps
template <typename F> __device__ __forceinline__ float over_groups(float x, F f) {
    const unsigned u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned w = __float_as_uint(f(__uint_as_float(a[0]), __uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane16_swap(w, w, false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float group_max(float x) { return over_groups(x, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float group_sum(float x) { return over_groups(x, [](float a, float b) { return a + b; }); }

// the leading 8 significant bits of x; what is left over is x - lead(x), exactly
__device__ __forceinline__ float lead(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u); }

// eight floats as bf16 vectors: three parts of 8 significant bits, which hold them exactly, or two rounded ones, off by at most 2^-16 of the value.  INF:
// there may be infinities among them (which are their first part)
template <int PARTS, bool INF = false> __device__ __forceinline__ void to_parts(const float (&x)[8], bf16x8 (&o)[PARTS]) {
    static_assert(PARTS == 2 || PARTS == 3, "two parts or three");
    if constexpr (PARTS == 2) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            o[0][j] = (__bf16)x[j];
            o[1][j] = (__bf16)(x[j] - (float)o[0][j]);
        }
    } else {
        float r[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) r[j] = x[j];
#pragma unroll
        for (int s = 0; s < PARTS; ++s) {
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = __builtin_amdgcn_perm(__float_as_uint(r[2 * j + 1]), __float_as_uint(r[2 * j]), 0x07060302u);
                if (s + 1 < PARTS) {
#pragma unroll
                    for (int i = 2 * j; i < 2 * j + 2; ++i) r[i] = INF && r[i] == lead(r[i]) ? 0.f : r[i] - lead(r[i]);
                }
            }
            o[s] = __builtin_bit_cast(bf16x8, w);
        }
    }
}

__device__ __forceinline__ float bf16_of(unsigned w, int half) { return __uint_as_float(half ? w & 0xFFFF0000u : w << 16); }

// whether a wave's vote is set for this lane's column (lane & 15) in any of its four groups
__device__ __forceinline__ bool in_column(unsigned long long vote, int n) {
    vote |= vote >> 32;
    return ((vote | vote >> 16) >> n) & 1u;
}

// The sums of a wave over a bf16 cache from whole fp32 numbers: tiles t, t + step, ... below t_end of the sequence whose pages are trow, no key from hi on.
// Column n (its queries cut into the parts qb, which add up to them) sees the keys [first, len); the columns of a row are `group` neighbours.
// m, l, acc: maximum, sum and weighted sum so far, laid out as in the kernels below.  Rare, so built for size: a tile at a time, a row at a time.
template <int QS, int KC, int NT, typename VT>
__device__ __forceinline__ void whole_pass(const PagedCache& c, const char* kbase, const char* vbase, const int* trow, const bf16x8 (&qb)[QS][KC], float scale2, int t,
                                           int t_end, int step, int hi, int first, int len, int group, float& m, float& l, f32x4 (&acc)[NT]) {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, in_page = (1 << c.page_shift) - 1;
    for (; t < t_end; t += step) {
        f32x4 s[2];
        VT vr[8];
        unsigned ok = 0u;                            // bit j: key j of this lane's values has a page
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int key = min(t * 32 + 16 * u + n, hi - 1), id = trow[key >> c.page_shift];
            const char* base = kbase + ((long long)(id >= 0 && id < c.n_pages ? id : 0) * c.kp + (long long)(key & in_page) * c.ks) * 2 + 16 * g;
            s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < KC; ++x) {
                const u32x4 kr = *reinterpret_cast<const u32x4*>(base + 64 * x);
                u32x4 qw[QS];
#pragma unroll
                for (int part = 0; part < QS; ++part) {
                    qw[part] = __builtin_bit_cast(u32x4, qb[part][x]);
                    asm volatile("" : "+v"(qw[part]));   // (put together here, not kept whole for all tiles: registers)
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float q = bf16_of(qw[QS - 1][j >> 1], j & 1);
#pragma unroll
                    for (int part = QS - 2; part >= 0; --part) q += bf16_of(qw[part][j >> 1], j & 1);
                    s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(bf16_of(kr[j >> 1], j & 1), q, s[u], 0, 0, 0);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);           // (values after the scores: registers)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int at = t * 32 + 16 * (j >> 2) + 4 * g + (j & 3), key = min(at, hi - 1), id = trow[key >> c.page_shift];
            const bool good = id >= 0 && id < c.n_pages;
            ok |= good && at < hi ? 1u << j : 0u;
            vr[j] = *reinterpret_cast<const VT*>(vbase + ((long long)(good ? id : 0) * c.vp + (long long)(key & in_page) * c.vs) * 2 + sizeof(VT) * n);
        }
        float p[8], mx = m;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int key = t * 32 + 16 * (j >> 2) + 4 * g + (j & 3);
            p[j] = ((ok >> j) & 1u) && key >= first && key < len ? s[j >> 2][j & 3] * scale2 : -INFINITY;
            mx = fmaxf(mx, p[j]);
        }
        mx = group_max(mx);
        const float ref = mx > -INFINITY ? mx : 0.f, keep = m == mx ? 1.f : __builtin_amdgcn_exp2f(m - ref);
        m = mx;
        l *= keep;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            p[j] = p[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(p[j] - ref);
            l += p[j];
        }
#pragma unroll
        for (int e = 0; e < NT; ++e) acc[e] *= keep;
        for (int r = 0; r * group < 16; ++r) {
            const int f_r = __builtin_amdgcn_readlane(first, r * group), l_r = __builtin_amdgcn_readlane(len, r * group);
            unsigned of = 0u;                        // the keys that row r sees
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = t * 32 + 16 * (j >> 2) + 4 * g + (j & 3);
                of |= key >= f_r && key < l_r ? (ok >> j & 1u) << j : 0u;
            }
            if (__builtin_amdgcn_ballot_w64(of != 0u) == 0) continue;
#pragma unroll
            for (int e = 0; e < NT; ++e) {
                f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    o = __builtin_amdgcn_mfma_f32_16x16x4f32((of >> j) & 1u ? bf16_of(vr[j][e >> 1], e & 1) : 0.f, p[j], o, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[e][i] += n / group == r ? o[i] : 0.f;
            }
        }
    }
}

// from 2^16 up, but finite (a column of an infinite maximum comes out as NaN either way, and does not change how its neighbours are rounded)
__device__ __forceinline__ bool large(float x) { return (__float_as_uint(x) & 0x7FFFFFFFu) - 0x47800000u < 0x7F800000u - 0x47800000u; }

// the kernel's arguments, read again: what only a rare path needs of them is not kept in registers for it (the scalar registers that took cost every
// launch 0.6 us: the arguments' loads waited for each other)
__device__ __forceinline__ const PagedAttnArgs& arguments_again() {
    auto p = __builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const PagedAttnArgs*)p;
}

// what a part's sums count, its maximum being m and that of all parts top.  A part without a maximum saw no key, and its sums are 0, or it saw
// NaN scores alone, and they are NaN: taken as they are
__device__ __forceinline__ float part_factor(float m, float top) { return m > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : 1.f; }

constexpr int kMaxSplit = 64;      // blocks that share a row's keys at most

// which keys of a row a block works on: key tiles [t0, t1) of 1 << tile_shift, shared by `active` blocks of at most `per` tiles each
struct RowPlan {
    int first, len, t0, t1, per, active;
};
// len, first, s: the row's entries of lengths (>= 0), starts (or 0) and seq (or the row)
__device__ __forceinline__ RowPlan plan_row(const PagedAttnArgs& a, int len, int first, int s) {
    RowPlan p;
    long long n = (long long)len + a.length_add;
    const long long most = (long long)a.c.max_pages << a.c.page_shift;
    n = n > most ? most : n;
    p.first = max(first, 0);
    p.len = (s < 0 || s >= a.c.n_seqs) ? 0 : (int)n;
    p.t0 = p.first >> a.tile_shift;
    p.t1 = (p.len + (1 << a.tile_shift) - 1) >> a.tile_shift;
    const int tiles = p.len > p.first ? p.t1 - p.t0 : 0;
    if (tiles == 0) p.t1 = p.t0;
    const int want = min(a.n_split, (tiles + a.min_tiles - 1) / a.min_tiles);
    p.per = want > 0 ? (tiles + want - 1) / want : 1;
    p.active = tiles > 0 ? (tiles + p.per - 1) / p.per : 1;
    return p;
}

// QB, KB: bf16 queries, bf16 cache.  TK: keys of a tile, 32 or (fp32 cache) 16.  PAGES 0: pages of TK keys and more (a tile lies in one),
// 1: smaller ones of 4 keys and more, 2: of 1, 2.  PARTS: bf16 parts of a weight (bf16 cache only; otherwise 1).
template <bool QB, bool KB, int D, int TK, int PAGES, int PARTS>
__global__ __launch_bounds__(512, D == 64 ? (PAGES == 2 && KB && !QB ? 3 : 4) : (QB && PAGES == 1 ? 3 : 2)) void paged_attention_kernel(PagedAttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) float sm[];
    constexpr int EB = KB ? 2 : 4;                  // bytes of a cache element
    constexpr int KC = KB ? D / 32 : D / 16;        // 16-byte pieces of a key to a lane
    constexpr int VL = KB ? 1 : D / 64;             // loads of a value to a lane: D / 16 bf16 in one, or 4 floats of each 64
    constexpr int NT = D / 16;                      // 16 x 16 tiles of O^T
    constexpr int QS = QB ? 1 : 3;
    constexpr int U = TK / 16, J = 4 * U;           // 16-key halves of a tile, weights to a lane
    static_assert(TK == 32 || (TK == 16 && !KB), "the bf16 product takes 32 keys");
    using VT = std::conditional_t<KB && D == 64, u32x2, u32x4>;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    // waves: head_waves neighbouring key heads, and kw shares of each one's keys
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const int hw = a.head_waves, wh = wave % hw, wk = wave / hw, kw = nw / hw;
    const int group = a.q_heads / a.c.kv_heads, gt = (group + 15) >> 4, hg = (a.c.kv_heads + hw - 1) / hw;
    unsigned pair = blockIdx.x / (unsigned)a.n_split;
    const int q16 = (int)(pair % (unsigned)gt);
    pair /= (unsigned)gt;
    const int hk0 = (int)(pair % (unsigned)hg) * hw, row = (int)(pair / (unsigned)hg);
    // (a short row's last blocks have nothing to do: turned by the row, they do not all fall to the same XCDs.  128 rows of 60 to 4000 keys: 194 -> 181 us)
    const unsigned split = (blockIdx.x + (unsigned)row) % (unsigned)a.n_split;
    // what the row is, and its queries, are asked for together, before anything waits
    const int row_len = a.lengths[row], seq = a.seq ? a.seq[row] : row, row_first = a.starts ? a.starts[row] : 0;
    const int gn = min(16, group - q16 * 16);       // live query heads of a key head in this block
    const bool idle = hk0 + wh >= a.c.kv_heads;     // (a wave past the last key head: no tile, nothing stored)
    const int hk = idle ? a.c.kv_heads - 1 : hk0 + wh;
    const int h0 = hk * group + q16 * 16;

    // queries: lane (n, g) holds, for piece c, elements 32 c + 8 g + j (bf16 cache) or 16 c + 4 g + i (fp32 cache) of head n
    constexpr int QW = KB && !QB ? 2 : 1;           // 16-byte words of a piece
    u32x4 qw[KC][QW];
    {
        const long long qo = row * a.qr + (long long)(h0 + (n < gn ? n : 0)) * a.qh;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int w = 0; w < QW; ++w) {
                if constexpr (QB) qw[c][w] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + qo + 32 * c + 8 * g);
                else qw[c][w] = *reinterpret_cast<const u32x4*>(static_cast<const float*>(a.q) + qo + (KB ? 32 * c + 8 * g + 4 * w : 16 * c + 4 * g));
            }
    }
    if (row_len < 0) return;
    const RowPlan rp = plan_row(a, row_len, row_first, seq);
    if ((int)split >= rp.active) return;
    const int t_begin = rp.t0 + (int)split * rp.per, t_end = idle ? t_begin : min(rp.t1, t_begin + rp.per);
    // byte offsets of this lane inside a tile: keys 16 t + n, piece g; values of keys 16 t + 4 g + i, elements D / 16 * n (or 4 n)
    const unsigned ksb = (unsigned)a.c.ks * EB, vsb = (unsigned)a.c.vs * EB;
    const char* kbase = static_cast<const char*>(a.c.k) + (long long)hk * a.c.kh * EB;
    const char* vbase = static_cast<const char*>(a.c.v) + (long long)hk * a.c.vh * EB;
    const int* trow = a.c.table + (long long)(seq < 0 || seq >= a.c.n_seqs ? 0 : seq) * a.c.table_stride;
    const int in_page = (1 << a.c.page_shift) - 1;
    constexpr int NP = PAGES == 0 ? 1 : (PAGES == 1 ? 2 * U : U + J);   // page numbers of a tile: one; K and V of each 16; K of each 16, V of each key
    // key of page number x of tile t (clamped to the row's last: entries past it may hold anything)
    auto key_of = [&](int t, int x) {
        int k = t * TK;
        if (PAGES == 1) k += x < U ? 16 * x + n : 16 * (x - U) + 4 * g;
        if (PAGES == 2) k += x < U ? 16 * x + n : 16 * ((x - U) >> 2) + 4 * g + ((x - U) & 3);
        return PAGES == 0 ? k : min(k, rp.len - 1);
    };
    int ids[NP];
    auto ask = [&](int t) {
#pragma unroll
        for (int x = 0; x < NP; ++x) ids[x] = trow[key_of(t, x) >> a.c.page_shift];
    };
    u32x4 kr[U][KC];
    VT vr[J][VL];
    // what the loads of a tile need: page numbers clamped into the pool, and whether they were in it
    struct Pages { int id[NP]; bool ok; };
    auto settle = [&]() {
        Pages p;
        p.ok = true;
#pragma unroll
        for (int x = 0; x < NP; ++x) {
            const bool in = ids[x] >= 0 && ids[x] < a.c.n_pages;
            p.id[x] = in ? ids[x] : 0;
            p.ok &= in;
        }
        return p;
    };
    auto load_k = [&](int t, const Pages& p) {
        if constexpr (PAGES == 0) {
            const char* base = kbase + ((long long)p.id[0] * a.c.kp + (long long)((t * TK) & in_page) * a.c.ks) * EB;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int c = 0; c < KC; ++c) kr[u][c] = *reinterpret_cast<const u32x4*>(base + (unsigned)((16 * u + n) * ksb + 64 * c + 16 * g));
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int slot = key_of(t, u) & in_page;
                const char* base = kbase + ((long long)p.id[u] * a.c.kp + (long long)slot * a.c.ks) * EB + 16 * g;
#pragma unroll
                for (int c = 0; c < KC; ++c) kr[u][c] = *reinterpret_cast<const u32x4*>(base + 64 * c);
            }
        }
    };
    auto load_v = [&](int t, const Pages& p) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if constexpr (PAGES == 0) {
                const char* base = vbase + ((long long)p.id[0] * a.c.vp + (long long)((t * TK) & in_page) * a.c.vs) * EB;
#pragma unroll
                for (int h = 0; h < VL; ++h)
                    vr[j][h] = *reinterpret_cast<const VT*>(base + (unsigned)((16 * (j >> 2) + 4 * g + (j & 3)) * vsb + 256 * h + (unsigned)sizeof(VT) * n));
            } else {
                const int x = PAGES == 1 ? U + (j >> 2) : U + j;
                const int key = min(t * TK + 16 * (j >> 2) + 4 * g + (j & 3), rp.len - 1);
                // (PAGES 1: keys 4 g .. 4 g + 3 share a page; a clamped key may not, and then only its slot has to be inside)
                const int slot = key & in_page;
                const char* base = vbase + ((long long)p.id[x] * a.c.vp + (long long)slot * a.c.vs) * EB + sizeof(VT) * n;
#pragma unroll
                for (int h = 0; h < VL; ++h) vr[j][h] = *reinterpret_cast<const VT*>(base + 256 * h);
            }
        }
    };

    f32x4 acc[NT];
#pragma unroll
    for (int e = 0; e < NT; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const float scale2 = a.scale * 1.4426950408889634f;
    int t = t_begin + wk;
    if (t < t_end) {
        // page numbers are asked for one tile before the loads that need them, so that nothing waits for them
        ask(t);
        Pages pg = settle();
        ask(min(t + kw, t_end - 1));
        load_k(t, pg);
        load_v(t, pg);
        __builtin_amdgcn_sched_barrier(0);           // (the queries are cut while the first keys come)
        bf16x8 qb[KB ? QS : 1][KB ? KC : 1];
        f32x4 qf[KB ? 1 : KC];
        {
            const bool live = n < gn;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                if constexpr (QB) {
                    qb[0][c] = __builtin_bit_cast(bf16x8, live ? qw[c][0] : u32x4{0u, 0u, 0u, 0u});
                } else if constexpr (KB) {
                    float x[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = live ? __uint_as_float(qw[c][j >> 2][j & 3]) : 0.f;
                    bf16x8 o[3];
                    to_parts<3, true>(x, o);
#pragma unroll
                    for (int s = 0; s < QS; ++s) qb[s][c] = o[s];
                } else {
                    qf[c] = live ? __builtin_bit_cast(f32x4, qw[c][0]) : f32x4{0.f, 0.f, 0.f, 0.f};
                }
            }
        }
        while (true) {
            const int t_next = min(t + kw, t_end - 1);   // (past the end: a tile that is asked for again, from L2, and not used)
            f32x4 s[U];
#pragma unroll
            for (int u = 0; u < U; ++u) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
            if constexpr (KB) {
#pragma unroll
                for (int part = QS - 1; part >= 0; --part)   // small parts first
#pragma unroll
                    for (int c = 0; c < KC; ++c)
#pragma unroll
                        for (int u = 0; u < U; ++u) s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[u][c]), qb[part][c], s[u], 0, 0, 0);
            } else {
                f32x4 part[U][4];                        // four chains: less rounding than one, and none waits for another
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) part[u][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < KC; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int u = 0; u < U; ++u) part[u][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, kr[u][c])[i], qf[c][i], part[u][i], 0, 0, 0);
#pragma unroll
                for (int u = 0; u < U; ++u) s[u] = (part[u][0] + part[u][1]) + (part[u][2] + part[u][3]);
            }
            const Pages next = settle();
            ask(min(t + 2 * kw, t_end - 1));
            load_k(t_next, next);
            // softmax: x = scores in units of log2, keys TK t + 16 u + 4 g + i of head n
            float p[J];
#pragma unroll
            for (int j = 0; j < J; ++j) p[j] = s[j >> 2][j & 3] * scale2;
            const bool whole = t * TK >= rp.first && t * TK + TK <= rp.len;
            bool all_in = true;
            if constexpr (PAGES == 0) all_in = pg.ok;
            else all_in = __builtin_amdgcn_ballot_w64(!pg.ok) == 0;
            const bool masked = !(whole && all_in);
            unsigned dead = 0u;                          // bit j: key j of this lane is not to be seen
            if (masked) {
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const int key = t * TK + 16 * (j >> 2) + 4 * g + (j & 3);
                    bool live = key >= rp.first && key < rp.len;
                    if (!all_in) {
                        const int id = key < rp.len ? trow[key >> a.c.page_shift] : -1;
                        live = live && id >= 0 && id < a.c.n_pages;
                    }
                    if (!live) { p[j] = -INFINITY; dead |= 1u << j; }
#pragma unroll
                    for (int h = 0; h < VL; ++h)
#pragma unroll
                        for (int w = 0; w < (int)(sizeof(VT) / 4); ++w) vr[j][h][w] = live ? vr[j][h][w] : 0u;   // what is there may be NaN
                }
            }
            float mx = fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3]));
            if constexpr (U == 2) mx = fmaxf(mx, fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
            mx = fmaxf(m, group_max(mx));
            const float ref = mx > -INFINITY ? mx : 0.f;
            if (__builtin_amdgcn_ballot_w64(mx > m) != 0) {
                const float keep = __builtin_amdgcn_exp2f(m - ref);
                l *= keep;
#pragma unroll
                for (int e = 0; e < NT; ++e) acc[e] *= keep;
                m = mx;
            }
            // Scores of ordinary size: the product with the scale is not rounded before the maximum comes off.  Beyond 2^16 that rounding is what the
            // maximum itself carries, and has to cancel.
            if (__builtin_amdgcn_ballot_w64(large(ref)) == 0) {
#pragma unroll
                for (int j = 0; j < J; ++j) p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 2][j & 3], scale2, -ref));
                if (masked) {
#pragma unroll
                    for (int j = 0; j < J; ++j) p[j] = (dead >> j) & 1u ? 0.f : p[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < J; ++j) p[j] = __builtin_amdgcn_exp2f(p[j] - ref);
            }
            if constexpr (U == 2) l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            else l += (p[0] + p[1]) + (p[2] + p[3]);
            if constexpr (KB) {
                bf16x8 pb[PARTS];
                to_parts<PARTS>(p, pb);
#pragma unroll
                for (int e = 0; e < NT; ++e) {
                    u32x4 w;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        w[j] = __builtin_amdgcn_perm(vr[2 * j + 1][0][e >> 1], vr[2 * j][0][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
                    const bf16x8 av = __builtin_bit_cast(bf16x8, w);
#pragma unroll
                    for (int part = PARTS - 1; part >= 0; --part) acc[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, pb[part], acc[e], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int e = 0; e < NT; ++e)
                        acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[j][e >> 2][e & 3]), p[j], acc[e], 0, 0, 0);
            }
            load_v(t_next, next);
            t += kw;
            if (t >= t_end) break;
            pg = next;
        }
        if constexpr (KB) {
            f32x4 all = acc[0];                      // (its sum is NaN if any of them is; opposite infinities only cost the second pass)
#pragma unroll
            for (int e = 1; e < NT; ++e) all += acc[e];
            const float one = ((all[0] + all[1]) + (all[2] + all[3])) + l;
            const bool nan = one != one;
            if (const unsigned long long vote = __builtin_amdgcn_ballot_w64(nan && n < gn); __builtin_expect(vote != 0, 0)) {
                f32x4 acc2[NT];
#pragma unroll
                for (int e = 0; e < NT; ++e) acc2[e] = f32x4{0.f, 0.f, 0.f, 0.f};
                float m2 = -INFINITY, l2 = 0.f;
                const PagedAttnArgs& b = arguments_again();
                const int seq2 = b.seq ? b.seq[row] : row;
                const RowPlan r = plan_row(b, b.lengths[row], b.starts ? b.starts[row] : 0, seq2);
                const int begin = r.t0 + (int)split * r.per;
                whole_pass<QS, KC, NT, VT>(b.c, static_cast<const char*>(b.c.k) + (long long)hk * b.c.kh * EB, static_cast<const char*>(b.c.v) + (long long)hk * b.c.vh * EB,
                                           b.c.table + (long long)seq2 * b.c.table_stride, qb, b.scale * 1.4426950408889634f, begin + wk, min(r.t1, begin + r.per), kw, r.len,
                                           r.first, r.len, 16, m2, l2, acc2);
                const bool redo = in_column(vote, n);
                m = redo ? m2 : m;
                l = redo ? l2 : l;
#pragma unroll
                for (int e = 0; e < NT; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[e][i] = redo ? acc2[e][i] : acc[e][i];
            }
        }
    }
    l = group_sum(l);

    // the waves meet in LDS: maxima and sums [nw][16], then the weighted sums [nw][gn][D].  Lane (n, g) holds for head n the elements of
    // row 4 g + i of tile e: D / 16 (4 g + i) + e with a bf16 cache, 64 (e / 4) + 4 (4 g + i) + e % 4 with an fp32 one
    float* sm_m = sm;
    float* sm_l = sm + nw * 16;
    float* sm_o = sm + nw * 32;
    if (lane < 16) {
        sm_m[wave * 16 + n] = m;
        sm_l[wave * 16 + n] = l;
    }
    __syncthreads();
    float top = -INFINITY;
    for (int w = wh; w < nw; w += hw) top = fmaxf(top, sm_m[w * 16 + n]);
    if (n < gn) {
        const float f = part_factor(m, top);
        float* o = sm_o + (wave * gn + n) * D;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < NT; e += 4) {
                const f32x4 v = f32x4{acc[e][i], acc[e + 1][i], acc[e + 2][i], acc[e + 3][i]} * f;
                const int at = KB ? NT * (4 * g + i) + e : 64 * (e >> 2) + 4 * (4 * g + i);
                *reinterpret_cast<f32x4*>(o + at) = v;
            }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < hw * gn * (D / 4); x += blockDim.x) {
        const int d4 = (x % (D / 4)) * 4, hn = (x / (D / 4)) % gn, ho = x / (D / 4) / gn;
        if (hk0 + ho >= a.c.kv_heads) continue;
        const int h = (hk0 + ho) * group + q16 * 16 + hn;
        float big = -INFINITY, sum = 0.f;
        for (int w = ho; w < nw; w += hw) big = fmaxf(big, sm_m[w * 16 + hn]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        for (int w = ho; w < nw; w += hw) {
            const float mw = sm_m[w * 16 + hn];
            sum += sm_l[w * 16 + hn] * part_factor(mw, big);
            o += *reinterpret_cast<const f32x4*>(sm_o + (w * gn + hn) * D + d4);
        }
        if (rp.active > 1) {
            const long long part = ((long long)row * a.q_heads + h) * a.n_split + split;
            *reinterpret_cast<f32x4*>(a.ws + part * D + d4) = o;
            if (d4 == 0) *reinterpret_cast<float2*>(a.ws + (long long)a.rows * a.q_heads * a.n_split * D + part * 2) = float2{big, sum};
        } else {
            store_out(a, row, h, d4, o, sum);
        }
    }
}

// ---- attention of a prompt's rows -------------------------------------------------------------------------------------------------
// The same sums where neighbouring rows belong to one sequence: the 16 columns of a tile are 16 / G rows with the G heads of one key head, so a key
// is read once for all of them (from L2: the blocks that read it are kv_heads apart).  Bound: the matrix and vector work of a tile, a few hundred
// cycles for 32 keys x 16 columns (8000 rows of a prompt, 32 heads over 8 of 128, bf16: 2.2 ms, 237 TFLOP/s; row by row the reads take 4 to 10 times
// as long).  Rows of a block that belong to other sequences are taken in turn (a column that is not in turn has weight
// zero), so any rows come out right.  A key that some of the rows see and others do not has weight zero for the others; only if such a tile holds a
// value that is not finite (0 times it is not 0) are its rows summed one by one.
// SMALL: pages of fewer than TK keys.
template <bool QB, bool KB, int D, int TK, bool SMALL, int PARTS>
__global__ __launch_bounds__(256, D == 64 && !(SMALL && KB && !QB) ? 3 : 2) void paged_prompt_kernel(PagedAttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) float sm[];
    constexpr int EB = KB ? 2 : 4, KC = KB ? D / 32 : D / 16, VL = KB ? 1 : D / 64, NT = D / 16, QS = QB ? 1 : 3, U = TK / 16, J = 4 * U;
    using VT = std::conditional_t<KB && D == 64, u32x2, u32x4>;
    constexpr int VW = (int)sizeof(VT) / 4;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
    const int group = a.q_heads / a.c.kv_heads, R = 16 / group, cols = R * group;
    const int hk = (int)(blockIdx.x % (unsigned)a.c.kv_heads), r0 = (int)(blockIdx.x / (unsigned)a.c.kv_heads) * R;
    const int rn = n / group;                       // this column's row and head
    const bool col = n < cols && r0 + rn < a.rows;
    const int row = col ? r0 + rn : r0, h = hk * group + (col ? n - rn * group : 0);
    const int row_len = a.lengths[row], seq = a.seq ? a.seq[row] : row, first = a.starts ? max(a.starts[row], 0) : 0;
    bf16x8 qb[KB ? QS : 1][KB ? KC : 1];
    f32x4 qf[KB ? 1 : KC];
    {
        const long long qo = row * a.qr + h * a.qh;
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            if constexpr (QB) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + qo + 32 * c + 8 * g);
                qb[0][c] = __builtin_bit_cast(bf16x8, col ? w : u32x4{0u, 0u, 0u, 0u});
            } else if constexpr (KB) {
                float x[8];
                load_row<float, 4>(a.q, qo + 32 * c + 8 * g, *reinterpret_cast<float(*)[4]>(x));
                load_row<float, 4>(a.q, qo + 32 * c + 8 * g + 4, *reinterpret_cast<float(*)[4]>(x + 4));
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = col ? x[j] : 0.f;
                bf16x8 o[3];
                to_parts<3, true>(x, o);
#pragma unroll
                for (int s = 0; s < QS; ++s) qb[s][c] = o[s];
            } else {
                const f32x4 w = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.q) + qo + 16 * c + 4 * g);
                qf[c] = col ? w : f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
    }
    int len = 0;
    if (col && row_len >= 0 && seq >= 0 && seq < a.c.n_seqs) {
        const long long most = (long long)a.c.max_pages << a.c.page_shift, k = (long long)row_len + a.length_add;
        len = (int)(k > most ? most : k);
    }
    const bool has = len > first;

    const unsigned ksb = (unsigned)a.c.ks * EB, vsb = (unsigned)a.c.vs * EB;
    const char* kbase = static_cast<const char*>(a.c.k) + (long long)hk * a.c.kh * EB;
    const char* vbase = static_cast<const char*>(a.c.v) + (long long)hk * a.c.vh * EB;
    const int in_page = (1 << a.c.page_shift) - 1;
    constexpr int NP = SMALL ? U + J : 1;           // page numbers of a tile: of each key a lane loads, or one
    f32x4 acc[NT];
#pragma unroll
    for (int e = 0; e < NT; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const float scale2 = a.scale * 1.4426950408889634f;
    const unsigned alive = (unsigned)__builtin_amdgcn_ballot_w64(has) & 0xFFFFu;
    unsigned pending = alive;
    int sq, lo, hi, lo_all, hi_all;
    unsigned in;
    bool mine;
    // the columns of the first pending one's sequence sq, and the keys they span: [lo, hi), all of them see [lo_all, hi_all)
    auto next_sequence = [&]() {
        sq = __builtin_amdgcn_readlane(seq, __builtin_ctz(pending));
        in = (unsigned)__builtin_amdgcn_ballot_w64(has && seq == sq) & 0xFFFFu;
        pending &= ~in;
        mine = (in >> n) & 1u;
        lo = mine ? first : 0x7FFFFFFF, lo_all = mine ? first : 0, hi = mine ? len : 0, hi_all = mine ? len : 0x7FFFFFFF;
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
            lo = min(lo, __shfl_xor(lo, d, 64));
            lo_all = max(lo_all, __shfl_xor(lo_all, d, 64));
            hi = max(hi, __shfl_xor(hi, d, 64));
            hi_all = min(hi_all, __shfl_xor(hi_all, d, 64));
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        lo_all = __builtin_amdgcn_readfirstlane(lo_all);
        hi = __builtin_amdgcn_readfirstlane(hi);
        hi_all = __builtin_amdgcn_readfirstlane(hi_all);
    };
    while (pending != 0u) {
        next_sequence();
        const int* trow = a.c.table + (long long)sq * a.c.table_stride;
        const int t_end = (hi + TK - 1) / TK;
        int t = lo / TK + wave;
        if (t >= t_end) continue;
        auto key_of = [&](int at, int x) {           // (clamped to the last: entries past it may hold anything)
            int k = at * TK;
            if (SMALL) k += x < U ? 16 * x + n : 16 * ((x - U) >> 2) + 4 * g + ((x - U) & 3);
            return min(k, hi - 1);
        };
        int ids[NP];
        auto ask = [&](int at) {
#pragma unroll
            for (int x = 0; x < NP; ++x) ids[x] = trow[key_of(at, x) >> a.c.page_shift];
        };
        struct Pages { int id[NP]; unsigned ok; };   // clamped into the pool; ok: bit j, key j of this lane's values has a page
        auto settle = [&]() {
            Pages p;
            p.ok = 0u;
#pragma unroll
            for (int x = 0; x < NP; ++x) {
                const bool good = ids[x] >= 0 && ids[x] < a.c.n_pages;
                p.id[x] = good ? ids[x] : 0;
                if (!SMALL) p.ok = good ? 0xFFu : 0u;
                else if (x >= U) p.ok |= good ? 1u << (x - U) : 0u;
            }
            return p;
        };
        u32x4 kr[U][KC];
        VT vr[J][VL];
        auto load_k = [&](int at, const Pages& p) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int slot = SMALL ? key_of(at, u) & in_page : ((at * TK) & in_page) + 16 * u + n;
                const char* base = kbase + (long long)p.id[SMALL ? u : 0] * a.c.kp * EB + (long long)slot * ksb + 16 * g;
#pragma unroll
                for (int c = 0; c < KC; ++c) kr[u][c] = *reinterpret_cast<const u32x4*>(base + 64 * c);
            }
        };
        auto load_v = [&](int at, const Pages& p) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int slot = SMALL ? key_of(at, U + j) & in_page : ((at * TK) & in_page) + 16 * (j >> 2) + 4 * g + (j & 3);
                const char* base = vbase + (long long)p.id[SMALL ? U + j : 0] * a.c.vp * EB + (long long)slot * vsb + sizeof(VT) * n;
#pragma unroll
                for (int x = 0; x < VL; ++x) vr[j][x] = *reinterpret_cast<const VT*>(base + 256 * x);
            }
        };
        ask(t);
        Pages pg = settle();
        ask(min(t + nw, t_end - 1));
        load_k(t, pg);
        load_v(t, pg);
        while (true) {
            const int t_next = min(t + nw, t_end - 1);
            f32x4 s[U];
#pragma unroll
            for (int u = 0; u < U; ++u) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
            if constexpr (KB) {
#pragma unroll
                for (int part = QS - 1; part >= 0; --part)
#pragma unroll
                    for (int c = 0; c < KC; ++c)
#pragma unroll
                        for (int u = 0; u < U; ++u) s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[u][c]), qb[part][c], s[u], 0, 0, 0);
            } else {
                f32x4 part[U][4];
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) part[u][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < KC; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int u = 0; u < U; ++u) part[u][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, kr[u][c])[i], qf[c][i], part[u][i], 0, 0, 0);
#pragma unroll
                for (int u = 0; u < U; ++u) s[u] = (part[u][0] + part[u][1]) + (part[u][2] + part[u][3]);
            }
            const Pages next = settle();
            ask(min(t + 2 * nw, t_end - 1));
            load_k(t_next, next);
            float p[J];
#pragma unroll
            for (int j = 0; j < J; ++j) p[j] = s[j >> 2][j & 3] * scale2;
            const bool masked = !(in == alive && t * TK >= lo_all && t * TK + TK <= hi_all && __builtin_amdgcn_ballot_w64((~pg.ok & ((1u << J) - 1)) != 0u) == 0);
            unsigned dead = 0u;
            bool odd = false;                        // a value that is not finite in a tile that not all rows see
            if (masked) {
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const int key = t * TK + 16 * (j >> 2) + 4 * g + (j & 3);
                    const bool there = key >= lo && key < hi && ((pg.ok >> j) & 1u);
                    if (!(there && mine && key >= first && key < len)) { p[j] = -INFINITY; dead |= 1u << j; }
#pragma unroll
                    for (int x = 0; x < VL; ++x)
#pragma unroll
                        for (int w = 0; w < VW; ++w) {
                            const unsigned v = there ? vr[j][x][w] : 0u;
                            vr[j][x][w] = v;
                            if (KB) odd = odd || (v & 0x7F80u) == 0x7F80u || (v & 0x7F800000u) == 0x7F800000u;
                            else odd = odd || (v & 0x7F800000u) == 0x7F800000u;
                        }
                }
            }
            float mx = fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3]));
            if constexpr (U == 2) mx = fmaxf(mx, fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
            mx = fmaxf(m, group_max(mx));
            const float ref = mx > -INFINITY ? mx : 0.f;
            if (__builtin_amdgcn_ballot_w64(mx > m) != 0) {
                const float keep = __builtin_amdgcn_exp2f(m - ref);
                l *= keep;
#pragma unroll
                for (int e = 0; e < NT; ++e) acc[e] *= keep;
                m = mx;
            }
            if (__builtin_amdgcn_ballot_w64(large(ref)) == 0) {   // (as above)
#pragma unroll
                for (int j = 0; j < J; ++j) p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 2][j & 3], scale2, -ref));
            } else {
#pragma unroll
                for (int j = 0; j < J; ++j) p[j] = __builtin_amdgcn_exp2f(p[j] - ref);
            }
            if (masked) {
#pragma unroll
                for (int j = 0; j < J; ++j) p[j] = (dead >> j) & 1u ? 0.f : p[j];
            }
            if constexpr (U == 2) l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            else l += (p[0] + p[1]) + (p[2] + p[3]);
            bf16x8 pb[KB ? PARTS : 1];
            if constexpr (KB) to_parts<PARTS>(p, pb);
            // o += V^T P, of the values whose bit is set in `of`
            auto weigh = [&](auto of, int e, f32x4 o) {
                auto v = [&](int j, int x, int w) -> unsigned {
                    if constexpr (std::is_same_v<decltype(of), unsigned>) return (of >> j) & 1u ? vr[j][x][w] : 0u;
                    else return vr[j][x][w];
                };
                if constexpr (KB) {
                    u32x4 w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = __builtin_amdgcn_perm(v(2 * j + 1, 0, e >> 1), v(2 * j, 0, e >> 1), (e & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int part = PARTS - 1; part >= 0; --part) o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), pb[part], o, 0, 0, 0);
                } else {
#pragma unroll
                    for (int j = 0; j < J; ++j) o = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v(j, e >> 2, e & 3)), p[j], o, 0, 0, 0);
                }
                return o;
            };
            if (__builtin_amdgcn_ballot_w64(odd) == 0) {
#pragma unroll
                for (int e = 0; e < NT; ++e) acc[e] = weigh(true, e, acc[e]);
            } else {
                for (int r = 0; r < R; ++r) {
                    const int c = r * group, f_r = __builtin_amdgcn_readlane(first, c), l_r = (in >> c) & 1u ? __builtin_amdgcn_readlane(len, c) : 0;
                    unsigned of = 0u;                // the keys that row r sees
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        const int key = t * TK + 16 * (j >> 2) + 4 * g + (j & 3);
                        of |= key >= f_r && key < l_r ? 1u << j : 0u;
                    }
#pragma unroll
                    for (int e = 0; e < NT; ++e) {
                        const f32x4 o = weigh(of, e, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[e][i] += rn == r ? o[i] : 0.f;
                    }
                }
            }
            load_v(t_next, next);
            t += nw;
            if (t >= t_end) break;
            pg = next;
        }
    }
    if constexpr (KB) {
        f32x4 all = acc[0];                          // (as above)
#pragma unroll
        for (int e = 1; e < NT; ++e) all += acc[e];
        const float one = ((all[0] + all[1]) + (all[2] + all[3])) + l;
        const bool nan = one != one;
        if (const unsigned long long vote = __builtin_amdgcn_ballot_w64(nan && has); __builtin_expect(vote != 0, 0)) {
            f32x4 acc2[NT];
#pragma unroll
            for (int e = 0; e < NT; ++e) acc2[e] = f32x4{0.f, 0.f, 0.f, 0.f};
            float m2 = -INFINITY, l2 = 0.f;
            pending = alive;
            while (pending != 0u) {
                next_sequence();
                whole_pass<QS, KC, NT, VT>(a.c, kbase, vbase, a.c.table + (long long)sq * a.c.table_stride, qb, scale2, lo / TK + wave, (hi + TK - 1) / TK, nw, hi,
                                           first, mine ? len : 0, group, m2, l2, acc2);
            }
            const bool redo = in_column(vote, n);
            m = redo ? m2 : m;
            l = redo ? l2 : l;
#pragma unroll
            for (int e = 0; e < NT; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[e][i] = redo ? acc2[e][i] : acc[e][i];
        }
    }
    l = group_sum(l);
    if (!has) {
        m = -INFINITY;
        l = 0.f;
    }
    float* sm_m = sm;
    float* sm_l = sm + nw * 16;
    float* sm_o = sm + nw * 32;
    if (lane < 16) {
        sm_m[wave * 16 + n] = m;
        sm_l[wave * 16 + n] = l;
    }
    __syncthreads();
    float top = -INFINITY;
    for (int w = 0; w < nw; ++w) top = fmaxf(top, sm_m[w * 16 + n]);
    {
        const float f = part_factor(m, top);
        float* o = sm_o + (wave * 16 + n) * D;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < NT; e += 4) {
                f32x4 v = f32x4{acc[e][i], acc[e + 1][i], acc[e + 2][i], acc[e + 3][i]} * f;
                if (!has) v = f32x4{0.f, 0.f, 0.f, 0.f};
                *reinterpret_cast<f32x4*>(o + (KB ? NT * (4 * g + i) + e : 64 * (e >> 2) + 4 * (4 * g + i))) = v;
            }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < cols * (D / 4); x += blockDim.x) {
        const int d4 = (x % (D / 4)) * 4, c = x / (D / 4), r = r0 + c / group;
        if (r >= a.rows || a.lengths[r] < 0) continue;
        float big = -INFINITY, sum = 0.f;
        for (int w = 0; w < nw; ++w) big = fmaxf(big, sm_m[w * 16 + c]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        for (int w = 0; w < nw; ++w) {
            sum += sm_l[w * 16 + c] * part_factor(sm_m[w * 16 + c], big);
            o += *reinterpret_cast<const f32x4*>(sm_o + (w * 16 + c) * D + d4);
        }
        store_out(a, r, hk * group + c % group, d4, o, sum);
    }
}

// a row's few (at most 8) partial results joined in a fixed order, one wave per (row, query head), four to a block
template <int D>
__global__ __launch_bounds__(256) void paged_join_few_kernel(PagedAttnArgs a) {
    constexpr int LP = D / 4, NS = 64 / LP;         // lanes of a partial, partials at a time
    const int pair = blockIdx.x * 4 + (int)(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (pair >= a.rows * a.q_heads) return;
    const int row = pair / a.q_heads, h = pair - row * a.q_heads;
    const int len = a.lengths[row], seq = a.seq ? a.seq[row] : row, first = a.starts ? a.starts[row] : 0;
    const long long part = (long long)pair * a.n_split;
    const float2* ml = reinterpret_cast<const float2*>(a.ws + (long long)a.rows * a.q_heads * a.n_split * D) + part;
    const int sub = lane / LP, d4 = (lane % LP) * 4;
    // everything is asked for at once, the row's plan and the partial results; those that no block has written hold anything and are dropped
    float2 x[8];
    f32x4 v[8 / NS];
#pragma unroll
    for (int s = 0; s < 8; ++s) x[s] = ml[min(s, a.n_split - 1)];
#pragma unroll
    for (int k = 0; k < 8 / NS; ++k) v[k] = *reinterpret_cast<const f32x4*>(a.ws + (part + min(k * NS + sub, a.n_split - 1)) * D + d4);
    __builtin_amdgcn_sched_barrier(0);
    if (len < 0) return;
    const RowPlan rp = plan_row(a, len, first, seq);
    if (rp.active <= 1) return;
#pragma unroll
    for (int s = 0; s < 8; ++s) x[s] = s < rp.active ? x[s] : float2{-INFINITY, 0.f};
#pragma unroll
    for (int k = 0; k < 8 / NS; ++k) v[k] = k * NS + sub < rp.active ? v[k] : f32x4{0.f, 0.f, 0.f, 0.f};
    float big = x[0].x, sum = 0.f, f[8];
#pragma unroll
    for (int s = 1; s < 8; ++s) big = fmaxf(big, x[s].x);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        f[s] = part_factor(x[s].x, big);
        sum += x[s].y * f[s];
    }
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 8 / NS; ++k) {
        float w = f[k * NS];
#pragma unroll
        for (int q = 1; q < NS; ++q) w = sub == q ? f[k * NS + q] : w;
        o += v[k] * w;
    }
#pragma unroll
    for (int d = LP; d < 64; d <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], d, 64);
    if (sub == 0) store_out(a, row, h, d4, o, sum);
}

// many partial results: one block per (row, query head).  Three memory latencies: the row's plan, the maxima and sums, the partial results
template <int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
    constexpr int LP = D / 4, NS = 256 / LP;        // threads of a partial, partials at a time
    __shared__ __attribute__((aligned(16))) float sm_o[NS][D];
    __shared__ float sm_f[kMaxSplit], sm_l;
    const int row = blockIdx.x / a.q_heads, h = blockIdx.x % a.q_heads, tid = threadIdx.x;
    const int len = a.lengths[row], seq = a.seq ? a.seq[row] : row, first = a.starts ? a.starts[row] : 0;
    if (len < 0) return;
    const RowPlan rp = plan_row(a, len, first, seq);
    if (rp.active <= 1) return;
    const long long part = (long long)blockIdx.x * a.n_split;
    const int sub = tid / LP, d4 = (tid % LP) * 4;
    if (tid < 64) {                                 // kMaxSplit = 64: a lane each
        const float2* ml = reinterpret_cast<const float2*>(a.ws + (long long)a.rows * a.q_heads * a.n_split * D) + part;
        const float2 x = tid < rp.active ? ml[tid] : float2{-INFINITY, 0.f};
        float big = x.x;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor(big, o, 64));
        const float f = part_factor(x.x, big);
        sm_f[tid] = f;
        float sum = x.y * f;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (tid == 0) sm_l = sum;
    }
    f32x4 x[kMaxSplit / NS];
#pragma unroll
    for (int k = 0; k < kMaxSplit / NS; ++k) {
        const int s = k * NS + sub;
        x[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (k * NS < rp.active && s < rp.active) x[k] = *reinterpret_cast<const f32x4*>(a.ws + (part + s) * D + d4);
    }
    __syncthreads();
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kMaxSplit / NS; ++k) o += x[k] * sm_f[k * NS + sub];
    *reinterpret_cast<f32x4*>(&sm_o[sub][d4]) = o;
    __syncthreads();
    if (sub == 0) {
#pragma unroll
        for (int k = 1; k < NS; ++k) o += *reinterpret_cast<const f32x4*>(&sm_o[k][d4]);
        store_out(a, row, h, d4, o, sm_l);
    }
}

}  // namespace

namespace {

template <typename IN, typename KV> hipError_t launch_append_t(const PagedAppendArgs& a, hipStream_t s) {
    const long long threads = (long long)a.rows * (a.q_heads + 2 * a.c.kv_heads) * (a.c.head_dim / 2) * (long long)sizeof(IN) / 16;
    if (threads > 0xFFFFFF00LL) return hipErrorInvalidValue;
    const dim3 grid((unsigned)((threads + 255) / 256)), block(256);
    if (a.c.head_dim == 64) hipLaunchKernelGGL((paged_append_kernel<IN, KV, 64>), grid, block, 0, s, a);
    else if (a.c.head_dim == 128) hipLaunchKernelGGL((paged_append_kernel<IN, KV, 128>), grid, block, 0, s, a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s) {
    if (a.rows <= 0 || (a.q == nullptr) != (a.q_heads == 0)) return hipErrorInvalidValue;
    if (a.in_bf16) return a.c.bf16 ? launch_append_t<uint16_t, uint16_t>(a, s) : launch_append_t<uint16_t, float>(a, s);
    return a.c.bf16 ? launch_append_t<float, uint16_t>(a, s) : launch_append_t<float, float>(a, s);
}

namespace {

template <bool QB, bool KB, int D, int TK, int PARTS>
void launch_attention_p(const PagedAttnArgs& a, unsigned blocks, unsigned threads, size_t lds, hipStream_t s) {
    const dim3 grid(blocks), block(threads);
    if (a.c.page_shift >= a.tile_shift) hipLaunchKernelGGL((paged_attention_kernel<QB, KB, D, TK, 0, PARTS>), grid, block, lds, s, a);
    else if (a.c.page_shift >= 2) hipLaunchKernelGGL((paged_attention_kernel<QB, KB, D, TK, 1, PARTS>), grid, block, lds, s, a);
    else hipLaunchKernelGGL((paged_attention_kernel<QB, KB, D, TK, 2, PARTS>), grid, block, lds, s, a);
}
template <int D>
void launch_prompt_d(const PagedAttnArgs& a, unsigned blocks, unsigned threads, size_t lds, hipStream_t s) {
    const dim3 grid(blocks), block(threads);
    const bool small = a.c.page_shift < a.tile_shift;
    if (!a.c.bf16) {
        if (small) hipLaunchKernelGGL((paged_prompt_kernel<false, false, D, 16, true, 1>), grid, block, lds, s, a);
        else hipLaunchKernelGGL((paged_prompt_kernel<false, false, D, 16, false, 1>), grid, block, lds, s, a);
    } else if (a.q_bf16 && a.out_bf16) {
        if (small) hipLaunchKernelGGL((paged_prompt_kernel<true, true, D, 32, true, 2>), grid, block, lds, s, a);
        else hipLaunchKernelGGL((paged_prompt_kernel<true, true, D, 32, false, 2>), grid, block, lds, s, a);
    } else if (a.q_bf16) {
        if (small) hipLaunchKernelGGL((paged_prompt_kernel<true, true, D, 32, true, 3>), grid, block, lds, s, a);
        else hipLaunchKernelGGL((paged_prompt_kernel<true, true, D, 32, false, 3>), grid, block, lds, s, a);
    } else if (a.out_bf16) {
        if (small) hipLaunchKernelGGL((paged_prompt_kernel<false, true, D, 32, true, 2>), grid, block, lds, s, a);
        else hipLaunchKernelGGL((paged_prompt_kernel<false, true, D, 32, false, 2>), grid, block, lds, s, a);
    } else {
        if (small) hipLaunchKernelGGL((paged_prompt_kernel<false, true, D, 32, true, 3>), grid, block, lds, s, a);
        else hipLaunchKernelGGL((paged_prompt_kernel<false, true, D, 32, false, 3>), grid, block, lds, s, a);
    }
}
template <int D>
void launch_attention_d(const PagedAttnArgs& a, unsigned blocks, unsigned threads, size_t lds, hipStream_t s) {
    if (!a.c.bf16) launch_attention_p<false, false, D, 16, 1>(a, blocks, threads, lds, s);
    else if (a.q_bf16 && a.out_bf16) launch_attention_p<true, true, D, 32, 2>(a, blocks, threads, lds, s);
    else if (a.q_bf16) launch_attention_p<true, true, D, 32, 3>(a, blocks, threads, lds, s);
    else if (a.out_bf16) launch_attention_p<false, true, D, 32, 2>(a, blocks, threads, lds, s);
    else launch_attention_p<false, true, D, 32, 3>(a, blocks, threads, lds, s);
    // (96 rows of 32 heads, 3 partial results each: 8.3 us with a block to each, 5.1 with a wave)
    if (a.n_split > 8) hipLaunchKernelGGL((paged_join_kernel<D>), dim3((unsigned)(a.rows * a.q_heads)), dim3(256), 0, s, a);
    else if (a.n_split > 1) hipLaunchKernelGGL((paged_join_few_kernel<D>), dim3((unsigned)(a.rows * a.q_heads + 3) / 4), dim3(256), 0, s, a);
}

}  // namespace

// shared memory of a block: maxima and sums, and the weighted sums of its waves
static size_t attention_lds(const PagedAttnArgs& a) {
    const int group = a.q_heads / a.c.kv_heads;
    return (size_t)a.waves * (32 + (size_t)(group < 16 && !a.prompt ? group : 16) * a.c.head_dim) * 4;
}

static long long prompt_blocks(const PagedAttnArgs& a) {
    const int r = 16 / (a.q_heads / a.c.kv_heads);
    return ((long long)a.rows + r - 1) / r * a.c.kv_heads;
}

void plan_paged_attention(PagedAttnArgs& a) {
    const int group = a.q_heads / a.c.kv_heads, eb = a.c.bf16 ? 2 : 4;
    a.tile_shift = a.c.bf16 ? 5 : 4;
    const long long tiles = ((long long)a.max_length + (1 << a.tile_shift) - 1) >> a.tile_shift;
    const long long pairs = (long long)a.rows * a.c.kv_heads * ((group + 15) / 16);
    // Rows that share their keys read them once, but no block of theirs is split: it goes through the whole length with its few waves.  A tile takes a block
    // of theirs 0.16 to 0.31 us, a (row, key head) pair on its own 1.2 (heads of 64) to 2.6 ns, so sharing pays from some 190 pairs on at any length (32 / 8
    // heads of 128, bf16, 131071 keys of one sequence: 4 rows 1527 us shared, 369 row by row; 16 rows 1312, 1210; 32 rows 1283, 2520; 8 / 1 heads 4 rows
    // 1096, 48; 256 rows 1110, 1151; 16 fp32 heads of 64 8 rows 1851, 1414; 16 rows 1853, 2653).  Where the rows' order is not known, a block may hold as
    // many sequences as rows and take them in turn: sharing then gains so many times in one order what it loses in the other only from sqrt(turns) times the
    // pairs on.  (4 sequences of 131071 keys, 32 / 8 heads, rows sequence by sequence, in turn, and either row by row: 16 rows 1576, 7522, 1350 us; 64 rows
    // 1371, 7505, 4900; 128 rows 1340, 7517, 9700.)
    const long long turns = a.prompt == 2 ? std::min(16 / std::min(group, 16), a.c.n_seqs) : 1;
    a.prompt = a.prompt && group <= 8 && pairs * pairs >= 192LL * 192LL * turns;   // (group: two rows at least to a tile)
    if (a.prompt) {
        const long long blocks = prompt_blocks(a);
        a.head_waves = 1;
        a.n_split = 1;
        // one wave to a block where there are enough (2000 rows of two prompts, 8 key heads of 128, bf16: 1 / 2 / 4 waves 310 / 317 / 342 us; 300 rows
        // of one 18.1 / 14.7 / 19.2; 64 rows 11.2 / 9.3 / 8.7); fp32 products take longer than the waves' joining (2000 rows of 16 heads 143 / 126 / 112)
        a.waves = a.c.bf16 ? (blocks >= 2000 ? 1 : (blocks >= 512 ? 2 : 4)) : (blocks >= 8192 ? 2 : 4);
        a.min_tiles = 1;
        return;
    }
    // 128-byte rows that lie beside those of the other heads: blocks of four heads, two waves each, so that a block reads 512 bytes in a
    // row (512 rows of 16 key heads of 64 bf16, 264 keys each: 104 us, a head a block 121; with the heads apart in memory 99).  Up to 24 tiles
    // the row is one block (450 keys: 169 us, in two 210), longer ones, which differ more, are split (128 rows of 60 to 1100 keys: 3 blocks 68 us,
    // 1 73; up to 4000 keys: 8 211 us, 1 254), where there are not so many that they even out by themselves (2048 rows of 60 to 1100: 1 856 us, 3 873).
    if (group <= 16 && a.c.head_dim * eb == 128 && a.c.kh < a.c.ks && a.c.kv_heads >= 4 && pairs >= 1024) {
        a.head_waves = 4;
        a.waves = 8;
        a.min_tiles = 12;
        a.n_split = tiles <= 24 || pairs >= 4096 ? 1 : (int)std::min((tiles + 6) / 12, 8LL);
        return;
    }
    // Otherwise a block works on one key head.  Over 236 shapes (1 to 600 rows, 5 to 4096 tiles) this is 3.2 to 4.0 % above the best of the plans that were
    // timed on average, by type and head_dim (profiles/paged_attention_plans.txt).  `wide`: the kernel of 128 bf16 elements has registers for two waves to a SIMD, the others for four or (fp32, half the work to a
    // tile) for as many as are useful.
    const bool wide = a.c.bf16 && a.c.head_dim == 128;
    const long long all = pairs * tiles;             // if every row is as long as the longest
    // rows differ more, the longer they are: so many blocks even out, unless the rows do so by their number (1024 rows of 400 to 2000 keys, 8 key heads
    // of 128: 1 block a row 912 us, 3 943)
    const long long ragged = pairs >= 4096 ? 1 : std::min(tiles / (wide ? 16 : 20), 8LL);
    a.head_waves = 1;
    a.n_split = 1;
    if (tiles <= (wide ? 16 : a.c.bf16 ? 40 : 32) && (wide || pairs >= 64 || tiles <= 16)) {
        // short rows: one block, no second launch (16 rows of 16 bf16 heads of 64, up to 464 keys: 9.7 us, in four 12.2)
        a.waves = wide ? 2 : 4;
    } else if (all < 65536) {
        // as many blocks as the card takes well at once (heads of 128, bf16 or long: one to a CU), of two waves, about two tiles and more to a wave; where that
        // asks for more than 8 partial results of a shortish row, 8 blocks of four waves (2 rows of 16 fp32 heads, up to 4000 keys: 16.0 us, 16 of
        // two 17.4).  (One to a CU: three rows of 60000 bf16 keys, 8 key heads of 128, 10 x 2 131 us, 43 x 4 141; a row of 10397 fp32 keys, 16 heads
        // of 128, 16 x 4 41 us, 40 x 4 48)
        const bool to_cus = wide || (a.c.head_dim == 128 && tiles > 512);
        long long n = to_cus ? std::max(256 / pairs, 1LL) : ((a.c.bf16 ? 384 : 640) + pairs - 1) / pairs;
        n = std::min(std::max(n, ragged), std::max((tiles + 2) / (wide ? 8 : 4), 1LL));
        a.waves = 2;
        if (n > 8 && tiles <= (wide ? 128 : 512)) {
            n = 8;
            a.waves = 4;
        } else if (!a.c.bf16 && tiles >= 16 * n) {
            a.waves = 4;
        }
        a.n_split = (int)std::min(n, (long long)kMaxSplit);
    } else {
        // much work: a wave to 8 tiles of the call, at most 8192 of them, in blocks that grow with it: the fewer partial results, the shorter the join
        // (8 rows of 131071 bf16 keys, 8 key heads of 128: 8 x 32 628 us, 2 x 4 651; 96 rows of 8190: 4 x 5 329, 8 x 3 338)
        const long long share = (std::min(all / 8, 8192LL) + pairs - 1) / pairs;   // of a pair
        a.waves = share > 128 ? 8 : 4;
        a.n_split = (int)std::min(std::max((share + a.waves - 1) / a.waves, std::max(std::min(ragged, 5LL), 1LL)), (long long)kMaxSplit);
    }
    // more than 16 heads to a key head: the blocks that read the same keys are n_split apart, in the same L2 where that is a multiple of the 8 XCDs
    // (2 rows of 40 heads over one, 60001 keys: 42 blocks a row 37.4 us, 32 29.5)
    if (group > 16 && a.n_split >= 8) a.n_split &= ~7;
    if (attention_lds(a) > 65536) a.waves = 4;   // (8 waves of 16 heads of 128)
    if (pairs > 1 << 22) a.waves = 1;            // (a launch has at most 2^32 threads)
    a.min_tiles = 2 * a.waves;
}

size_t paged_attention_workspace(const PagedAttnArgs& a) {
    return a.n_split <= 1 ? 0 : (size_t)a.rows * a.q_heads * a.n_split * (a.c.head_dim + 2) * 4;
}

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t s) {
    const int group = a.q_heads / a.c.kv_heads;
    if (a.head_waves < 1 || a.waves % a.head_waves) return hipErrorInvalidValue;
    const long long blocks = (long long)a.rows * ((a.c.kv_heads + a.head_waves - 1) / a.head_waves) * ((group + 15) / 16) * a.n_split;
    if (a.rows <= 0 || a.n_split < 1 || a.n_split > kMaxSplit || a.min_tiles < 1 || a.waves < 1 || a.waves > 8 || blocks > 0x7FFFFFFFLL) return hipErrorInvalidValue;
    if (a.n_split > 1 && a.ws == nullptr) return hipErrorInvalidValue;
    const size_t lds = attention_lds(a);
    if (lds > 65536) return hipErrorInvalidValue;
    if (a.prompt) {
        if (a.n_split != 1 || a.waves > 4 || group > 8) return hipErrorInvalidValue;
        if (a.c.head_dim == 64) launch_prompt_d<64>(a, (unsigned)prompt_blocks(a), 64u * a.waves, lds, s);
        else if (a.c.head_dim == 128) launch_prompt_d<128>(a, (unsigned)prompt_blocks(a), 64u * a.waves, lds, s);
        else return hipErrorInvalidValue;
        return hipGetLastError();
    }
    if (a.c.head_dim == 64) launch_attention_d<64>(a, (unsigned)blocks, 64u * a.waves, lds, s);
    else if (a.c.head_dim == 128) launch_attention_d<128>(a, (unsigned)blocks, 64u * a.waves, lds, s);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace t3k
