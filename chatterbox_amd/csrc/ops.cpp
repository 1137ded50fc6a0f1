// t3mi C ABI: the serving operators on caller-owned device tensors (include/t3mi.h).  Argument checks and launches; no state.
#include "t3mi.h"

#include <hip/hip_runtime_api.h>

#include <string>

#include "ops_kernels.hpp"

int t3mi_set_error(int code, const std::string& msg);   // t3mi.cpp

namespace {

// (no exception leaves these: without memory for its text an error keeps its code)
int say(int code, const char* where, const char* what) {
    try {
        return t3mi_set_error(code, std::string(where) + ": " + what);
    } catch (...) {
        return code;
    }
}
int bad(const char* where, const char* what) { return say(T3MI_ERR_ARG, where, what); }

// the operators' device, for the length of a call; the caller's current device afterwards
struct OnDevice {
    int before = -1, device;
    hipError_t err;
    explicit OnDevice(int d) : device(d) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
    }
    ~OnDevice() {
        if (before >= 0 && before != device) (void)hipSetDevice(before);
    }
};

int done(const char* where, hipError_t e) {
    if (e == hipSuccess) return T3MI_OK;
    return say(T3MI_ERR_HIP, where, hipGetErrorString(e));
}

bool is_type(int t) { return t == T3MI_W_F32 || t == T3MI_W_BF16; }
bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool at4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
bool step16(int64_t s, int dtype) { return s >= 0 && ((s * (dtype == T3MI_W_BF16 ? 2 : 4)) & 15) == 0; }
template <int N> bool steps16(const int64_t (&s)[N], int dtype) {
    for (int i = 0; i < N; ++i)
        if (!step16(s[i], dtype)) return false;
    return true;
}

// whether what is written through N strides never falls on itself: sorted by stride, each dimension steps over all that lies within it
template <int N> bool disjoint(const int64_t (&stride)[N], const int64_t (&count)[N], int64_t inner) {
    int by[N];
    for (int i = 0; i < N; ++i) {
        int j = i;
        for (; j > 0 && stride[by[j - 1]] > stride[i]; --j) by[j] = by[j - 1];
        by[j] = i;
    }
    int64_t extent = inner;
    for (int i = 0; i < N; ++i) {
        if (count[by[i]] <= 1) continue;
        if (stride[by[i]] < extent) return false;
        if (stride[by[i]] > (INT64_MAX - extent) / (count[by[i]] - 1)) return true;   // (past any address)
        extent += stride[by[i]] * (count[by[i]] - 1);
    }
    return true;
}

// runs of `inner` elements of `bytes` each, in up to three dimensions
struct Runs {
    const void* p;
    int64_t stride[3], count[3];
    int64_t inner;
    int bytes;
};
// whether two tensors share no memory: apart as a whole, or woven into each other with the same strides and a distance that keeps them apart
// (anything else is taken to share)
bool apart(const Runs& a, const Runs& b) {
    if (!a.p || !b.p) return true;
    typedef __int128 wide;
    const auto from = [](const Runs& t) { return (wide)reinterpret_cast<uintptr_t>(t.p); };
    const auto to = [&](const Runs& t) {
        wide n = t.inner;
        for (int d = 0; d < 3; ++d) n += (wide)(t.count[d] - 1) * t.stride[d];
        return from(t) + n * t.bytes;
    };
    for (int d = 0; d < 3; ++d)
        if (a.count[d] <= 0 || b.count[d] <= 0) return true;
    if (to(a) <= from(b) || to(b) <= from(a)) return true;
    int64_t stride[3];                               // common to both; 0: neither takes a second step, or has one to take
    int by[3];                                       // dimensions, the largest step first
    for (int d = 0; d < 3; ++d) {
        if (a.count[d] > 1 && b.count[d] > 1 && a.stride[d] != b.stride[d]) return false;
        stride[d] = a.count[d] > 1 ? a.stride[d] : b.count[d] > 1 ? b.stride[d] : 0;
        int j = d;
        for (; j > 0 && stride[by[j - 1]] < stride[d]; --j) by[j] = by[j - 1];
        by[j] = d;
    }
    const wide off = from(b) - from(a);
    if (a.bytes != b.bytes || off % a.bytes) return false;
    // within one step of a dimension that every larger step is a multiple of: what lies in the smaller dimensions, side by side
    for (int i = 0; i < 3 && stride[by[i]] > 0; ++i) {
        const int64_t step = stride[by[i]];
        bool whole = true;
        for (int j = 0; j < i; ++j) whole = whole && stride[by[j]] % step == 0;
        wide at = off / a.bytes % step, in_a = a.inner, in_b = b.inner;
        if (at < 0) at += step;
        for (int j = i + 1; j < 3; ++j) {
            in_a += (wide)(a.count[by[j]] - 1) * stride[by[j]];
            in_b += (wide)(b.count[by[j]] - 1) * stride[by[j]];
        }
        if (whole && at >= in_a && at + in_b <= step) return true;
    }
    return false;
}
Runs runs(const void* p, const int64_t (&stride)[2], int64_t rows, int64_t heads, int64_t inner, int dtype) {
    return {p, {stride[0], stride[1], 0}, {rows, heads, 1}, inner, dtype == T3MI_W_BF16 ? 2 : 4};
}
Runs pages(const t3mi_paged_cache* c, const void* p, const int64_t (&s)[3]) {
    return {p, {s[0], s[1], s[2]}, {c->n_pages, c->page_size, c->kv_heads}, c->head_dim, c->dtype == T3MI_W_BF16 ? 2 : 4};
}

int take_cache(const char* where, const t3mi_paged_cache* c, t3k::PagedCache& o) {
    if (!c) return bad(where, "null cache");
    if (!c->k || !c->v || !c->block_table) return bad(where, "the cache has a null pointer");
    if (!is_type(c->dtype)) return bad(where, "cache dtype must be T3MI_W_F32 or T3MI_W_BF16");
    if (c->head_dim != 64 && c->head_dim != 128) return bad(where, "head_dim must be 64 or 128");
    if (c->kv_heads <= 0 || c->n_seqs <= 0 || c->max_pages <= 0 || c->n_pages <= 0) return bad(where, "cache extents must be positive");
    if (c->page_size <= 0 || c->page_size > 65536 || (c->page_size & (c->page_size - 1))) return bad(where, "page_size must be a power of two, at most 65536");
    if ((int64_t)c->max_pages * c->page_size > 0x7FFFFF00LL) return bad(where, "a sequence may have at most 2^31 - 256 keys");
    if (!at16(c->k) || !at16(c->v) || !steps16(c->k_stride, c->dtype) || !steps16(c->v_stride, c->dtype))
        return bad(where, "cache addresses and strides must be multiples of 16 bytes");
    if (!at4(c->block_table) || c->table_stride < 0) return bad(where, "bad block table");
    o.k = c->k; o.v = c->v;
    o.kp = c->k_stride[0]; o.ks = c->k_stride[1]; o.kh = c->k_stride[2];
    o.vp = c->v_stride[0]; o.vs = c->v_stride[1]; o.vh = c->v_stride[2];
    o.table = c->block_table; o.table_stride = c->table_stride;
    o.n_seqs = c->n_seqs; o.max_pages = c->max_pages; o.n_pages = c->n_pages;
    o.page_shift = __builtin_ctz((unsigned)c->page_size);
    // (the attention kernel addresses a tile of 32 slots by 32-bit offsets)
    if (c->k_stride[1] > (1 << 24) || c->v_stride[1] > (1 << 24)) return bad(where, "slot strides may be at most 2^24 elements");
    o.kv_heads = c->kv_heads; o.head_dim = c->head_dim; o.bf16 = c->dtype == T3MI_W_BF16;
    return T3MI_OK;
}

int take_attention(const char* where, const t3mi_paged_cache* cache, const t3mi_attention_args* a, t3k::PagedAttnArgs& o) {
    int rc = take_cache(where, cache, o.c);
    if (rc) return rc;
    if (!a) return bad(where, "null arguments");
    if (a->rows < 0 || a->q_heads <= 0 || a->q_heads % cache->kv_heads) return bad(where, "q_heads must be a positive multiple of kv_heads");
    if (!is_type(a->q_dtype) || !is_type(a->out_dtype)) return bad(where, "dtypes must be T3MI_W_F32 or T3MI_W_BF16");
    if (a->q_dtype == T3MI_W_BF16 && cache->dtype != T3MI_W_BF16) return bad(where, "bf16 queries need a bf16 cache");
    if (a->max_length < 0 || (a->length_add != 0 && a->length_add != 1)) return bad(where, "max_length must be >= 0, length_add 0 or 1");
    if ((int64_t)a->rows * a->q_heads > 0x1000000LL) return bad(where, "at most 2^24 (row, head) pairs a call");
    if (!(a->scale == a->scale) || a->scale - a->scale != 0.f) return bad(where, "scale must be finite");
    if (a->rows && (!a->q || !a->out || !a->lengths)) return bad(where, "null pointer");
    if (!at16(a->q) || !at16(a->out) || !steps16(a->q_stride, a->q_dtype) || !steps16(a->out_stride, a->out_dtype))
        return bad(where, "q and out: addresses and strides must be multiples of 16 bytes");
    if (!at4(a->lengths) || !at4(a->starts) || !at4(a->seq)) return bad(where, "lengths, starts and seq must be aligned to 4 bytes");
    if (!a->seq && a->rows > cache->n_seqs) return bad(where, "more rows than sequences (seq says which row belongs to which)");
    if (a->q == a->out && (a->q_dtype != a->out_dtype || a->q_stride[0] != a->out_stride[0] || a->q_stride[1] != a->out_stride[1]))
        if (a->rows) return bad(where, "out may be q only with the same strides and type");
    if (!disjoint<2>(a->out_stride, {a->rows, a->q_heads}, cache->head_dim)) return bad(where, "the rows and heads of out must not overlap");
    if (a->q != a->out && !apart(runs(a->q, a->q_stride, a->rows, a->q_heads, cache->head_dim, a->q_dtype),
                                 runs(a->out, a->out_stride, a->rows, a->q_heads, cache->head_dim, a->out_dtype)))
        return bad(where, "out must not share memory with q (but be q)");
    o.q = a->q; o.out = a->out;
    o.qr = a->q_stride[0]; o.qh = a->q_stride[1]; o.outr = a->out_stride[0]; o.outh = a->out_stride[1];
    o.lengths = a->lengths; o.starts = a->starts; o.seq = a->seq;
    o.scale = a->scale; o.rows = a->rows; o.q_heads = a->q_heads;
    o.q_bf16 = a->q_dtype == T3MI_W_BF16; o.out_bf16 = a->out_dtype == T3MI_W_BF16;
    const int64_t most = (int64_t)cache->max_pages * cache->page_size;
    o.max_length = (int)(a->max_length > 0 && a->max_length < most ? a->max_length : most);
    o.length_add = a->length_add;
    if (a->prompt < -1 || a->prompt > 1) return bad(where, "prompt must be -1, 0 or 1");
    // (of one sequence any rows are neighbours)
    o.prompt = a->prompt > 0 ? 1 : (a->prompt == 0 && a->seq && (int64_t)a->rows >= 4LL * cache->n_seqs ? (cache->n_seqs == 1 ? 1 : 2) : 0);
    return T3MI_OK;
}

}  // namespace

extern "C" {

int t3mi_paged_append(const t3mi_paged_cache* cache, const t3mi_append_args* a, void* stream) {
    const char* me = "t3mi_paged_append";
    t3k::PagedAppendArgs o;
    int rc = take_cache(me, cache, o.c);
    if (rc) return rc;
    if (!a) return bad(me, "null arguments");
    if (a->rows < 0) return bad(me, "rows must be >= 0");
    if (!is_type(a->dtype)) return bad(me, "dtype must be T3MI_W_F32 or T3MI_W_BF16");
    if ((a->q != nullptr) != (a->q_out != nullptr)) return bad(me, "q and q_out go together");
    if (a->q && a->q_heads <= 0) return bad(me, "q_heads must be positive");
    if ((a->cos != nullptr) != (a->sin != nullptr)) return bad(me, "cos and sin go together");
    if (a->cos && (a->rope_len <= 0 || a->rope_stride < 0)) return bad(me, "bad rotation tables");
    if (a->rows && (!a->k || !a->v || !a->positions)) return bad(me, "null pointer");
    if (!at16(a->k) || !at16(a->v) || !at16(a->q) || !at16(a->q_out) || !steps16(a->k_stride, a->dtype) || !steps16(a->v_stride, a->dtype) ||
        (a->q && (!steps16(a->q_stride, a->dtype) || !steps16(a->q_out_stride, a->dtype))))
        return bad(me, "k, v, q and q_out: addresses and strides must be multiples of 16 bytes");
    if (!at4(a->cos) || !at4(a->sin)) return bad(me, "rotation tables must be aligned to 4 bytes");
    if (!at4(a->positions) || !at4(a->seq)) return bad(me, "positions and seq must be aligned to 4 bytes");
    if (a->q && a->q == a->q_out && (a->q_stride[0] != a->q_out_stride[0] || a->q_stride[1] != a->q_out_stride[1]))
        return bad(me, "q_out may be q only with the same strides");
    if (!a->seq && a->rows > cache->n_seqs) return bad(me, "more rows than sequences (seq says which row belongs to which)");
    if ((int64_t)a->rows * ((a->q ? a->q_heads : 0) + 2LL * cache->kv_heads) > 0x8000000LL) return bad(me, "at most 2^27 (row, head) pairs a call");
    if (a->rows == 0) return T3MI_OK;
    if (a->q && !disjoint<2>(a->q_out_stride, {a->rows, a->q_heads}, cache->head_dim)) return bad(me, "the rows and heads of q_out must not overlap");
    if (!disjoint<3>(cache->k_stride, {cache->n_pages, cache->page_size, cache->kv_heads}, cache->head_dim) ||
        !disjoint<3>(cache->v_stride, {cache->n_pages, cache->page_size, cache->kv_heads}, cache->head_dim) ||
        !apart(pages(cache, cache->k, cache->k_stride), pages(cache, cache->v, cache->v_stride)))
        return bad(me, "the pages, slots and heads of the cache must not overlap");
    if (a->q) {
        const Runs out = runs(a->q_out, a->q_out_stride, a->rows, a->q_heads, cache->head_dim, a->dtype);
        if ((a->q != a->q_out && !apart(runs(a->q, a->q_stride, a->rows, a->q_heads, cache->head_dim, a->dtype), out)) ||
            !apart(runs(a->k, a->k_stride, a->rows, cache->kv_heads, cache->head_dim, a->dtype), out) ||
            !apart(runs(a->v, a->v_stride, a->rows, cache->kv_heads, cache->head_dim, a->dtype), out))
            return bad(me, "q_out must not share memory with q (but be q), k or v");
    }
    o.k = a->k; o.v = a->v; o.q = a->q; o.q_out = a->q_out;
    o.kr = a->k_stride[0]; o.kh = a->k_stride[1]; o.vr = a->v_stride[0]; o.vh = a->v_stride[1];
    o.qr = a->q_stride[0]; o.qh = a->q_stride[1]; o.qor = a->q_out_stride[0]; o.qoh = a->q_out_stride[1];
    o.cos = a->cos; o.sin = a->sin; o.rope_stride = a->rope_stride; o.rope_len = a->rope_len;
    o.positions = a->positions; o.seq = a->seq; o.rows = a->rows; o.q_heads = a->q ? a->q_heads : 0; o.in_bf16 = a->dtype == T3MI_W_BF16;
    OnDevice dev(cache->device);
    if (dev.err != hipSuccess) return done(me, dev.err);
    return done(me, t3k::launch_paged_append(o, (hipStream_t)stream));
}

int t3mi_paged_attention_workspace(const t3mi_paged_cache* cache, const t3mi_attention_args* args, size_t* bytes) {
    const char* me = "t3mi_paged_attention_workspace";
    if (!bytes) return bad(me, "null result");
    t3k::PagedAttnArgs o;
    int rc = take_attention(me, cache, args, o);
    if (rc) return rc;
    *bytes = 0;
    if (o.rows == 0) return T3MI_OK;
    t3k::plan_paged_attention(o);
    *bytes = t3k::paged_attention_workspace(o);
    return T3MI_OK;
}

int t3mi_paged_attention(const t3mi_paged_cache* cache, const t3mi_attention_args* args, void* stream) {
    const char* me = "t3mi_paged_attention";
    t3k::PagedAttnArgs o;
    int rc = take_attention(me, cache, args, o);
    if (rc) return rc;
    if (o.rows == 0) return T3MI_OK;
    t3k::plan_paged_attention(o);
    const size_t need = t3k::paged_attention_workspace(o);
    if (need > 0 && (!args->workspace || !at16(args->workspace) || args->workspace_bytes < need))
        return bad(me, "the workspace is smaller than t3mi_paged_attention_workspace says, or not aligned to 16 bytes");
    o.ws = static_cast<float*>(args->workspace);
    OnDevice dev(cache->device);
    if (dev.err != hipSuccess) return done(me, dev.err);
    return done(me, t3k::launch_paged_attention(o, (hipStream_t)stream));
}

int t3mi_process_logits(const t3mi_logits_args* a, void* stream) {
    const char* me = "t3mi_process_logits";
    if (!a) return bad(me, "null arguments");
    if (a->rows < 0 || a->rows > 65535 || a->vocab <= 0 || a->vocab > (1 << 28)) return bad(me, "rows must be 0..65535, vocab 1..2^28");
    if (!is_type(a->dtype)) return bad(me, "dtype must be T3MI_W_F32 or T3MI_W_BF16");
    if (a->rows && (!a->logits || !a->out)) return bad(me, "null logits or out");
    const uintptr_t low = a->dtype == T3MI_W_BF16 ? 1u : 3u;
    if (((reinterpret_cast<uintptr_t>(a->logits) | reinterpret_cast<uintptr_t>(a->uncond) | reinterpret_cast<uintptr_t>(a->out)) & low) != 0)
        return bad(me, "logits must be aligned to their elements");
    if (a->logits_stride < 0 || a->uncond_stride < 0 || a->tokens_stride < 0 || a->bias_ids_stride < 0 || a->bias_values_stride < 0 || a->allowed_stride < 0)
        return bad(me, "strides must be >= 0");
    if (a->rows > 1 && a->out_stride < a->vocab) return bad(me, "the rows of out must not overlap");
    if (a->out == a->logits && a->rows > 1 && a->out_stride != a->logits_stride) return bad(me, "out may be logits only with the same stride");
    if (a->tokens && (!a->n_tokens || a->token_cap < 0 || a->token_cap > 1048575)) return bad(me, "tokens need n_tokens and a token_cap of 0..1048575");
    if (a->n_bias < 0 || a->n_bias > 4094 || (a->n_bias > 0 && (!a->bias_ids || !a->bias_values))) return bad(me, "n_bias must be 0..4094, with ids and values");
    if (!a->repetition_each && !(a->repetition > 0.f)) return bad(me, "repetition must be > 0");
    if (!at4(a->tokens) || !at4(a->n_tokens) || !at4(a->bias_ids) || !at4(a->bias_values) || !at4(a->allowed) || !at4(a->repetition_each) ||
        !at4(a->frequency_each) || !at4(a->presence_each))
        return bad(me, "arrays must be aligned to 4 bytes");
    if (a->rows == 0) return T3MI_OK;
    const Runs out = runs(a->out, {a->out_stride, 0}, a->rows, 1, a->vocab, a->dtype);
    if ((a->out != a->logits && !apart(runs(a->logits, {a->logits_stride, 0}, a->rows, 1, a->vocab, a->dtype), out)) ||
        !apart(runs(a->uncond, {a->uncond_stride, 0}, a->rows, 1, a->vocab, a->dtype), out))
        return bad(me, "out must not share memory with logits (but be logits) or uncond");
    t3k::LogitsArgs o;
    o.logits = a->logits; o.uncond = a->uncond; o.out = a->out;
    o.lr = a->logits_stride; o.ur = a->uncond_stride; o.outr = a->out_stride;
    o.bf16 = a->dtype == T3MI_W_BF16; o.rows = a->rows; o.vocab = a->vocab; o.cfg_weight = a->cfg_weight;
    o.tokens = a->tokens; o.n_tokens = a->n_tokens; o.tr = a->tokens_stride; o.cap = a->token_cap;
    o.repetition = a->repetition_each; o.frequency = a->frequency_each; o.presence = a->presence_each;
    o.repetition_s = a->repetition; o.frequency_s = a->frequency; o.presence_s = a->presence;
    o.bias_ids = a->bias_ids; o.bias_values = a->bias_values; o.br = a->bias_ids_stride; o.bvr = a->bias_values_stride; o.n_bias = a->n_bias;
    o.allowed = a->allowed; o.ar = a->allowed_stride;
    OnDevice dev(a->device);
    if (dev.err != hipSuccess) return done(me, dev.err);
    return done(me, t3k::launch_process_logits(o, (hipStream_t)stream));
}

}  // extern "C"
