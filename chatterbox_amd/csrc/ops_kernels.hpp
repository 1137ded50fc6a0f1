// Launch wrappers of the serving operators on caller-owned device tensors (paged key-value cache, logits rules).
#pragma once
#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

namespace t3k {

// One layer's keys and values in pages: element (page, slot, head, i) of the keys is k[page * kp + slot * ks + head * kh + i].
// Key j of sequence s lives in page table[s * table_stride + j / page_size], slot j % page_size.
struct PagedCache {
    void* k = nullptr;
    void* v = nullptr;
    long long kp = 0, ks = 0, kh = 0, vp = 0, vs = 0, vh = 0;   // strides in elements (multiples of 16 bytes)
    const int* table = nullptr;
    long long table_stride = 0;
    int n_seqs = 0, max_pages = 0, n_pages = 0;
    int page_shift = 0;           // page_size = 1 << page_shift
    int kv_heads = 0, head_dim = 0, bf16 = 0;
};

struct PagedAppendArgs {
    PagedCache c;
    const void* k = nullptr;      // [rows, kv_heads, head_dim], float or bf16 (in_bf16)
    const void* v = nullptr;
    const void* q = nullptr;      // [rows, q_heads, head_dim] or nullptr
    void* q_out = nullptr;        // may be q
    long long kr = 0, kh = 0, vr = 0, vh = 0, qr = 0, qh = 0, qor = 0, qoh = 0;   // row and head strides in elements
    const float* cos = nullptr;   // [rope_len, >= head_dim / 2], row stride rope_stride; both nullptr: no rotation
    const float* sin = nullptr;
    long long rope_stride = 0;
    int rope_len = 0;
    const int* positions = nullptr;  // [rows]; < 0: the row is skipped
    const int* seq = nullptr;        // [rows] block-table row, or nullptr: row r belongs to sequence r
    int rows = 0, q_heads = 0, in_bf16 = 0;
};

struct PagedAttnArgs {
    PagedCache c;
    const void* q = nullptr;      // [rows, q_heads, head_dim], float or bf16 (q_bf16)
    void* out = nullptr;          // the same shape, float or bf16 (out_bf16)
    long long qr = 0, qh = 0, outr = 0, outh = 0;
    const int* lengths = nullptr; // [rows] keys of the row (+ length_add); < 0: the output row is left as it was
    const int* starts = nullptr;  // [rows] first key, or nullptr: 0
    const int* seq = nullptr;     // [rows] block-table row, or nullptr: identity
    float scale = 1.f;
    int rows = 0, q_heads = 0, q_bf16 = 0, out_bf16 = 0, max_length = 0, length_add = 0;
    int prompt = 0;               // 1: neighbouring rows mostly share a sequence; 2: in the mean four rows or more do, in any order (plan_paged_attention clears it where that is of no use)
    // filled by plan_paged_attention
    int n_split = 1;              // blocks a row's keys are shared by at most
    int tile_shift = 5;           // keys of a tile: 32, or 16 (fp32 cache)
    int min_tiles = 1;            // tiles that are worth a block
    int waves = 4;                // waves of a block
    int head_waves = 1;           // neighbouring key heads of a block (waves / head_waves share the keys of each)
    float* ws = nullptr;          // n_split > 1: [rows * q_heads * n_split] partial results of head_dim floats, then as many (max, sum)
};

struct LogitsArgs {
    const void* logits = nullptr; // [rows, vocab] float or bf16, row stride lr
    const void* uncond = nullptr; // [rows, vocab] or nullptr, row stride ur
    void* out = nullptr;          // [rows, vocab], row stride outr; may be logits
    long long lr = 0, ur = 0, outr = 0;
    int bf16 = 0, rows = 0, vocab = 0;
    float cfg_weight = 0.f;
    const int* tokens = nullptr;  // [rows, cap] row stride tr, or nullptr
    const int* n_tokens = nullptr;
    long long tr = 0;
    int cap = 0;
    const float* repetition = nullptr;  // [rows] or nullptr: the scalar
    const float* frequency = nullptr;
    const float* presence = nullptr;
    float repetition_s = 1.f, frequency_s = 0.f, presence_s = 0.f;
    const int* bias_ids = nullptr;      // [rows, n_bias], row stride br (0: one list for all rows)
    const float* bias_values = nullptr; // row stride bvr
    long long br = 0, bvr = 0;
    int n_bias = 0;
    const uint32_t* allowed = nullptr;  // [rows, >= ceil(vocab / 32)] bits, row stride ar (0: one mask for all rows)
    long long ar = 0;
};

// all launches are asynchronous on `s`, on the current device
hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s);
// how a call is cut into blocks, from its sizes and types alone; the workspace that takes
void plan_paged_attention(PagedAttnArgs& a);
size_t paged_attention_workspace(const PagedAttnArgs& a);
hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t s);
hipError_t launch_process_logits(const LogitsArgs& a, hipStream_t s);

}  // namespace t3k
