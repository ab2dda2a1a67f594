// iam_kv8.h -- the 8-bit paged KV cache: what its launchers take (iam_kv8.cu: handle and append;
// iam_kv8_decode.cu, iam_kv8_rows.cu, iam_kv8_prompt.cu: attention of few query rows, of some and of prompts).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/iam_b200.h"

namespace iam {

constexpr int kKv8MaxItems = 1 << 16;  // row tiles of one attention call at most
constexpr int kKv8MaxTokens = 1 << 26; // tokens that a sequence's table can name
constexpr int kKv8Group = 16;          // tokens that share a page for sure (the smallest page)
constexpr unsigned kKv8ErrRange = 1u;  // error word: a page, length or row offset out of range, or more work than a call takes
constexpr unsigned kKv8ErrWait = 2u;   // a bounded wait gave up

// Scratch of a handle: partial results of row tiles whose context is split over several CTAs, the
// arrival counters of their joins (zero between calls) and the row-tile kernel's schedule.
struct Kv8Scratch {
    float* part;        // [2 * ctas][rows][head_dim + 4]
    size_t part_floats;
    int* ctr;           // one per CTA
    int max_ctas;
    int* plan;          // Kv8Plan words
    unsigned* err;
};

struct Kv8Attn {
    iam_kv8_cache c;
    const int32_t* cu;    // null: one row per sequence
    const int32_t* lens;
    int n_rows, n_heads, gq, window;
    float scale_log2;     // score scale times log2(e)
    iam_rows q, out;
    float* lse;
    Kv8Scratch s;
    int sms;
};

int kv8_decode_launch(const Kv8Attn& a, int dtype, cudaStream_t s);
int kv8_rows_launch(const Kv8Attn& a, int dtype, cudaStream_t s);
int kv8_prompt_launch(const Kv8Attn& a, int dtype, cudaStream_t s);  // 16-bit queries, head_dim 64 or 128
size_t kv8_decode_part_floats(int head_dim, int sms);
size_t kv8_rows_part_floats(int head_dim, int sms);
size_t kv8_prompt_part_floats(int head_dim, int sms);
int kv8_max_ctas(int sms);
size_t kv8_plan_words();

}  // namespace iam
