// Launch interface of the attention kernels (kv4.hip, prompt.hip) towards the
// C ABI (capi.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "grinqh.h"

namespace grinqh {

// Rows of a tensor [tokens][heads][head size]: element distances of tokens and
// heads, channels adjacent.
struct HeadRows {
  const uint16_t* p;
  int64_t token, head;
};

// The 4-bit cache, uint8 [pages][heads][sub][record]: sub records of 16 tokens
// per page and head.
struct Kv4Cache {
  uint8_t* p;
  int64_t pages;
  int heads, sub, head_size, groups;
};

constexpr int kv4_record_bytes(int head_size, int groups) { return 16 * head_size + 64 * (groups + 1); }

int launch_kv4_store(HeadRows k, HeadRows v, const int64_t* slots, int64_t tokens, const Kv4Cache& cache, int dtype,
                     hipStream_t st);
int launch_kv4_load(const Kv4Cache& cache, const int64_t* slots, int64_t tokens, uint16_t* k, uint16_t* v, int dtype,
                    hipStream_t st);

// How kv4_attention splits its sequences: runs of `chunk` steps of 32 tokens,
// at most `splits` of them.
struct Kv4Plan {
  int splits, chunk;
  size_t workspace;  // bytes, 0 if splits == 1
};
Kv4Plan plan_kv4(int64_t seqs, int heads, int kv_heads, int head_size, int64_t max_length);

struct Kv4Params {
  HeadRows q;
  uint16_t* out;  // [seqs][heads][head size]
  Kv4Cache cache;
  const int32_t* table;  // page table [seqs][table_width], rows table_stride apart
  int64_t table_stride;
  int table_width;
  const int32_t* lengths;
  int seqs, heads;
  float scale;
  Kv4Plan plan;
  float* partial;  // [seqs][heads][splits][head size + 2]
};
int launch_kv4_attention(const Kv4Params& p, int dtype, hipStream_t st);

struct PromptParams {
  HeadRows q, k, v;
  uint16_t* out;  // [q_tokens][heads][head size]
  const int32_t* ends;      // [seqs + 1] query row offsets
  const int32_t* key_ends;  // [seqs + 1] key offsets
  int64_t q_tokens, k_tokens;
  int seqs, heads, kv_heads, head_size;
  float scale;
};
int launch_prompt_attention(const PromptParams& p, int dtype, hipStream_t st);

}  // namespace grinqh
