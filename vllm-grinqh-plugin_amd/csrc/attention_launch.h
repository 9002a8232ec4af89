// Launch interface of the attention kernels (kv4.hip, prompt.hip, chunk.hip,
// append.hip, select.hip) towards the C ABI (capi.hip).
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
  int heads, sub, head_size, groups;  // sub: a power of two
};

constexpr int kv4_record_bytes(int head_size, int groups) { return 16 * head_size + 64 * (groups + 1); }

int launch_kv4_store(HeadRows k, HeadRows v, const int64_t* slots, int64_t tokens, const Kv4Cache& cache, int dtype,
                     hipStream_t st);
int launch_kv4_load(const Kv4Cache& cache, const int64_t* slots, int64_t tokens, uint16_t* k, uint16_t* v, int dtype,
                    hipStream_t st);

// How kv4_attention shares its work out (find_share in kv4.hip); the lengths are
// known on the device only.
constexpr int64_t kKv4Counters = 1 << 15;  // units that can be shared by several blocks, one counter each
struct Kv4Plan {
  int waves;         // per block: 4 or 8
  int blocks;        // blocks that the steps of all units are shared out over
  int least, most;   // steps of a run at least, runs of a unit at most
  int slot;          // floats of a run's result in the workspace
  int64_t grid;      // blocks launched: one per unit and those that share one
  size_t workspace;  // bytes, 0 if no unit is shared
};
Kv4Plan plan_kv4(int64_t seqs, int heads, int kv_heads, int head_size, int64_t capacity);

struct Kv4Params {
  HeadRows q;
  uint16_t* out;  // [seqs][heads][head size]
  Kv4Cache cache;
  const int32_t* table;  // page table [seqs][table_width], rows table_stride apart
  int64_t table_stride;
  int64_t table_head;  // from one key/value head's row to the next; 0: one row for all heads
  int table_width;
  const int32_t* lengths;
  int seqs, heads;
  int sub_shift;  // log2(cache.sub)
  float scale;
  Kv4Plan plan;
  int units;          // per sequence: key/value heads x tiles of their query heads
  uint32_t* counters;  // [kKv4Counters], zero on entry and on exit
  float* partial;      // [plan.grid][plan.slot]
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

// Room for new tokens (append.hip).
struct AppendParams {
  int32_t* table;  // [seqs][table_width], rows table_stride apart; new pages are written
  int64_t table_stride;
  int table_width, page_shift;  // log2(page size)
  const int32_t *lengths, *counts;
  int seqs;
  const int32_t *free_pages, *free_count;
  int free_size;
  int tokens;
  int64_t* slots;      // [tokens]
  int32_t* positions;  // [tokens]
  int32_t* ends;       // [seqs + 1]
  int32_t* new_lengths;
  int32_t* new_free_count;
};
int launch_kv4_append(const AppendParams& p, hipStream_t st);

// How kv4_chunk_attention shares its work out (chunk.hip).
struct ChunkPlan {
  int waves;          // per block, 32 rows each
  int64_t units;      // blocks of rows, at most
  int blocks;         // runs that all tiles are shared out over where a unit may be split
  int least, most;    // tiles of a run at least, runs of a unit at most
  int64_t grid;
  int64_t slot;       // floats of a run's result in the workspace
  size_t workspace;   // bytes, 0 if no unit is split
};
ChunkPlan plan_chunk(int64_t tokens, int64_t seqs, int heads, int kv_heads, int head_size, int64_t capacity);

struct ChunkParams {
  HeadRows q;
  uint16_t* out;  // [tokens][heads][head size]
  Kv4Cache cache;
  const int32_t* table;
  int64_t table_stride;
  int table_width;
  const int32_t* lengths;
  const int32_t* ends;  // [seqs + 1]
  int64_t tokens;
  int seqs, heads;
  int sub_shift;
  float scale;
  ChunkPlan plan;
  float* partial;  // [plan.grid][plan.slot]
};
int launch_chunk_attention(const ChunkParams& p, int dtype, hipStream_t st);

// Summaries of pages and the selection by them (select.hip): int8 [pages][heads][head size + 16].
constexpr int summary_bytes(int head_size) { return head_size + 16; }
struct SummarizeParams {
  Kv4Cache cache;
  int8_t* summary;
  const int32_t* table;
  int64_t table_stride;
  int table_width;
  const int32_t *starts, *lengths;
  int seqs, sub_shift;
};
int launch_kv4_summarize(const SummarizeParams& p, hipStream_t st);

struct SelectParams {
  HeadRows q;
  const int8_t* summary;
  int64_t pages;
  int seqs, heads, kv_heads, head_size;
  const int32_t* table;
  int64_t table_stride;
  int table_width, page_shift;
  const int32_t* lengths;
  int count;
  float* scores;          // [seqs][kv_heads][table_width]
  int32_t* selected;      // [seqs][kv_heads][count]
  int32_t* new_lengths;   // [seqs]
};
int launch_kv4_select(const SelectParams& p, int dtype, hipStream_t st);

}  // namespace grinqh
