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

// A packed batch of chunks, and how one of the kernels that serve it shares its part
// out (chunk_share.h).
struct ChunkBatch {
  const int32_t* ends;     // [seqs + 1] row offsets
  const int32_t* lengths;  // tokens in the cache
  int tokens, seqs, capacity;
  int kv_heads, per;       // query heads of a key/value head
  int64_t least_rows, most_rows;  // (token, query head) pairs of the sequences that this kernel takes
  bool edges;              // and the rows in front of the first and behind the last
  int block_rows, tile;    // powers of two, as `blocks`
  // tiles are shared out over so many blocks, runs of at least so many tiles, a unit split into so many at most
  int blocks, least, most;
  int64_t units;            // at most
  int pieces;               // results that the workspace holds, where the tile kernel's blocks take equal pieces; or 0
  int rows_shift, tile_shift, blocks_shift, heads_shift, per_shift;  // log2 (of kv_heads and per: -1 if it is none)
};

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
// The same for chunks of few tokens: q and out [tokens][heads][head size], plan.most, .blocks and .least from the batch.
int launch_kv4_attention_rows(const Kv4Params& p, const ChunkBatch& batch, int dtype, hipStream_t st);

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

// How kv4_chunk_attention is served: sequences with up to few_rows (token, query head) pairs
// per key/value head by the single-token kernel (kv4.hip), the others by the tile
// kernel (chunk.hip), or all by one of them (plan_chunk).
struct ChunkPart {
  int64_t grid;             // blocks; 0: not used
  int64_t units;            // blocks of rows and head, at most
  int waves, block_rows, tile;
  int blocks, least, most;  // as in ChunkBatch
  int64_t slot;             // floats of a run's (piece's) result
  int pieces;               // results in the workspace
  size_t partial;           // where the runs' results stand in the workspace, in bytes
};
struct ChunkPlan {
  ChunkPart few, tiles;
  int few_rows;
  size_t workspace;  // bytes, 0 if no unit is split; kKv4Counters counters, then the runs' results
};
ChunkPlan plan_chunk(int64_t tokens, int64_t seqs, int heads, int kv_heads, int head_size, int64_t capacity);

struct ChunkParams {
  HeadRows q;
  uint16_t* out;  // [tokens][heads][head size]
  Kv4Cache cache;
  const int32_t* table;
  int64_t table_stride;
  int sub_shift, heads;
  float scale;
  ChunkBatch batch;
  int64_t grid, slot;
  float* partial;  // [batch.pieces][slot]
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
bool kv4_select_fits(int table_width);  // in one launch, without scores in the workspace
int launch_kv4_select(const SelectParams& p, int dtype, hipStream_t st);

}  // namespace grinqh
