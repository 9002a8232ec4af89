// Which rows and tokens of a packed batch of chunks a block takes (kv4.hip for
// sequences with few rows, chunk.hip for the others).
#pragma once
#include "attention_launch.h"
#include "wave_scan.h"

namespace grinqh {

// Sequence -1 stands for the rows in front of the first sequence, sequence `seqs` for
// those behind the last: they see no token, and their results are zeros.
struct ChunkSequence {
  int row0, rows;  // tokens of the chunk
  int length;      // tokens in the cache that count
  bool bad;        // more than the page table covers
};
__device__ __forceinline__ ChunkSequence chunk_sequence(const ChunkBatch& b, int s) {
  // all loads at once, whatever s stands for
  const int from = b.ends[min(max(s, 0), b.seqs)], to = b.ends[min(max(s + 1, 0), b.seqs)];
  const int held = b.seqs > 0 ? b.lengths[min(max(s, 0), b.seqs - 1)] : 0;
  const bool inside = s >= 0 && s < b.seqs;
  ChunkSequence q;
  q.row0 = s < 0 ? 0 : min(max(from, 0), b.tokens);
  q.rows = max((s >= b.seqs ? b.tokens : min(max(to, 0), b.tokens)) - q.row0, 0);
  q.bad = inside && held > b.capacity;
  q.length = inside ? min(max(held, 0), b.capacity) : 0;
  return q;
}

// x / d for x >= 0, d > 0; shift: log2(d) where d is a power of two, otherwise negative.
__device__ __forceinline__ int quotient(int x, int d, int shift) { return shift >= 0 ? x >> shift : x / d; }

// Blocks of rows of sequence s that this kernel takes, and tiles of its tokens.
__device__ __forceinline__ int chunk_blocks(const ChunkBatch& b, const ChunkSequence& q, int s) {
  const int64_t rows = (int64_t)q.rows * b.per;
  const bool edge = s < 0 || s >= b.seqs;
  if (edge ? !b.edges : rows < b.least_rows || rows > b.most_rows) return 0;
  return (int)((rows + b.block_rows - 1) >> b.rows_shift);
}
__device__ __forceinline__ int chunk_tiles(const ChunkBatch& b, const ChunkSequence& q) {
  return (int)(((int64_t)q.length + b.tile - 1) >> b.tile_shift);
}

struct ChunkShare {
  ChunkSequence q;
  int seq, head;   // key/value head
  int block;       // of rows, in the sequence
  int run, runs;
  int64_t unit;    // of a split unit: its number,
  int64_t slot;    // its first place in the workspace, its runs one after the other
};

// Every block plans by itself from the offsets and lengths, which only the device
// knows: units are blocks of b.block_rows rows ((token, query head) pairs) of a
// key/value head, and the tiles of b.tile tokens that they read are shared out over
// b.blocks: a unit is split into as many runs as it has shares of at least b.least
// tiles, all units of a sequence alike, so that split units have b.blocks runs at most
// and a batch with fewer units than that runs in one round.  All blocks look at all
// sequences, 64 at a time: single rows of 500 tokens, 8 heads of 128 channels, take 13, 41, 240 and 1710 us
// in batches of 64, 256, 1024 and 4096 (kv4_attention: 13, 34, 135, 561).  With `joined` blocks stand
// for split units.  False: past the last one.
__device__ __forceinline__ bool find_chunk(const ChunkBatch& b, int64_t id, bool joined, int lane, ChunkShare& out) {
  const int heads = b.kv_heads;
  auto blocks_of = [&](const ChunkSequence& q, int s) { return chunk_blocks(b, q, s); };
  auto tiles_of = [&](const ChunkSequence& q) { return chunk_tiles(b, q); };
  // the first 64 are looked at once
  ChunkSequence q = {0, 0, 0, false};
  if (lane - 1 <= b.seqs) q = chunk_sequence(b, lane - 1);
  int chunk = 1;
  if (b.most > 1) {
    float tiles = lane - 1 <= b.seqs ? (float)blocks_of(q, lane - 1) * (float)tiles_of(q) : 0.f;
    for (int s = lane + 63; s < b.seqs; s += 64) {
      const ChunkSequence other = chunk_sequence(b, s);
      tiles += (float)blocks_of(other, s) * (float)tiles_of(other);
    }
    const float total =
        __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_scan(tiles)), 63));
    chunk = max(b.least, (int)ceilf(fminf(total * (float)heads / (float)b.blocks, 0x1p26f)));
  }
  int64_t before = 0, units_before = 0, slots_before = 0;
  for (int s0 = -1;;) {
    const int s = s0 + lane;
    int units = 0, runs = 1, units_per_head = 0;
    if (s <= b.seqs) {
      units_per_head = blocks_of(q, s);
      units = units_per_head * heads;
      if (b.most > 1) runs = min(max(tiles_of(q) / chunk, 1), b.most);
    }
    const int slots = runs > 1 ? units * runs : 0, items = joined ? (runs > 1 ? units : 0) : units * runs;
    const int upto = wave_scan(items);
    const uint64_t after = __ballot(before + upto > id);
    if (after != 0) {
      const int owner = __builtin_ctzll(after);
      auto of_owner = [&](int v) { return __builtin_amdgcn_readlane(v, owner); };
      out.seq = s0 + owner;
      out.q = {of_owner(q.row0), of_owner(q.rows), of_owner(q.length), of_owner((int)q.bad) != 0};
      out.runs = of_owner(runs);
      const int count = of_owner(units), rest = (int)(id - before) - (of_owner(upto) - of_owner(items));
      const int unit = joined || out.runs == 1 ? rest : rest / out.runs;
      if (unit < 0 || unit >= count) return false;  // offsets that are not ascending
      out.run = joined ? 0 : rest - unit * out.runs;
      out.unit = out.slot = 0;  // for the workspace
      if (out.runs > 1) {
        out.unit = units_before + of_owner(wave_scan(units)) - count + unit;
        out.slot = slots_before + of_owner(wave_scan(slots) - slots) + (int64_t)unit * out.runs;
      }
      const int block = quotient(unit, heads, b.heads_shift);
      out.head = unit - block * heads;
      out.block = of_owner(units_per_head) - 1 - block;  // those with the most tokens first
      // more than the workspace was made for: offsets that are not ascending
      return out.runs == 1 || (out.unit < b.units && out.slot + out.runs <= b.blocks);
    }
    s0 += 64;
    if (s0 > b.seqs) return false;
    before += __builtin_amdgcn_readlane(upto, 63);
    units_before += __builtin_amdgcn_readlane(wave_scan(units), 63);
    slots_before += __builtin_amdgcn_readlane(wave_scan(slots), 63);
    if (s0 + lane <= b.seqs) q = chunk_sequence(b, s0 + lane);
  }
}

}  // namespace grinqh
