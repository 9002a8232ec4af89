// Attention of chunks of new tokens over the 4-bit cache: packed rows, paged keys
// and values, causal, grouped heads.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j),  j <= i + (length - rows) of the sequence
//
// Rows of a block are (token, query head of one key/value head) pairs, so that all
// heads that share keys share the work of unpacking them: a tile of 64 tokens is
// loaded as it is kept, turned into fp16 by all threads together and left in LDS.
//
// A wave has 32 rows.  S^T = K Q^T and O^T = V^T P^T with 32x32x16 matrix instructions: a
// lane then holds one row's logits, so that its maximum and sum need one exchange with
// lane + 32, and the weights are the second product's operand as they come out (the
// values are read transposed, whose order of tokens is the logits').  The reference that
// is taken off the logits is raised only where a weight would pass 2^15, so most tiles
// leave O alone; it then is 7 below the largest logit (kRoom).
//
// Precision: queries are brought to 2^13 <= max < 2^14 by a power of two and rounded to fp16
// (exact unless a row spans more than fp16 holds); keys and values are rounded to fp16
// once, minimum + scale * code in one fused operation; weights to fp16, and summed as
// rounded.  A row's largest weight is between 2^7 and 2^15, so weights are normal fp16 numbers
// down to 2^-21 of it, and off by 2^-32 of it at most below: with one token above 32768 others by
// 17 nats, its value near zero, results are as exact as any (with the largest weight at 1 they were
// 3e-2 off).  Logits, references, sums and O are fp32.  Against 64 bits, fp16
// tensors, relative in the norm: 4.8e-4, which is half a step of the type (the results' own
// rounding is 2.1e-4 of that, and the single-token kernel, whose codes are exact, has
// 2.9e-4); bf16 tensors: 1.7e-3, their rounding alone.
//
// Bound by the vector unit's work for every token beside the products (2048 rows, a
// sequence of 32768 tokens, 32 query and 8 key/value heads of 128, 1065 GFLOP: 1090 us, 975
// TFLOP/s, a large library product reaches 1300; matrix unit 47 % of the cycles, vector unit
// 49, LDS 32, at the 1.77 GHz that the card holds under this load).  The tokens are unpacked
// by each of a head's 32 blocks of rows, 13 instructions for 8 codes or about a fifth of the
// vector unit's; the exponentials, their sums and their rounding are most of the rest.
// 256 rows share a tile: with 128, two blocks to a CU, 819 TFLOP/s instead of 917 (of an
// earlier version of both).  Heads of 256
// channels have registers for one wave per SIMD and 128 rows, so that nothing runs
// beside a wave that waits (2 sequences of 2500 tokens, 700 rows, 16 and 8 heads: 163 us, 400
// TFLOP/s, matrix unit 16 % of the cycles; 176 units on 256 CUs, and the longest of 40 tiles
// takes all that time).
#include <cfloat>
#include <type_traits>

#include "attention_launch.h"
#include "chunk_share.h"
#include "grinqh_common.h"

namespace grinqh {

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4_t;

constexpr int kKeys = 64;         // tokens per tile
constexpr float kLow = -FLT_MAX;  // running reference before the first token (finite: -inf - -inf would be NaN)
// A raised reference is so far below the largest logit that its weight is 2^7, and one that would pass 2^15 raises it
// again.  Less than 8, half of fp32's step at 2^27: the difference is rounded to one step at most there, and to none beyond.
constexpr float kRoom = 7.f, kRaise = 15.f;

__device__ __forceinline__ f32x16_t mfma32x32x16(const u32x4_t& a, const u32x4_t& b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0,
                                                0);
}
__device__ __forceinline__ uint32_t f16_pair(float lo, float hi) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{lo, hi}), f16x2_t));
}
__device__ __forceinline__ float half_lo(uint32_t w) { return f16_bits_to_f32((uint16_t)w); }
__device__ __forceinline__ float half_hi(uint32_t w) { return f16_bits_to_f32((uint16_t)(w >> 16)); }

// A result in the tensors' type; a mean of values next to fp16's limit may pass it by
// its weights' rounding and is limited.  NaN stays.
template <bool BF>
__device__ __forceinline__ uint32_t result_pair(float lo, float hi) {
  if constexpr (BF) return f32x2_to_bf16x2(lo, hi);
  lo = __builtin_elementwise_maximum(__builtin_elementwise_minimum(lo, 65504.f), -65504.f);
  hi = __builtin_elementwise_maximum(__builtin_elementwise_minimum(hi, 65504.f), -65504.f);
  return f16_pair(lo, hi);
}

// ---------------------------------------------------------------- which rows and tiles a block takes

// Units are blocks of rows of a sequence and a key/value head, and one block of threads fills a
// CU.  Where there is little to do a unit is split into equal runs if there are few
// (find_chunk).  That leaves half of the card idle with 128 long units, and 320 take as
// long as 512.  So long ones stand on a line, each as long as its tiles take, and all blocks
// take equal pieces of it: the end of one unit, whole ones, the beginning of another (2
// sequences of 8000 tokens, 512 rows each, 8 heads: 270 us split into runs, 200 so; 5 of
// 4000: 306, 248).  A unit that is cut leaves its parts in the workspace, two per block at
// most, and a second kernel joins them, which costs as much as some 22 tiles: blocks
// take a unit each where that is cheaper.  Lengths are in sixteenths of a tile; the d-th
// last block of rows of a sequence is c0 + (B - d) c1 long, so that sums have a closed form
// and every block finds its place by itself from the offsets and lengths, which only the
// device knows.
constexpr int kStart = 4;    // tiles that a unit takes beside its own
constexpr int kJoining = 22;  // tiles that cutting takes
struct Line {
  int total, width;
  bool pieces;  // otherwise a unit is 1 long, and its block's
};
struct Weight {
  int blocks, c0, c1;
  __device__ int before(int d) const { return d * c0 + c1 * (blocks * d - d * (d - 1) / 2); }  // blocks 0 .. d - 1
  __device__ int of(int d) const { return c0 + (blocks - d) * c1; }
};
__device__ __forceinline__ Weight weight_of(const ChunkBatch& b, const ChunkSequence& q, int s, bool pieces) {
  Weight w = {s <= b.seqs ? chunk_blocks(b, q, s) : 0, 1, 0};
  if (pieces) {
    w.c0 = 16 * kStart + max(q.length - q.rows, 0) / 4;
    w.c1 = s >= 0 && s < b.seqs ? (b.block_rows + 4 * b.per - 1) / (4 * b.per) : 0;
  }
  return w;
}
// `mine`: sequence lane - 1.
__device__ __forceinline__ Line line_of(const ChunkBatch& b, const ChunkSequence& mine, int lane) {
  int count = 0, all = 0, longest = 0;
  auto add = [&](const ChunkSequence& q, int s) {
    const Weight w = weight_of(b, q, s, true);
    count += w.blocks * b.kv_heads;
    all += w.before(w.blocks) * b.kv_heads;
    longest = w.blocks > 0 ? max(longest, chunk_tiles(b, q)) : longest;
  };
  if (lane - 1 <= b.seqs) add(mine, lane - 1);
  for (int s = lane + 63; s <= b.seqs; s += 64) add(chunk_sequence(b, s), s);
  count = wave_sum(count);
  all = wave_sum(all);
  longest = wave_reduce(longest, [](int x, int y) { return max(x, y); });
  const int piece = (all + b.blocks - 1) >> b.blocks_shift, rounds = (count + b.blocks - 1) >> b.blocks_shift;
  const float by_units = fmaxf((float)(longest + kStart), (float)rounds * ((float)all / (float)count) * (1.f / 16.f));
  if (count > 0 && all > 0 && (float)piece * (1.f / 16.f) + kJoining < by_units) return {all, piece, true};
  return {count, 1, false};
}

struct Piece {
  ChunkSequence q;
  int seq, head, block;  // of rows, in the sequence
  int length, at;        // the unit's length, and where in it the place is
};
// What stands at place x of the line.  False: past its end.
__device__ __forceinline__ bool find_piece(const ChunkBatch& b, const Line& l, const ChunkSequence& mine, int x, int lane,
                                           Piece& out) {
  int before = 0;
  for (int s0 = -1; s0 <= b.seqs; s0 += 64) {
    const int s = s0 + lane;
    const ChunkSequence q = s0 < 0 ? mine : chunk_sequence(b, s);
    const Weight w = weight_of(b, q, s, l.pieces);
    const int all = w.before(w.blocks) * b.kv_heads, upto = wave_scan(all);
    const uint64_t after = __ballot(before + upto > x);
    if (after != 0) {
      const int owner = __builtin_ctzll(after);
      auto of_owner = [&](int v) { return __builtin_amdgcn_readlane(v, owner); };
      const Weight o = {of_owner(w.blocks), of_owner(w.c0), of_owner(w.c1)};
      out.seq = s0 + owner;
      out.q = {of_owner(q.row0), of_owner(q.rows), of_owner(q.length), of_owner((int)q.bad) != 0};
      const int rest = x - before - (of_owner(upto) - of_owner(all));
      int d = 0, end = o.blocks;  // before(d) kv_heads <= rest < before(end) kv_heads
      if (rest < 0 || end <= 0) return false;  // offsets that are not ascending
      while (end - d > 1) {
        const int mid = (d + end) >> 1;
        if (o.before(mid) * b.kv_heads <= rest)
          d = mid;
        else
          end = mid;
      }
      out.length = o.of(d);
      const int inside = rest - o.before(d) * b.kv_heads;
      if (out.length <= 0 || inside < 0) return false;
      out.head = __builtin_amdgcn_readfirstlane(inside / out.length);  // a division leaves the scalar registers
      out.at = inside - out.head * out.length;
      out.block = o.blocks - 1 - d;  // those with the most tokens first
      return out.head < b.kv_heads;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}
// The tile at which a place in a unit of `tiles` tiles begins.
__device__ __forceinline__ int tile_at(int at, int length, int tiles) {
  return at >= length ? tiles : (int)((float)at * ((float)tiles / (float)length));
}

// ---------------------------------------------------------------- unpacking

// 8 codes as fp16 pairs minimum + scale * code (rounded once).  A nibble under the
// exponent of 1024 is 1024 + code, one in the upper half of a byte 1024 + 16 code.
__device__ __forceinline__ u32x4_t unpack8(uint32_t w, uint32_t pair) {
  const f16x2_t params = __builtin_bit_cast(f16x2_t, pair);
  const f16x2_t scale = {params[0], params[0]}, low = {params[1], params[1]};
  const uint32_t u = w >> 8;
  const f16x2_t one = (f16x2_t)((_Float16)-1024.f), sixteenth = (f16x2_t)((_Float16)0.0625f),
                less = (f16x2_t)((_Float16)-64.f);
  // (x & mask) | exponents in one operation: written out, as its two constants have to be in registers
  auto two = [&](uint32_t x, uint32_t mask, bool upper) {
    uint32_t bits;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(bits) : "v"(x), "s"(mask), "v"(0x64006400u));
    const f16x2_t c = __builtin_bit_cast(f16x2_t, bits);
    const f16x2_t code = upper ? __builtin_elementwise_fma(c, sixteenth, less) : c + one;
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(code, scale, low));
  };
  return u32x4_t{two(w, 0x000F000Fu, false), two(w, 0x00F000F0u, true), two(u, 0x000F000Fu, false),
                 two(u, 0x00F000F0u, true)};
}
// What the largest code of a group stands for.
__device__ __forceinline__ float reach_of(uint32_t pair) { return fmaf(15.f, half_lo(pair), half_hi(pair)); }
// Parameters whose codes fp16 can hold.  A scale that was rounded up makes the largest
// code stand for up to 65536: one step down brings it to 65504 at most (and the others
// a 2^-11 of the group's range lower at most).
__device__ __forceinline__ uint32_t within(uint32_t pair) {
  const float most = reach_of(pair);
  return most > 65504.f && most <= 65568.f ? pair - 1 : pair;
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&to)[N], const uint32_t* __restrict__ from) {
  if constexpr (N == 1) {
    to[0] = *from;
  } else if constexpr (N == 2) {
    const u32x2_t x = *reinterpret_cast<const u32x2_t*>(from);
    to[0] = x[0];
    to[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4_t x = *reinterpret_cast<const u32x4_t*>(from + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) to[i + j] = x[j];
    }
  }
}

// What a thread holds of a tile's keys and of its values, as the cache keeps them.
template <int D, int WAVES>
struct Raw {
  static constexpr int WORDS = D / (8 * WAVES);
  static constexpr int PAIRS = WORDS < D / 32 ? WORDS : D / 32;  // of the keys' parameters
  static constexpr int VEC = WORDS < 4 ? WORDS : 4;              // tokens of one chunk of the values
  static constexpr int VECS = WORDS / VEC;
};
template <int D, int WAVES>
struct RawKeys {
  uint32_t w[Raw<D, WAVES>::WORDS], pair[Raw<D, WAVES>::PAIRS];
  uint32_t value_pair;  // the token's values' parameters
  bool lost;            // its page is outside the cache
};
template <int D, int WAVES>
struct RawValues {
  uint32_t w[Raw<D, WAVES>::VECS][Raw<D, WAVES>::VEC], pair[Raw<D, WAVES>::VECS][Raw<D, WAVES>::VEC];
  bool lost;
};

// ---------------------------------------------------------------- the kernel

// PIECES: blocks take equal pieces of all work, not a run of a unit.
template <bool BF, int D, int WAVES, bool PIECES>
__global__ __launch_bounds__(64 * WAVES, D > 128 ? 1 : 2) void chunk_attention_kernel(const ChunkParams p) {
  constexpr int STEPS = D / 16, MT = D / 32, W = D / 32, THREADS = 64 * WAVES;
  // A row of keys (values) is 16 (64) bytes longer than it need be: the 32 adjacent
  // keys' chunks of one read, and 4 adjacent values' 64 bytes, then lie in different banks.
  constexpr int KEY_ROW = 2 * D + 16, VALUE_ROW = 2 * D + 64;
  __shared__ __align__(16) uint8_t s_k[2][kKeys * KEY_ROW], s_v[2][kKeys * VALUE_ROW];
  const int per = p.batch.per;
  ChunkSequence mine_of_lane;
  Line line;
  int begin = 0, end = 1;
  if constexpr (PIECES) {
    const int lane = threadIdx.x & 63;
    mine_of_lane = chunk_sequence(p.batch, lane - 1);
    line = line_of(p.batch, mine_of_lane, lane);
    if ((int64_t)blockIdx.x * line.width >= line.total) return;
    begin = (int)blockIdx.x * line.width;
    end = min(begin + line.width, line.total);
  }
  for (int x = begin; x < end;) {
  int tid = threadIdx.x;
  if constexpr (PIECES && D <= 128) asm volatile("" : "+v"(tid));  // what follows from it is not kept between units
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, half = lane >> 5;
  ChunkSequence sq;
  int seq, kvh, block, part, place, run = 0, runs = 1, unit_length = 1, unit_at = 0;
  bool whole;
  if constexpr (PIECES) {
    Piece share;
    if (!find_piece(p.batch, line, mine_of_lane, x, lane, share)) return;
    sq = share.q;
    seq = share.seq;
    kvh = share.head;
    block = share.block;
    unit_length = share.length;
    unit_at = share.at;
    part = min(unit_length - unit_at, end - x);
    whole = part == unit_length;
    place = 2 * (int)blockIdx.x + (x == begin ? 0 : 1);
    if (!whole && place >= p.batch.pieces) return;  // offsets that are not ascending
  } else {
    ChunkShare share;
    if (!find_chunk(p.batch, blockIdx.x, false, lane, share)) return;
    sq = share.q;
    seq = share.seq;
    kvh = share.head;
    block = share.block;
    run = share.run;
    runs = share.runs;
    part = 1;
    whole = runs == 1;
    place = (int)share.slot + run;
  }
  const int rows = sq.rows * per;                      // of the sequence: (token, head)
  const int row0 = (block * WAVES + wave) * 32;  // of this wave
  const bool live = row0 < rows;
  const int shift = sq.length - sq.rows;
  // this lane's row; past the last one it stands for the last and is not stored
  const int row = min(row0 + n, rows - 1);
  const int token = quotient(row, per, p.batch.per_shift), head = kvh * per + row - token * per;
  const int seen = token + shift;  // last token it sees

  // tiles of the block's last row, and this run's share
  const int last_row = min((block + 1) * (32 * WAVES), rows) - 1;
  const int tiles = max(quotient(last_row, per, p.batch.per_shift) + shift + kKeys, 0) / kKeys;
  int first = 0, last = tiles;
  if (!whole) {
    if constexpr (PIECES) {
      first = tile_at(unit_at, unit_length, tiles);
      last = tile_at(unit_at + part, unit_length, tiles);
    } else {
      const int each = (tiles + runs - 1) / runs;
      first = min(run * each, tiles);
      last = min(first + each, tiles);
    }
  }
  // this wave's: up to what its last row sees; masked from where its first one ends
  const int wave_seen = __builtin_amdgcn_readfirstlane(seen), wave_last = __builtin_amdgcn_readlane(seen, 31);
  const int my_last = live ? min(last, max(wave_last + kKeys, 0) / kKeys) : 0;

  // ---- a thread's share of a tile: WORDS words of one token's keys, as many of the values
  using R = Raw<D, WAVES>;
  const int key = tid / WAVES, key_word = tid % WAVES * R::WORDS;
  const int rec_of_tile = wave * 64 / (16 * WAVES), value_id = tid % (16 * WAVES);  // a wave's threads share a record
  static_assert(WAVES >= 4, "");
  const int groups = p.cache.groups, record = kv4_record_bytes(D, groups);
  const int pair_shift = __builtin_ctz((unsigned)(D / groups)) - 5;  // words i of a group share parameters
  const int last_rec = max((sq.length - 1) >> 4, 0);
  const int32_t* table = p.table + (int64_t)seq * p.table_stride;
  // tiles past the sequence's end stand for its last record: nothing uses them, and every load is in bounds
  auto page_of = [&](int tile) { return table[min(4 * tile + rec_of_tile, last_rec) >> p.sub_shift]; };
  auto record_of = [&](int tile, int page, bool& lost) {
    page = __builtin_amdgcn_readfirstlane(page);
    lost = (uint32_t)page >= (uint64_t)p.cache.pages;
    const int rec = min(4 * tile + rec_of_tile, last_rec);
    return reinterpret_cast<const uint32_t*>(
        p.cache.p + ((((int64_t)(lost ? 0 : page) * p.cache.heads + kvh) << p.sub_shift) +
                     (rec & (p.cache.sub - 1))) * record);
  };
  auto load_keys = [&](RawKeys<D, WAVES>& t, int tile, int page) {
    const uint32_t* w = record_of(tile, page, t.lost);
    load_words(t.w, w + (key & 15) * (D / 8) + key_word);
#pragma unroll
    for (int i = 0; i < R::PAIRS; ++i) t.pair[i] = w[2 * D + (((key_word + i) % W) >> pair_shift) * 16 + (key & 15)];
    t.value_pair = w[4 * D + 16 * groups + (key & 15)];
  };
  auto load_values = [&](RawValues<D, WAVES>& t, int tile, int page) {
    const uint32_t* v = record_of(tile, page, t.lost) + 2 * D + 16 * groups;
#pragma unroll
    for (int j = 0; j < R::VECS; ++j) {
      const int id = value_id + 16 * WAVES * j, chunk = id % (D / 8), token = id / (D / 8) * R::VEC;
      load_words(t.w[j], v + chunk * 16 + token);
      load_words(t.pair[j], v + 2 * D + token);
    }
  };
  // A token whose values are NaN (or lie outside the cache) gives zeros, and NaN as
  // its key: that reaches the rows that see it and no others, as the others' logits are
  // masked.  So does what no token was stored as, its largest code past what fp16 holds to either
  // side: it stands behind a sequence's end and must only stay finite.  All that takes one
  // test in most tiles.
  auto beyond = [](uint32_t pair) { return !(fabsf(reach_of(within(pair))) <= 65504.f); };
  auto settle_keys = [&](RawKeys<D, WAVES>& k) {
#pragma unroll
    for (int i = 0; i < R::PAIRS; ++i) k.pair[i] = k.lost || beyond(k.value_pair) ? 0x7E007E00u : within(k.pair[i]);
  };
  auto settle_raw = [&](RawKeys<D, WAVES>& k, RawValues<D, WAVES>& v) {
    float reach = fabsf(reach_of(k.value_pair));
#pragma unroll
    for (int i = 0; i < R::PAIRS; ++i) reach += fabsf(reach_of(k.pair[i]));
#pragma unroll
    for (int j = 0; j < R::VECS; ++j)
#pragma unroll
      for (int e = 0; e < R::VEC; ++e) reach += fabsf(reach_of(v.pair[j][e]));
    if (!__any(!(reach <= 65504.f)) && !k.lost && !v.lost) return;
    settle_keys(k);
#pragma unroll
    for (int j = 0; j < R::VECS; ++j)
#pragma unroll
      for (int e = 0; e < R::VEC; ++e) v.pair[j][e] = v.lost || beyond(v.pair[j][e]) ? 0u : within(v.pair[j][e]);
  };
  auto write_key = [&](const RawKeys<D, WAVES>& t, int i, uint8_t* to) {
    const int word = key_word + i, chunk = word / W + 4 * (word % W);
    const u32x4_t x = unpack8(t.w[i], t.pair[i % R::PAIRS]);
    *reinterpret_cast<u32x4_t*>(to + key * KEY_ROW + chunk * 16) = x;
  };
  auto write_value = [&](const RawValues<D, WAVES>& t, int i, uint8_t* to) {
    const int j = i / R::VEC, e = i % R::VEC;
    const int id = value_id + 16 * WAVES * j, chunk = id % (D / 8), token = id / (D / 8) * R::VEC + e;
    const u32x4_t x = unpack8(t.w[j][e], t.pair[j][e]);
    *reinterpret_cast<u32x4_t*>(to + (16 * rec_of_tile + token) * VALUE_ROW + chunk * 16) = x;
  };

  // ---- queries: row n, channels 16 s + 8 half + e, brought to 2^13 <= max < 2^14 by a power of two
  u32x4_t qf[STEPS];
  float unit;  // of the logits, in powers of two
  if (live) {
    const uint16_t* q = p.q.p + ((int64_t)sq.row0 + token) * p.q.token + (int64_t)head * p.q.head + 8 * half;
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      qf[s] = *reinterpret_cast<const u32x4_t*>(q + 16 * s);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint16_t x = (uint16_t)(qf[s][e >> 1] >> (16 * (e & 1)));
        top = fmaxf(top, fabsf(BF ? to_f32<BF16>(x) : to_f32<F16>(x)));
      }
    }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    int ex = 0;
    if (top > 0.f && top < __builtin_inff()) ex = min(13 - ilogbf(top), 100);
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint16_t a = (uint16_t)qf[s][i], b = (uint16_t)(qf[s][i] >> 16);
        qf[s][i] = BF ? f16_pair(ldexpf(to_f32<BF16>(a), ex), ldexpf(to_f32<BF16>(b), ex))
                      : f16_pair(ldexpf(to_f32<F16>(a), ex), ldexpf(to_f32<F16>(b), ex));
      }
    // never 0 or infinite, which times an infinite or a zero logit would be NaN
    unit = fminf(fmaxf(ldexpf(p.scale * 1.44269504088896f, -ex), FLT_MIN), FLT_MAX);
  }

  f32x16_t O[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) O[m] = (f32x16_t)(0.f);
  float M = kLow, sum = 0.f, zs = unit;
  bool far = false;  // logits are rounded before the reference is taken off (settle)

  // LDS reads.  Keys: row n of key block b, channels 16 s + 8 half + e.  Values, transposed:
  // channel 32 m + n, keys 16 t + 4 half + 0..3 and + 8.
  const int key_base = n * KEY_ROW + 16 * half;
  const int value_base = (4 * half + ((lane & 15) >> 2)) * VALUE_ROW + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
  auto read_key = [&](const uint8_t* kt, int b, int s) {
    return *reinterpret_cast<const u32x4_t*>(kt + key_base + 32 * b * KEY_ROW + 32 * s);
  };
  auto read_value = [&](const uint8_t* vt, int t, int m) {
    u32x4_t a;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4_t)(vt + value_base + (16 * t + 8 * u) * VALUE_ROW + 64 * m));
      const u32x2_t y = __builtin_bit_cast(u32x2_t, x);
      a[2 * u] = y[0];
      a[2 * u + 1] = y[1];
    }
    return a;
  };
  // S zs is exact in the exponent and M is not: the same factor for all tokens of a row,
  // but of more than 2^16 for logits past 2^28.  With `far` the product is rounded first.
  auto product_first = [&](f32x16_t (&S)[2]) {
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        S[b][e] *= unit;
        asm volatile("" : "+v"(S[b][e]));  // not contracted with the subtraction
      }
  };
  auto largest = [&](const f32x16_t (&S)[2]) {
    float top = -__builtin_inff();
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 16; e += 2) top = fmaxf(fmaxf(top, S[b][e]), S[b][e + 1]);
    return top;
  };
  // Makes S of a tile ready for its weights: the mask where the tile reaches past the
  // wave's first row's last token, and the reference raised where a weight would pass 2^15.
  auto settle = [&](f32x16_t (&S)[2], float top, int tile) {
    if (tile * kKeys + kKeys - 1 > wave_seen) {
      asm volatile("");  // a branch: as selects, this is a fourth of every tile's instructions
      // last token of this tile that the row sees, less the half's 4 (compared with constants)
      const int upto = seen - tile * kKeys - 4 * half;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (32 * b + (e & 3) + 8 * (e >> 2) > upto) S[b][e] = -__builtin_inff();
      top = largest(S);
    }
    if (far) {
      product_first(S);
      top = largest(S);
    }
    if (__any(fmaf(top, zs, -M) > kRaise)) {
      float m = fmaxf(M, top * zs - kRoom);
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      if (!far && __any(fabsf(m) > 0x1p24f && m != kLow)) {
        far = true;
        zs = 1.f;
        product_first(S);
        m = fmaxf(M, largest(S) - kRoom);
        m = fmaxf(m, __shfl_xor(m, 32, 64));
      }
      const float f = __builtin_amdgcn_exp2f(M - m);
      M = m;
      sum *= f;
#pragma unroll
      for (int t = 0; t < MT; ++t) O[t] *= f;
    }
  };
  u32x4_t P[4];
  // Weights of two tokens, pair q of key block b, as fp16 for the second product (off by 2^-11 of
  // them, or by 2^-25 below 2^-14); they are summed as rounded, in fp32.
  auto weigh = [&](const f32x16_t (&S)[2], int b, int q) {
    const float p0 = __builtin_amdgcn_exp2f(fmaf(S[b][2 * q], zs, -M));
    const float p1 = __builtin_amdgcn_exp2f(fmaf(S[b][2 * q + 1], zs, -M));
    const uint32_t pair = f16_pair(p0, p1);
    sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, pair), (f16x2_t)((_Float16)1.f), sum, false);
    P[2 * b + (q >> 2)][q & 3] = pair;
  };

  RawKeys<D, WAVES> keys;
  RawValues<D, WAVES> values;
  // One tile: its weights and its part of O, and the products of the next tile, slot by
  // slot: every slot gives the matrix unit one product and the vector unit a share
  // of the exponentials and, under the keys' products, of the unpacking (keys two tiles
  // ahead, values one).  What was unpacked makes room for the next loads, which then have
  // more than half a tile's time to arrive (1 sequence of 32768 tokens, 2048 rows, 32 heads of
  // 128: 1085 us, 1140 with loads at the tile's end).  Heads of 256 channels have no registers
  // for that: their values are unpacked under the values' products.
  constexpr bool EARLY = D <= 128;
  constexpr int KSLOTS = 2 * STEPS, VSLOTS = 4 * MT, AHEAD = PIECES && D == 128 ? 2 : 3, SETTLE = KSLOTS / 4;
  auto step = [&](f32x16_t (&S)[2], f32x16_t (&N)[2], const uint8_t* kt, const uint8_t* vt, uint8_t* k_to, uint8_t* v_to,
                  float& top, auto&& refill) {
    u32x4_t f[AHEAD + 1];
    auto read = [&](int at) {  // the A operand of slot `at`
      f[at % (AHEAD + 1)] =
          at < KSLOTS ? read_key(kt, at / STEPS, at % STEPS) : read_value(vt, (at - KSLOTS) / MT, (at - KSLOTS) % MT);
    };
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) read(k);
    if constexpr (!EARLY) settle_raw(keys, values);
    int done = 0, packed = 0;
#pragma unroll
    for (int k = 0; k < KSLOTS; ++k) {
      const int b = k / STEPS, s = k % STEPS;
      if (EARLY && k == SETTLE) settle_raw(keys, values);
      read(k + AHEAD);
      N[b] = mfma32x32x16(f[k % (AHEAD + 1)], qf[s], s == 0 ? (f32x16_t)(0.f) : N[b]);
#pragma unroll
      for (; done < (k + 1) * 8 / KSLOTS; ++done) weigh(S, 0, done);
      if constexpr (EARLY) {
#pragma unroll
        for (; k >= SETTLE && packed < (k + 1 - SETTLE) * 2 * R::WORDS / (KSLOTS - SETTLE); ++packed) {
          if (packed < R::WORDS)
            write_key(keys, packed, k_to);
          else
            write_value(values, packed - R::WORDS, v_to);
        }
      } else {
#pragma unroll
        for (; packed < (k + 1) * R::WORDS / KSLOTS; ++packed) write_key(keys, packed, k_to);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (EARLY) refill();
    done = packed = 0;
    int seen_of = 0;
    top = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < VSLOTS; ++k) {
      const int t = k / MT, m = k % MT;
      if (k + AHEAD < VSLOTS) read(KSLOTS + k + AHEAD);
      O[m] = mfma32x32x16(f[(KSLOTS + k) % (AHEAD + 1)], P[t], O[m]);
      if (k < VSLOTS / 2) {
#pragma unroll
        for (; done < (k + 1) * 8 / (VSLOTS / 2); ++done) weigh(S, 1, done);
      } else {
#pragma unroll
        for (; seen_of < (k + 1 - VSLOTS / 2) * 16 / (VSLOTS / 2); ++seen_of)
          top = fmaxf(fmaxf(top, N[seen_of >> 3][2 * (seen_of & 7)]), N[seen_of >> 3][2 * (seen_of & 7) + 1]);
      }
      if constexpr (!EARLY) {
#pragma unroll
        for (; packed < (k + 1) * R::WORDS / VSLOTS; ++packed) write_value(values, packed, v_to);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto for_keys = [&](const RawKeys<D, WAVES>& t, uint8_t* to) {
#pragma unroll
    for (int i = 0; i < R::WORDS; ++i) write_key(t, i, to);
  };
  auto feed_keys = [&](uint8_t* to) { for_keys(keys, to); };
  auto feed_values = [&](uint8_t* to) {
#pragma unroll
    for (int i = 0; i < R::WORDS; ++i) write_value(values, i, to);
  };

  // Keys run one tile ahead of the values: while tile j is weighed, S of tile j + 1 is
  // computed, keys of j + 2 and values of j + 1 are unpacked, and those of j + 3 and j + 2
  // are on their way.  After the wave's last tile S is computed from whatever LDS
  // holds, and not used.
  f32x16_t Sa[2], Sb[2];
  float top = 0.f;
  int page = 0, page_before = 0;  // of the keys' and the values' next loads
  if (first < last) {
    const int page0 = page_of(first), page1 = page_of(first + 1);
    page_before = page_of(first + 2);
    page = page_of(first + 3);
    RawKeys<D, WAVES> second;
    load_keys(keys, first, page0);
    load_values(values, first, page0);
    load_keys(second, first + 1, page1);
    settle_raw(keys, values);
    feed_keys(s_k[0]);
    feed_values(s_v[0]);
    load_values(values, first + 1, page1);
    load_keys(keys, first + 2, page_before);
    settle_keys(second);
    for_keys(second, s_k[1]);
    __syncthreads();
    if (first < my_last) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        Sa[b] = (f32x16_t)(0.f);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) Sa[b] = mfma32x32x16(read_key(s_k[0], b, s), qf[s], Sa[b]);
      }
      settle(Sa, largest(Sa), first);
    }
  }
  auto turn = [&](f32x16_t (&S)[2], f32x16_t (&N)[2], int j, int at) {  // at: j - first is odd
    __syncthreads();
    auto refill = [&]() {
      load_values(values, j + 2, page_before);
      load_keys(keys, j + 3, page);
      page_before = page;
      page = page_of(j + 4);
    };
    if (j < my_last) {
      step(S, N, s_k[at ^ 1], s_v[at], s_k[at], s_v[at ^ 1], top, refill);
    } else {
      settle_raw(keys, values);
      feed_keys(s_k[at]);
      feed_values(s_v[at ^ 1]);
      if constexpr (EARLY) refill();
    }
    if constexpr (!EARLY) refill();
    if (j + 1 < my_last) settle(N, top, j + 1);
  };
  for (int j = first; j < last; j += 2) {
    turn(Sa, Sb, j, 0);
    if (j + 1 >= last) break;
    turn(Sb, Sa, j + 1, 1);
  }
  if (live) {
    sum += __shfl_xor(sum, 32, 64);
    if (sq.bad) sum = __builtin_nanf("");
    const bool mine = row0 + n < rows;
    if (!whole) {
      const int r = wave * 32 + n;
      float* slot = p.partial + (int64_t)place * p.slot;
      if (mine) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<f32x4_t*>(slot + r * D + 32 * m + 2 * e + 4 * half) =
                f32x4_t{O[m][e], O[m][e + 1], O[m][e + 2], O[m][e + 3]};
        if (half == 0) {
          slot[32 * WAVES * D + r] = M;
          slot[32 * WAVES * (D + 1) + r] = sum;
        }
      }
    } else {
      // a row that sees no token gives zeros
      const float inv = seen >= 0 || sum != sum ? 1.f / sum : 0.f;
      uint16_t* o = p.out + (((int64_t)sq.row0 + token) * p.heads + head) * D + 4 * half;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          if (mine)
            *reinterpret_cast<u32x2_t*>(o + 32 * m + 2 * e) =
                u32x2_t{result_pair<BF>(O[m][e] * inv, O[m][e + 1] * inv),
                        result_pair<BF>(O[m][e + 2] * inv, O[m][e + 3] * inv)};
    }
  }
  x += part;
  if constexpr (PIECES)
    if (x < end) {
      mine_of_lane = chunk_sequence(p.batch, lane - 1);  // again, and not kept through the products
      __syncthreads();                                   // the tiles in LDS have been read
    }
  }
}

// Joins the parts of units that were split or cut, 1024 results at a time, 4 per thread; those of
// a unit that was cut by the first end of a block's piece inside of it.  How many there are
// only the device knows, so that few blocks are launched, which take them in turn.
constexpr int kJoinBlocks = 2048;
template <bool BF, int D, bool PIECES>
__global__ __launch_bounds__(256) void chunk_join_kernel(const ChunkParams p) {
  constexpr int ROWS = 1024 / D;
  const int block_rows = p.batch.block_rows, parts = block_rows / ROWS, per = p.batch.per;
  const int lane = threadIdx.x & 63, c = threadIdx.x % (D / 4) * 4;
  ChunkSequence mine_of_lane;
  Line line;
  if constexpr (PIECES) {
    mine_of_lane = chunk_sequence(p.batch, lane - 1);
    line = line_of(p.batch, mine_of_lane, lane);
    if (!line.pieces) return;
  }
  for (int id = blockIdx.x;; id += kJoinBlocks) {
    ChunkSequence sq;
    int block, kvh, runs, place;
    bool second = false;  // the first part is the second one of its block
    if constexpr (PIECES) {
      const int cut = id / parts + 1;  // the end of block cut - 1
      if ((int64_t)cut * line.width >= line.total) return;
      Piece share;
      if (!find_piece(p.batch, line, mine_of_lane, cut * line.width, lane, share)) return;
      if (share.at == 0 || share.at > line.width) continue;
      sq = share.q;
      block = share.block;
      kvh = share.head;
      runs = (share.length - share.at + line.width - 1) / line.width + 1;
      place = 2 * (cut - 1);
      second = share.at < line.width;
      if (place + 2 * (runs - 1) >= p.batch.pieces) continue;  // offsets that are not ascending
    } else {
      ChunkShare share;
      if (!find_chunk(p.batch, id / parts, true, lane, share)) return;
      sq = share.q;
      block = share.block;
      kvh = share.head;
      runs = share.runs;
      place = (int)share.slot;
    }
    const int r = id % parts * ROWS + threadIdx.x / (D / 4);
    const int row = block * block_rows + r;
    if (row >= sq.rows * per) continue;
    const int token = quotient(row, per, p.batch.per_shift), head = kvh * per + row - token * per;
    auto slot_of = [&](int i) {
      return p.partial + (int64_t)(place + (PIECES ? 2 * i + (i == 0 && second ? 1 : 0) : i)) * p.slot;
    };
    float M = kLow, sum = 0.f;
    for (int i = 0; i < runs; ++i) M = fmaxf(M, slot_of(i)[block_rows * D + r]);
    f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < runs; ++i) {
      const float* slot = slot_of(i);
      const float f = __builtin_amdgcn_exp2f(slot[block_rows * D + r] - M);
      sum = fmaf(f, slot[block_rows * (D + 1) + r], sum);
      const f32x4_t v = *reinterpret_cast<const f32x4_t*>(slot + r * D + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(f, v[e], o[e]);
    }
    const bool sees = token + sq.length - sq.rows >= 0;
    const float inv = sees || sum != sum ? 1.f / sum : 0.f;
    *reinterpret_cast<u32x2_t*>(p.out + (((int64_t)sq.row0 + token) * p.heads + head) * D + c) =
        u32x2_t{result_pair<BF>(o[0] * inv, o[1] * inv), result_pair<BF>(o[2] * inv, o[3] * inv)};
  }
}

}  // namespace

// The single-token kernel unpacks a token once for 16 rows, the tile kernel for 256
// (128), whether it has them or not, and takes longer to start.  Which is the faster by
// the rows of a sequence and the tiles that all have (32 query and 8 key/value heads, us;
// 16 seqs of 2000, 32 rows: 17, 46; 1 of 32768, 64: 34, 53; 32 of 2000, 64: 44, 61,
// 128: 78, 66; 8 of 2000, 128: 27, 40; 1 of 2000, 256: 17, 34; 32 of 2000, 256: 150, 98).
// How many rows each sequence has is known on the device only: a batch with few on
// average goes to the first as a whole (any number is right in either kernel), one
// sequence with more to the second, and several with more on average to both, each
// kernel taking its own.  Those times are of sequences with equally many rows.  A long chunk
// among many single rows stays below the average and with the first kernel: 63 rows of
// sequences of 2000 tokens and 900 rows behind 1100 take 83 us (88 as two calls), 127 and 1900
// behind 2100 256 (190), 255 and 3800 behind 4200 817 (516).
ChunkPlan plan_chunk(int64_t tokens, int64_t seqs, int heads, int kv_heads, int head_size, int64_t capacity) {
  constexpr int kRows = 16;  // of the single-token kernel's blocks
  const int64_t per = heads / kv_heads, rows = tokens * per, all = seqs * kv_heads * ((capacity + kKeys - 1) / kKeys);
  ChunkPlan plan = {};
  plan.few_rows = all <= 512 ? 256 : all <= 2048 ? 128 : 64;
  const bool few = rows <= plan.few_rows * seqs, both = !few && seqs > 1 && per <= plan.few_rows;
  auto reserve = [&](ChunkPart& part, int64_t units, int pieces) {
    part.units = units;
    part.slot = (int64_t)part.block_rows * (head_size + 2);
    part.pieces = part.most == 1 ? 0 : pieces;
    if (part.most == 1) return;
    if (plan.workspace == 0) plan.workspace = kKv4Counters * sizeof(uint32_t);
    part.partial = plan.workspace;
    plan.workspace += ((size_t)pieces * part.slot * sizeof(float) + 255) / 256 * 256;
  };
  const int64_t most_tiles = (capacity + kKeys - 1) / kKeys;
  // a partial block for every sequence and for the rows in front of them and behind
  auto units_of = [&](int64_t block_rows) { return ((rows + block_rows - 1) / block_rows + seqs + 2) * kv_heads; };
  if (few || both) {
    const int64_t units = both ? seqs * kv_heads * (plan.few_rows / kRows) : units_of(kRows);
    // as many as there are if all sequences have equally many rows
    const Kv4Plan like = plan_kv4(seqs * kv_heads * (few ? (rows / seqs + kRows - 1) / kRows : 1), 1, 1, head_size,
                                  capacity);
    plan.few.waves = like.waves;
    plan.few.block_rows = kRows;
    plan.few.tile = 32;
    plan.few.blocks = like.blocks;
    // Of a few thousand tokens (8 sequences of 3000, 2 tokens each: 15.8 us with 16 steps, 18.0
    // with 32); short ones are not split (32 of 600: 11.5, 9.9 unsplit).
    plan.few.least = 16;
    const int64_t longest = (capacity + 31) / 32 / plan.few.least;
    plan.few.most = units > kKv4Counters || longest < 2 ? 1 : longest < 256 ? (int)longest : 256;
    const int64_t more = units * (plan.few.most - 1);
    plan.few.grid = units + (more < plan.few.blocks ? more : plan.few.blocks);
    reserve(plan.few, units, plan.few.blocks);
  }
  if (!few) {
    plan.tiles.waves = head_size > 128 ? 4 : 8;
    plan.tiles.block_rows = 32 * plan.tiles.waves;
    plan.tiles.tile = kKeys;
    plan.tiles.blocks = 256;
    plan.tiles.least = 8;
    const int64_t units = units_of(plan.tiles.block_rows);
    // four rounds of blocks are even enough by themselves
    const bool cut = units < 4 * plan.tiles.blocks && most_tiles > plan.tiles.least && units * most_tiles < 1 << 26;
    // equal pieces where a block has some 48 tiles: finding them takes 10 us
    const int64_t tiles = (rows + plan.tiles.block_rows - 1) / plan.tiles.block_rows * kv_heads * most_tiles;
    const bool pieces = cut && tiles >= 48 * plan.tiles.blocks;
    const int64_t longest = most_tiles / plan.tiles.least;
    plan.tiles.most = !cut || longest < 2 ? 1 : longest < 64 ? (int)longest : 64;
    const int64_t more = plan.tiles.most == 1 ? 0 : plan.tiles.blocks;
    plan.tiles.grid = pieces ? (units > plan.tiles.blocks ? units : plan.tiles.blocks) : units + more;
    reserve(plan.tiles, units, (pieces ? 2 : 1) * plan.tiles.blocks);
    if (!pieces) plan.tiles.pieces = 0;
  }
  return plan;
}

int launch_chunk_attention(const ChunkParams& p, int dtype, hipStream_t st) {
  const bool split = p.batch.most > 1;
  if (p.grid > INT32_MAX) return GRINQH_ERR_INVALID;
  auto go = [&](auto bf, auto d) -> int {
    constexpr bool BF = decltype(bf)::value;
    constexpr int D = decltype(d)::value, WAVES = D > 128 ? 4 : 8;
    const bool pieces = p.batch.pieces > 0;
    auto kernel = pieces ? chunk_attention_kernel<BF, D, WAVES, true> : chunk_attention_kernel<BF, D, WAVES, false>;
    auto join = pieces ? chunk_join_kernel<BF, D, true> : chunk_join_kernel<BF, D, false>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)p.grid), dim3(64 * WAVES), 0, st, p);
    if (split) hipLaunchKernelGGL(join, dim3(kJoinBlocks), dim3(256), 0, st, p);
    return hipGetLastError() == hipSuccess ? GRINQH_OK : GRINQH_ERR_HIP;
  };
  auto sized = [&](auto bf) -> int {
    switch (p.cache.head_size) {
      case 64: return go(bf, std::integral_constant<int, 64>{});
      case 128: return go(bf, std::integral_constant<int, 128>{});
      case 256: return go(bf, std::integral_constant<int, 256>{});
    }
    return GRINQH_ERR_INVALID;
  };
  return dtype == GRINQH_DTYPE_BF16 ? sized(std::true_type{}) : sized(std::false_type{});
}

}  // namespace grinqh
