// A key/value cache held in 4 bits: filling it, reading it back, and the
// attention of one query token per sequence over it.
//
// Layout: uint8 [pages][heads][sub][record], a record being 16 tokens of one
// head (D channels, G = D / group groups for the keys, one for the values):
//
//   keys          [16 tokens][D / 8 words], word (chunk % 4) * (D / 32) + chunk / 4 of channel chunk = channel / 8
//   key params    [G][16 tokens] (scale, minimum) as two fp16
//   values        [D / 8 words][16 tokens], word = channel / 8
//   value params  [16 tokens] (scale, minimum)
//
// Channel c of a word's 8 is nibble c / 2 + 4 * (c % 2).  A code stands for
// minimum + scale * code; both parameters are rounded to fp16 first and the
// codes then chosen for the rounded ones, so the rounding costs no accuracy
// beyond that of the 4 bits.
//
// Why this layout: a lane of v_mfma_f32_16x16x32 holds 8 consecutive values
// of the summed axis for one row.  For q.k the axis is the channel, so a lane
// (token, quarter) reads the D / 32 words of its quarter as one load; for p.v it
// is the token, so a lane (channel chunk, quarter) reads 4 tokens' words as one
// 16-byte load.  Masking a word with 0x000F000F gives two codes as fp16
// subnormals c * 2^-24 (exact), with 0x00F000F0 two more as 16 c * 2^-24: 5 VALU
// operations unpack 8 key codes, 6 unpack 8 value codes, and nothing is rounded.
#include <cfloat>
#include <type_traits>

#include "attention_launch.h"
#include "chunk_share.h"
#include "grinqh_common.h"
#include "splitk_complete.h"
#include "wave_scan.h"

namespace grinqh {

namespace {

constexpr float kLimit = 65504.f;  // largest finite fp16

// one v_cvt_pk_f16_f32 (round to nearest even)
__device__ __forceinline__ uint32_t f16_pair(float lo, float hi) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{lo, hi}), f16x2_t));
}
__device__ __forceinline__ float half_lo(uint32_t w) { return f16_bits_to_f32((uint16_t)w); }
__device__ __forceinline__ float half_hi(uint32_t w) { return f16_bits_to_f32((uint16_t)(w >> 16)); }

// What is kept is within +-kLimit, but a scale that was rounded up makes the
// largest code stand for up to 65536, and weights round too: fp16 results are
// limited, as they would be infinite otherwise (bf16 holds 65536).  NaN stays.
template <typename DT>
__device__ __forceinline__ uint16_t limited(float v) {
  if constexpr (DT::id == F16::id)
    v = __builtin_elementwise_maximum(__builtin_elementwise_minimum(v, kLimit), -kLimit);
  return from_f32<DT>(v);
}

// ---------------------------------------------------------------- store, load

// The value of the lane that DPP control `CTRL` names.
template <int CTRL>
__device__ __forceinline__ float lane_value(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// op over WIDTH adjacent lanes, in all of them: neighbours within 4 by quad
// permutes, then the mirrored half of 8 and of 16 (any lane of the other half
// will do), then the other 16 of 32.
template <int WIDTH, typename F>
__device__ __forceinline__ float group_reduce(float v, F&& op) {
  v = op(v, lane_value<0xB1>(v));
  v = op(v, lane_value<0x4E>(v));
  if constexpr (WIDTH >= 8) v = op(v, lane_value<0x141>(v));
  if constexpr (WIDTH >= 16) v = op(v, lane_value<0x140>(v));
  if constexpr (WIDTH >= 32) v = op(v, __shfl_xor(v, 16, 64));
  return v;
}

// Codes and (scale, minimum) of one lane's 8 channels; the WIDTH adjacent lanes
// of a group share the parameters.  A NaN becomes +inf in the maximum, which
// the limit keeps finite inputs from, and makes the group's parameters NaN.
// Channels past the limit need no limiting of their own: their codes do it.
// Storing 8192 tokens of 8 heads of 128 channels takes 12.0 us (43 MB, 3.6 TB/s; the
// copy rate would be 9): a lane waits for its slot before its rows leave, and of
// its 399 VALU operations some 130 divide the slot's record by a page's (64 bits,
// record_of).  Loading them takes 9.5 (4.6 TB/s).
template <typename DT, int WIDTH>
__device__ __forceinline__ uint32_t quantize8(const u32x4_t& in, uint32_t& params) {
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = to_f32<DT>((uint16_t)(in[e >> 1] >> (16 * (e & 1))));
  float mn = x[0], mx = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    mn = fminf(mn, x[e]);
    mx = __builtin_elementwise_maximum(mx, x[e]);  // NaN if one is
  }
  mn = fmaxf(mn, -kLimit);
  mx = mx != mx ? __builtin_inff() : fminf(mx, kLimit);
  mn = group_reduce<WIDTH>(mn, [](float a, float b) { return fminf(a, b); });
  mx = group_reduce<WIDTH>(mx, [](float a, float b) { return fmaxf(a, b); });
  if (mx > kLimit) {
    params = 0x7E007E00u;  // NaN, NaN
    return 0;
  }
  mn = fminf(mn, kLimit);   // where every channel is past the limit
  mx = fmaxf(mx, -kLimit);
  const uint16_t mh = f32_to_f16_bits(mn + 0.f);  // zeros are kept as +0, whichever zero came first
  const float m = f16_bits_to_f32(mh);
  const uint16_t sh = f32_to_f16_bits((mx - m) * (1.f / 15.f) + 0.f);
  const float s = f16_bits_to_f32(sh);
  const float inv = s > 0.f ? 1.f / s : 0.f;
  params = (uint32_t)sh | ((uint32_t)mh << 16);
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float c = fminf(fmaxf(rintf((x[e] - m) * inv), 0.f), 15.f);
    w |= (uint32_t)c << (4 * (e / 2 + 4 * (e % 2)));
  }
  return w;
}

// Where a slot's token lives: its record of `head`, or nullptr outside the cache.
__device__ __forceinline__ uint8_t* record_of(const Kv4Cache& c, int64_t slot, int head, int record) {
  const int64_t rec = slot >> 4, page = rec / c.sub;  // sub is a power of two
  if (slot < 0 || page >= c.pages) return nullptr;
  return c.p + ((page * c.heads + head) * c.sub + (rec & (c.sub - 1))) * record;
}

// One lane per 8 channels of a (token, head), keys and values alike.
template <typename DT, int D, int G>
__global__ __launch_bounds__(256) void kv4_store_kernel(HeadRows k, HeadRows v, const int64_t* __restrict__ slots,
                                                        int64_t tokens, Kv4Cache cache) {
  constexpr int LANES = D / 8, ROWS = 256 / LANES, R = kv4_record_bytes(D, G);
  const int n = threadIdx.x % LANES;
  const int head = blockIdx.x % cache.heads;
  const int64_t t = (int64_t)(blockIdx.x / cache.heads) * ROWS + threadIdx.x / LANES;
  const int64_t row = t < tokens ? t : tokens - 1;
  uint8_t* rec = t < tokens ? record_of(cache, slots[t], head, R) : nullptr;
  const int tok = rec != nullptr ? (int)(slots[t] & 15) : 0;
  const u32x4_t kx = *reinterpret_cast<const u32x4_t*>(k.p + row * k.token + head * k.head + 8 * n);
  const u32x4_t vx = *reinterpret_cast<const u32x4_t*>(v.p + row * v.token + head * v.head + 8 * n);
  uint32_t kp, vp;
  const uint32_t kw = quantize8<DT, LANES / G>(kx, kp);
  const uint32_t vw = quantize8<DT, LANES>(vx, vp);
  if (rec == nullptr) return;
  uint32_t* w = reinterpret_cast<uint32_t*>(rec);
  w[tok * LANES + (n & 3) * (D / 32) + (n >> 2)] = kw;
  if (n % (LANES / G) == 0) w[2 * D + (n / (LANES / G)) * 16 + tok] = kp;
  w[2 * D + 16 * G + n * 16 + tok] = vw;
  if (n == 0) w[4 * D + 16 * G + tok] = vp;
}

template <typename DT>
__device__ __forceinline__ u32x4_t dequantize8(uint32_t w, uint32_t params) {
  const float s = half_lo(params), m = half_hi(params);
  u32x4_t out;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const float a = fmaf(s, (float)((w >> (4 * p)) & 15u), m);
    const float b = fmaf(s, (float)((w >> (4 * p + 16)) & 15u), m);
    out[p] = (uint32_t)limited<DT>(a) | ((uint32_t)limited<DT>(b) << 16);
  }
  return out;
}

template <typename DT, int D, int G>
__global__ __launch_bounds__(256) void kv4_load_kernel(Kv4Cache cache, const int64_t* __restrict__ slots,
                                                       int64_t tokens, uint16_t* __restrict__ k,
                                                       uint16_t* __restrict__ v) {
  constexpr int LANES = D / 8, ROWS = 256 / LANES, R = kv4_record_bytes(D, G);
  const int n = threadIdx.x % LANES;
  const int head = blockIdx.x % cache.heads;
  const int64_t t = (int64_t)(blockIdx.x / cache.heads) * ROWS + threadIdx.x / LANES;
  if (t >= tokens) return;
  const uint8_t* rec = record_of(cache, slots[t], head, R);
  u32x4_t kx = u32x4_t{0u, 0u, 0u, 0u}, vx = kx;
  if (rec != nullptr) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(rec);
    const int tok = (int)(slots[t] & 15);
    kx = dequantize8<DT>(w[tok * LANES + (n & 3) * (D / 32) + (n >> 2)], w[2 * D + (n / (LANES / G)) * 16 + tok]);
    vx = dequantize8<DT>(w[2 * D + 16 * G + n * 16 + tok], w[4 * D + 16 * G + tok]);
  }
  const int64_t at = (t * cache.heads + head) * D + 8 * n;
  *reinterpret_cast<u32x4_t*>(k + at) = kx;
  *reinterpret_cast<u32x4_t*>(v + at) = vx;
}

// ---------------------------------------------------------------- attention, one token per sequence

constexpr int kRows = 16;       // query heads of one key/value head per block
constexpr int kGroup = 16;     // sequences a lane looks at: plans cover 64 of these
constexpr int kRuns = 256;      // most blocks that share one sequence and head
constexpr float kLow = -FLT_MAX;  // running reference before the first token (finite: -inf - -inf would be NaN)

// Which run of 32-token steps a block takes.
struct Share {
  int seq, unit;         // unit: key/value head and tile of its query heads
  int first, last;       // steps
  int run, runs;         // this is run `run` of the unit's
  int length;            // of the sequence, in tokens
  bool bad;              // it is longer than the page table
};

__device__ __forceinline__ int length_of(const Kv4Params& p, int seq, bool& bad) {
  const int64_t capacity = (int64_t)p.table_width << (p.sub_shift + 4);
  const int length = max(p.lengths[seq], 0);
  bad = length > capacity;
  return bad ? (int)capacity : length;
}
// Every block plans by itself from the lengths, which only the device knows:
// the steps of all sequences and heads shared out over plan.blocks, in runs of
// at least plan.least steps that never leave their sequence, all runs of a
// sequence alike.  A lane looks at seqs / 64 sequences (at most kGroup: with more
// there are blocks enough, and a plan would take longer), a scan over the lanes
// finds the block's.  Where no sequence can be shared (plan.most == 1) a block
// is a unit.  False: more blocks than runs.
__device__ __forceinline__ bool find_share(const Kv4Params& p, int id, int lane, Share& s) {
  if (p.plan.most == 1) {
    s.seq = id / p.units;
    s.unit = id - s.seq * p.units;
    s.length = length_of(p, s.seq, s.bad);
    s.run = s.first = 0;
    s.runs = 1;
    s.last = (s.length + 31) >> 5;
    return true;
  }
  const int group = (p.seqs + 63) >> 6, s0 = lane * group;
  int mine[kGroup];  // lengths of the lane's sequences
  bool bad = false;
  mine[0] = s0 < p.seqs ? length_of(p, s0, bad) : 0;
#pragma unroll
  for (int i = 1; i < kGroup; ++i) {
    bool b;
    mine[i] = group > 1 && i < group && s0 + i < p.seqs ? length_of(p, s0 + i, b) : 0;
  }
  float steps = 0.f;
#pragma unroll
  for (int i = 0; i < kGroup; ++i) steps += (float)((mine[i] + 31) >> 5);
  const float total = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_scan(steps)), 63));
  const int chunk = max(p.plan.least, (int)ceilf(fminf(total * (float)p.units / (float)p.plan.blocks, 0x1p26f)));
  auto runs_of = [&](int length) { return min(max((((length + 31) >> 5) + chunk - 1) / chunk, 1), p.plan.most); };
  int runs = 0;
#pragma unroll
  for (int i = 0; i < kGroup; ++i)
    if (i < group && s0 + i < p.seqs) runs += runs_of(mine[i]) * p.units;
  const int upto = wave_scan(runs);
  const uint64_t after = __ballot(upto > id);
  if (after == 0) return false;
  const int owner = __builtin_ctzll(after);
  int rest = id - __builtin_amdgcn_readlane(upto - runs, owner);
  int seq = owner * group, k = 0;
  s.length = 0;
#pragma unroll
  for (int i = 0; i < kGroup; ++i) {
    if (i >= group || k > 0) break;
    s.length = __builtin_amdgcn_readlane(mine[i], owner);
    const int r = runs_of(s.length);
    if (rest < r * p.units) {
      k = r;
    } else {
      rest -= r * p.units;
      ++seq;
    }
  }
  s.bad = group == 1 ? (__ballot(bad) >> owner) & 1 : p.lengths[seq] > s.length;  // limited, hence past the table
  const int n = (s.length + 31) >> 5, per = (n + k - 1) / k;
  s.seq = seq;
  s.runs = k;
  s.unit = rest / k;
  s.run = rest - s.unit * k;
  s.first = s.run * per;
  s.last = min(s.first + per, n);
  return true;
}

// What a lane holds of 32 tokens (two records).  The parameters are loaded once
// per wave, a word or a few per lane, and handed round through LDS when they
// are used: a lane needs those of 8 tokens, 8 (G + 1) words, and the prefetch
// would have no registers for them.
template <int D, int G>
struct Tokens {
  static constexpr int kParams = 32 * (G + 1);  // words
  uint32_t k[2][D / 32];
  u32x4_t v[2][D < 128 ? 1 : D / 128];
  uint32_t par[(kParams + 63) / 64];
};

template <int D, int G>
__device__ __forceinline__ void load_tokens(Tokens<D, G>& t, const uint8_t* __restrict__ rec0,
                                            const uint8_t* __restrict__ rec1, int lane) {
  const int n = lane & 15, quad = lane >> 4;
  constexpr int W = D / 32, PER = 16 * (G + 1);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint8_t* rec = r == 0 ? rec0 : rec1;
    const uint8_t* kb = rec + (uint32_t)(n * (D / 2) + quad * (D / 8));
    if constexpr (W == 2) {
      const u32x2_t x = *reinterpret_cast<const u32x2_t*>(kb);
      t.k[r][0] = x[0];
      t.k[r][1] = x[1];
    } else {
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const u32x4_t x = *reinterpret_cast<const u32x4_t*>(kb + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) t.k[r][i + j] = x[j];
      }
    }
    const uint8_t* vb = rec + (uint32_t)(8 * D + 64 * G + (D < 128 ? n & 7 : n) * 64 + 16 * quad);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(t.v[r]) / 16); ++i) t.v[r][i] = *reinterpret_cast<const u32x4_t*>(vb + 1024 * i);
  }
#pragma unroll
  for (int j = 0; j < (int)(sizeof(t.par) / 4); ++j) {
    const int i = min(lane + 64 * j, 2 * PER - 1), w = i < PER ? i : i - PER;
    const uint32_t at = w < 16 * G ? 8 * D + 4 * w : 16 * D + 4 * w;
    t.par[j] = *reinterpret_cast<const uint32_t*>((i < PER ? rec0 : rec1) + at);
  }
}

// Block = one sequence, one key/value head (up to 16 of its query heads) and
// one run of tokens; its waves take 32-token steps in turn, each with a softmax
// of its own, joined at the end.  Where a sequence is shared by several blocks,
// each leaves its result in the workspace and the one that arrives last joins
// them, in their order.
//
// Bound by HBM for long contexts: 64 sequences of 8192 tokens, 32 query and 8
// key/value heads of 128 (570 MB) take 103 us, 5.5 TB/s; a kernel that only reads
// the same pages takes 95, the difference is the blocks' start and end.  One
// sequence of 131072 tokens: 37 us (147 MB, 4.0 TB/s with planning and joining).
// Short ones are latency: lengths, pages, tokens, one after the other, 8-11 us.
// Past 1024 sequences nothing is shared (find_share): one of 32768 tokens among short
// ones, 2 heads, takes 55 us in a batch of 1024 and 206 in one of 1025.
//
// S^T = K Q^T leaves a lane with one query row and 8 of the 32 tokens, which
// is the B operand of O^T = V^T P^T: nothing crosses lanes in the loop.  With
// value = m + s c:  o = sum_t (p_t s_t) c_t + sum_t p_t m_t, so P carries the
// value scale and the minimum is one sum per row.
//
// The exponent's reference M is raised only when a weight p s passes 2^8
// (checked for all lanes at once; as a branch apart from the weights, or the
// compiler keeps the accumulators twice), so the accumulators are rarely rescaled;
// M includes the value scale, which keeps the fp16 weights in range whatever
// the values' size.  Queries are brought to 2^13 <= max < 2^14 by a power of two
// (exact), so fp16 holds them for both types and the nibbles that come out
// 16-fold can be undone on the query's side.
//
// With a batch of chunks (B is ChunkBatch) a block's rows are up to 16 (token, query
// head) pairs of a sequence, each of which sees one token more per token of the chunk.
struct OneRow {  // one token per sequence
  static constexpr int per_shift = 0;
};
template <typename DT, int D, int G, int WAVES, typename B>
__global__ __launch_bounds__(64 * WAVES, D > 128 ? 2 : 3) void kv4_attention_kernel(const Kv4Params p, const B batch) {
  constexpr bool CHUNK = std::is_same_v<B, ChunkBatch>;
  constexpr int kWaves = WAVES, kThreads = 64 * WAVES;
  constexpr int R = kv4_record_bytes(D, G), W = D / 32, M_TILES = D < 128 ? 1 : D / 128, ACCS = D < 128 ? 4 : 8;
  __shared__ union {
    float o[kWaves][kRows][D + 4];
    struct {
      float weight[kRows][kRuns];
      f32x4_t sum[kThreads];
    } join;
  } sh;
  __shared__ float s_m[kWaves][kRows], s_l[kWaves][kRows], s_off[kWaves][kRows];
  __shared__ __align__(16) uint32_t s_par[kWaves][Tokens<D, G>::kParams];
  __shared__ int s_last;
  const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = p.heads / p.cache.heads;
  int seq, first, last, run, runs, unit, length, kvh, rows;
  bool bad;
  int limit, seen;        // tokens that the block's first row and the lane's row see (negative: none)
  int row0 = 0, shift = 0;  // chunks: first of the sequence's rows, tokens in front of it
  int64_t place = blockIdx.x;  // of this run's result in the workspace
  int64_t q_at, out_row;  // the lane's query, the block's first result
  if constexpr (CHUNK) {
    ChunkShare share;
    if (!find_chunk(batch, blockIdx.x, false, lane, share)) return;
    // offsets that are not ascending: runs that no block takes would be waited for
    if (share.runs > 1 && (int64_t)blockIdx.x - share.run + share.runs > gridDim.x) return;
    const int all = share.q.rows * per;
    row0 = share.block * kRows;
    rows = min(kRows, all - row0);
    seq = share.seq;
    kvh = share.head;
    run = share.run;
    runs = share.runs;
    unit = (int)share.unit;
    place = share.slot + share.run;
    length = share.q.length;
    bad = share.q.bad;
    shift = length - share.q.rows;
    const int row = row0 + min(n, rows - 1), token = quotient(row, per, batch.per_shift);
    limit = __builtin_amdgcn_readfirstlane(token) + shift + 1;
    seen = token + shift + 1;
    const int steps = max(__builtin_amdgcn_readlane(token, 15) + shift + 1 + 31, 0) >> 5;
    const int part = runs == 1 ? steps : (steps + runs - 1) / runs;
    first = min(run * part, steps);
    last = min(first + part, steps);
    q_at = (int64_t)(share.q.row0 + token) * p.q.token + (int64_t)(kvh * per + row - token * per) * p.q.head;
    out_row = (int64_t)share.q.row0 * p.heads + kvh * per;
  } else {
    Share share;
    if (!find_share(p, blockIdx.x, lane, share)) return;
    const int tiles = p.units / p.cache.heads;
    kvh = share.unit / tiles;
    const int tile = share.unit - kvh * tiles, h0 = kvh * per + tile * kRows;
    rows = min(kRows, per - tile * kRows);
    seq = share.seq;
    first = share.first;
    last = share.last;
    run = share.run;
    runs = share.runs;
    unit = seq * p.units + share.unit;
    length = limit = seen = share.length;
    bad = share.bad;
    q_at = (int64_t)seq * p.q.token + (int64_t)(h0 + min(n, rows - 1)) * p.q.head;
    out_row = (int64_t)seq * p.heads + h0;
  }
  // where a row's results go, and whether it sees any token
  auto result_row = [&](int row) -> int64_t {
    if constexpr (!CHUNK) return out_row + row;
    const int token = quotient(row0 + row, per, batch.per_shift);
    return out_row + (int64_t)token * p.heads + (row0 + row - token * per);
  };
  auto sees = [&](int row) {
    if constexpr (CHUNK) return quotient(row0 + row, per, batch.per_shift) + shift >= 0;
    return length > 0;
  };

  u32x4_t qf[W];
  {
    const uint16_t* q = p.q.p + q_at + 8 * quad;
#pragma unroll
    for (int s = 0; s < W; ++s) qf[s] = *reinterpret_cast<const u32x4_t*>(q + 32 * s);
  }
  // Two slots of tokens: one is computed while the other's loads are in flight
  // (8 waves per CU then have 35 KB on their way; a third slot gave nothing).
  constexpr int SLOTS = 2;
  const int32_t* table = p.table + (int64_t)seq * p.table_stride + (int64_t)kvh * p.table_head;
  const int last_rec = max((length - 1) >> 4, 0);
  auto record = [&](int step, int r, int page) -> const uint8_t* {
    if ((uint32_t)page >= (uint64_t)p.cache.pages) {
      bad = true;
      page = 0;
    }
    const int rec = min(2 * step + r, last_rec);
    return p.cache.p + ((((int64_t)page * p.cache.heads + kvh) << p.sub_shift) + (rec & (p.cache.sub - 1))) * R;
  };
  Tokens<D, G> slots[SLOTS];
  const int begin = first + wave;
  // Pages: a lane holds one of the next 64 records', loaded once for ROUND steps
  // (a load per step would sit behind the tokens' loads, and waiting for it would
  // be waiting for them).  Past the end a step stands for the last one: a load
  // under a condition would make every wait a wait for all loads.
  constexpr int ROUND = 27 / SLOTS * SLOTS;  // ROUND + SLOTS <= 32
  auto pages_from = [&](int step) {
    const int at = min(step + (lane >> 1) * kWaves, last - 1);
    return table[min(2 * at + (lane & 1), last_rec) >> p.sub_shift];
  };
  int pages = 0;
  auto fetch = [&](Tokens<D, G>& t, int step, int place) {
    const int at = min(step, last - 1);
    load_tokens<D, G>(t, record(at, 0, __builtin_amdgcn_readlane(pages, 2 * place)),
                      record(at, 1, __builtin_amdgcn_readlane(pages, 2 * place + 1)), lane);
  };
  if (begin < last) {
    pages = pages_from(begin);
    asm volatile("" : "+v"(pages));
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) fetch(slots[i], begin + i * kWaves, i);
  }

  float qsum[G], qs;
  {
    float x[W][8];
    float mx = 0.f;
#pragma unroll
    for (int s = 0; s < W; ++s) {
      const u32x4_t in = qf[s];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[s][e] = n < rows ? to_f32<DT>((uint16_t)(in[e >> 1] >> (16 * (e & 1)))) : 0.f;
        mx = fmaxf(mx, fabsf(x[s][e]));
      }
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    int ex = 0;
    if (mx > 0.f && mx < __builtin_inff()) ex = min(13 - ilogbf(mx), 100);
#pragma unroll
    for (int g = 0; g < G; ++g) qsum[g] = 0.f;
#pragma unroll
    for (int s = 0; s < W; ++s) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[s][e] = ldexpf(x[s][e], ex);
        qsum[s * G / W] += x[s][e];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = (i & 1) ? 0.0625f : 1.f;  // odd nibbles come out 16-fold
        qf[s][i] = f16_pair(x[s][2 * i] * f, x[s][2 * i + 1] * f);
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      qsum[g] += __shfl_xor(qsum[g], 16, 64);
      qsum[g] += __shfl_xor(qsum[g], 32, 64);
      qsum[g] *= 0x1p-24f;  // the codes' unit
    }
    // logits in powers of two; never 0 or infinite, which times an infinite or a zero
    // logit (a token past the end, a key of zeros) would be NaN
    qs = fminf(fmaxf(ldexpf(p.scale * 1.44269504088896f, 24 - ex), FLT_MIN), FLT_MAX);
  }

  f32x4_t O[M_TILES][ACCS];
#pragma unroll
  for (int i = 0; i < M_TILES; ++i)
#pragma unroll
    for (int j = 0; j < ACCS; ++j) O[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float M = kLow, L = 0.f, off = 0.f;
  float zs = qs;  // unit of the logits z
  bool far = false;

  auto compute = [&](const Tokens<D, G>& t, int step) {
#pragma unroll
    for (int j = 0; j < (int)(sizeof(t.par) / 4); ++j)
      if (64 * j + 64 <= Tokens<D, G>::kParams || lane < Tokens<D, G>::kParams - 64 * j)
        s_par[wave][64 * j + lane] = t.par[j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // other lanes of this wave read them
    float z[8];
    u32x4_t vp[2];  // (scale, minimum) of the values
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t* par = &s_par[wave][r * 16 * (G + 1) + 4 * quad];
      vp[r] = *reinterpret_cast<const u32x4_t*>(par + 16 * G);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const u32x4_t kp = *reinterpret_cast<const u32x4_t*>(par + 16 * g);
        f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = g * (W / G); s < (g + 1) * (W / G); ++s) {
          const uint32_t w = t.k[r][s], u = w >> 8;
          const u32x4_t a = u32x4_t{w & 0x000F000Fu, w & 0x00F000F0u, u & 0x000F000Fu, u & 0x00F000F0u};
          acc = mfma16x16x32<F16>(a, qf[s], acc);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          z[4 * r + i] = fmaf(acc[i], half_lo(kp[i]), fmaf(half_hi(kp[i]), qsum[g], g == 0 ? 0.f : z[4 * r + i]));
      }
    }
    if (32 * step + 32 > limit) {  // tokens past the end: whatever the record holds must not count
      asm volatile("");  // a branch: as selects, this is a sixth of every step's instructions
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (32 * step + 16 * (e >> 2) + 4 * quad + (e & 3) >= seen) {
          z[e] = -__builtin_inff();
          vp[e >> 2][e & 3] = 0;
        }
    }
    __builtin_amdgcn_sched_barrier(0);  // keys, weights, values: unpacking ahead would not fit the registers
    float pe[8], pw[8];
    // z qs is exact in here and M is not: the same factor for all tokens of a row, but
    // of more than 2^16 for logits past 2^28.  With `far` the product is rounded first.
    auto product_first = [&]() {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        z[e] *= qs;
        asm volatile("" : "+v"(z[e]));  // not contracted with the subtraction
      }
    };
    if (far) product_first();
    auto weights = [&]() {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pe[e] = __builtin_amdgcn_exp2f(fmaf(z[e], zs, -M));
        pw[e] = fmaf(pe[e], half_lo(vp[e >> 2][e & 3]), 0.f);  // + 0: one v_fma_mix_f32, no conversion
      }
    };
    weights();
    float top = 0.f, sum = 0.f;
    auto extent = [&]() {
      top = sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        top = fmaxf(top, pw[e]);
        sum += pe[e];
      }
    };
    extent();
    const bool raise = __any(top > 256.f || sum > 0x1p60f);
    float f = 1.f;
    if (raise) {
      float m;
      auto reach = [&]() {
        m = M;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          m = fmaxf(m, fmaf(z[e], zs, __log2f(fmaxf(half_lo(vp[e >> 2][e & 3]), 0x1p-24f))));
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
      };
      reach();
      if (!far && __any(fabsf(m) > 0x1p24f && m != kLow)) {
        far = true;
        zs = 1.f;
        product_first();
        reach();
      }
      f = __builtin_amdgcn_exp2f(M - m);
      M = m;
      L *= f;
      off *= f;
      weights();
      extent();
    }
    u32x4_t pf;
    L += sum;
#pragma unroll
    for (int e = 0; e < 8; ++e) off = fmaf(pe[e], half_hi(vp[e >> 2][e & 3]), off);
    // The weights' rounding to fp16 would be multiplied by codes of 7.5 on
    // average, where the values themselves are near zero: what it takes from the
    // codes' middle is added back (fp16 results 4.8e-4 -> 1.7e-4 off beside their own
    // rounding of 2.1e-4).
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pf[i] = f16_pair(pw[2 * i], pw[2 * i + 1]);
      off = fmaf(7.5f, fmaf(half_lo(pf[i]), -1.f, pw[2 * i]), off);
      off = fmaf(7.5f, fmaf(half_hi(pf[i]), -1.f, pw[2 * i + 1]), off);
    }

    if (raise) {  // apart from the above, where the compiler would keep the accumulators twice
#pragma unroll
      for (int i = 0; i < M_TILES; ++i)
#pragma unroll
        for (int j = 0; j < ACCS; ++j) O[i][j] *= f;
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int mt = 0; mt < M_TILES; ++mt) {
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e] = t.v[e >> 2][mt][e & 3];
        if constexpr (D < 128) w[e] >>= 4 * (n >> 3);  // lanes 8..15 take the odd nibbles
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        u32x4_t x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = perm(w[2 * i + 1], w[2 * i], 0x0C040C00u + (uint32_t)b * 0x00010001u);
        if constexpr (D < 128) {
          O[mt][b] = mfma16x16x32<F16>(x & 0x000F000Fu, pf, O[mt][b]);
        } else {
          O[mt][2 * b] = mfma16x16x32<F16>(x & 0x000F000Fu, pf, O[mt][2 * b]);
          O[mt][2 * b + 1] = mfma16x16x32<F16>(x & 0x00F000F0u, pf, O[mt][2 * b + 1]);
        }
      }
    }
  };
  for (int base = begin; base < last; base += ROUND * kWaves) {
    int pages_after = pages_from(base + ROUND * kWaves);
    for (int i = 0; i < ROUND; i += SLOTS) {
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
        const int step = base + (i + j) * kWaves;
        if (step < last) compute(slots[j], step);  // no loads in here
        fetch(slots[j], step + SLOTS * kWaves, i + j + SLOTS);
      }
      if (base + (i + SLOTS) * kWaves >= last) break;
    }
    asm volatile("" : "+v"(pages_after));  // waited for here, where it is the oldest load, and not in the loop above
    pages = pages_after;
  }

  L += __shfl_xor(L, 16, 64);
  L += __shfl_xor(L, 32, 64);
  off += __shfl_xor(off, 16, 64);
  off += __shfl_xor(off, 32, 64);
  if (bad) L = __builtin_nanf("");
  if (quad == 0) {
    s_m[wave][n] = M;
    s_l[wave][n] = L;
    s_off[wave][n] = off;
  }
#pragma unroll
  for (int mt = 0; mt < M_TILES; ++mt)
#pragma unroll
    for (int j = 0; j < ACCS; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int chunk = 16 * mt + 4 * quad + i;  // the A operand's row
        int channel;
        float unit = 0x1p24f;
        if constexpr (D < 128) {
          const int nib = 2 * j + (chunk >> 3);
          channel = 8 * (chunk & 7) + 2 * (nib & 3) + (nib >> 2);
        } else {
          channel = 8 * chunk + 2 * (j & 3) + (j >> 2);
          if (j & 1) unit = 0x1p20f;
        }
        sh.o[wave][n][channel] = O[mt][j][i] * unit;
      }
  __syncthreads();
  float* slot = p.partial + place * p.plan.slot;  // [rows][D], then m and l [kRows] each
  for (int at = threadIdx.x; at < rows * D; at += kThreads) {
    const int row = at / D, d = at % D;
    float m = s_m[0][row];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s_m[w][row]);
    float sum = 0.f, val = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(s_m[w][row] - m);
      sum = fmaf(f, s_l[w][row], sum);
      val = fmaf(f, sh.o[w][row][d] + s_off[w][row], val);
    }
    if (runs == 1) {
      p.out[result_row(row) * D + d] = limited<DT>(sees(row) || sum != sum ? val / sum : 0.f);
    } else {
      store_partial(slot + at, val);
      if (d == 0) {
        store_partial(slot + rows * D + row, m);
        store_partial(slot + rows * D + kRows + row, sum);
      }
    }
  }
  if (runs == 1) return;

  // as in splitk_complete: the stores have completed before the count says so
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(&p.counters[unit], 1u) == (unsigned)(runs - 1);
  __syncthreads();
  if (!s_last) return;
  // Threads share out the columns (4 adjacent ones each) and, where there are
  // more threads, the runs; the first loads leave before the weights are known.
  const int columns = rows * D / 4;
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      slot - (int64_t)run * p.plan.slot, (short)0, runs * p.plan.slot * 4, 0x00020000);
  constexpr int BATCH = 16;
  const int parts = max(kThreads / columns, 1), part = min((int)threadIdx.x / columns, parts);
  f32x4_t x[BATCH];
  auto load = [&](int column, int i0) {
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      x[u] = __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                             rs, (min(i0 + u * parts, runs - 1) * p.plan.slot + 4 * column) * 4, 0,
                                             kCpolSc1));
  };
  if (part < parts) load(threadIdx.x - part * columns, part);
  for (int row = wave; row < rows; row += kWaves) {
    float mi[kRuns / 64], li[kRuns / 64], m = kLow, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kRuns / 64; ++i) {
      const int run = lane + 64 * i, at = (run * p.plan.slot + rows * D + row) * 4;
      mi[i] = li[i] = 0.f;
      if (64 * i < runs) {  // past the last run: out of range, 0
        mi[i] = __uint_as_float((uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rs, at, 0, kCpolSc1));
        li[i] = __uint_as_float((uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rs, at, 4 * kRows, kCpolSc1));
      }
    }
#pragma unroll
    for (int i = 0; i < kRuns / 64; ++i) {
      if (lane + 64 * i >= runs) mi[i] = kLow;
      m = fmaxf(m, mi[i]);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
#pragma unroll
    for (int i = 0; i < kRuns / 64; ++i) {
      const float f = __builtin_amdgcn_exp2f(mi[i] - m);
      sum = fmaf(f, li[i], sum);
      if (lane + 64 * i < runs) sh.join.weight[row][lane + 64 * i] = f;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) s_l[0][row] = sum;
  }
  __syncthreads();
  for (int c0 = 0; c0 < columns; c0 += kThreads) {
    const int column = parts > 1 ? (int)threadIdx.x - part * columns : c0 + (int)threadIdx.x;
    const bool live = part < parts && column < columns;
    const int row = live ? column / (D / 4) : 0;
    f32x4_t val = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if (live) {
      if (c0 > 0) load(column, part);
      for (int i0 = part;;) {
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
          if (i0 + u * parts < runs) {
            const float f = sh.join.weight[row][i0 + u * parts];
#pragma unroll
            for (int e = 0; e < 4; ++e) val[e] = fmaf(f, x[u][e], val[e]);
          }
        i0 += BATCH * parts;
        if (i0 >= runs) break;
        load(column, i0);
      }
    }
    if (parts > 1) {  // one round: all columns fit the block
      sh.join.sum[threadIdx.x] = val;
      __syncthreads();
      for (int i = 1; i < parts && live && part == 0; ++i) val += sh.join.sum[i * columns + column];
    }
    if (live && part == 0) {
      const float l = s_l[0][row];
      const float inv = !CHUNK || sees(row) || l != l ? 1.f / l : 0.f;
      *reinterpret_cast<u32x2_t*>(p.out + result_row(row) * D + 4 * (column - row * (D / 4))) =
          u32x2_t{(uint32_t)limited<DT>(val[0] * inv) | ((uint32_t)limited<DT>(val[1] * inv) << 16),
                  (uint32_t)limited<DT>(val[2] * inv) | ((uint32_t)limited<DT>(val[3] * inv) << 16)};
    }
  }
  if (threadIdx.x == 0) atomicExch(&p.counters[unit], 0u);
}

// fn(DT, D, G) for the run-time dtype, head size and key groups
template <typename F>
int dispatch_layout(int dtype, int head_size, int groups, F&& fn) {
  auto with = [&](auto dt) {
    using DT = decltype(dt);
    auto sized = [&](auto d) {
      constexpr int D = decltype(d)::value;
      switch (groups) {
        case 1: return fn(DT{}, d, std::integral_constant<int, 1>{});
        case 2: return fn(DT{}, d, std::integral_constant<int, 2>{});
        case 4:
          if constexpr (D >= 128) return fn(DT{}, d, std::integral_constant<int, 4>{});
          break;
        case 8:
          if constexpr (D >= 256) return fn(DT{}, d, std::integral_constant<int, 8>{});
          break;
      }
      return GRINQH_ERR_INVALID;
    };
    switch (head_size) {
      case 64: return sized(std::integral_constant<int, 64>{});
      case 128: return sized(std::integral_constant<int, 128>{});
      case 256: return sized(std::integral_constant<int, 256>{});
    }
    return GRINQH_ERR_INVALID;
  };
  return dtype == GRINQH_DTYPE_BF16 ? with(BF16{}) : with(F16{});
}

int status() { return hipGetLastError() == hipSuccess ? GRINQH_OK : GRINQH_ERR_HIP; }

}  // namespace

int launch_kv4_store(HeadRows k, HeadRows v, const int64_t* slots, int64_t tokens, const Kv4Cache& cache, int dtype,
                     hipStream_t st) {
  return dispatch_layout(dtype, cache.head_size, cache.groups, [&](auto dt, auto d, auto g) -> int {
    constexpr int D = decltype(d)::value, ROWS = 2048 / D;
    const int64_t blocks = (tokens + ROWS - 1) / ROWS * cache.heads;
    if (blocks > INT32_MAX) return GRINQH_ERR_INVALID;
    hipLaunchKernelGGL((kv4_store_kernel<decltype(dt), D, decltype(g)::value>), dim3((uint32_t)blocks), dim3(256), 0,
                       st, k, v, slots, tokens, cache);
    return status();
  });
}

int launch_kv4_load(const Kv4Cache& cache, const int64_t* slots, int64_t tokens, uint16_t* k, uint16_t* v, int dtype,
                    hipStream_t st) {
  return dispatch_layout(dtype, cache.head_size, cache.groups, [&](auto dt, auto d, auto g) -> int {
    constexpr int D = decltype(d)::value, ROWS = 2048 / D;
    const int64_t blocks = (tokens + ROWS - 1) / ROWS * cache.heads;
    if (blocks > INT32_MAX) return GRINQH_ERR_INVALID;
    hipLaunchKernelGGL((kv4_load_kernel<decltype(dt), D, decltype(g)::value>), dim3((uint32_t)blocks), dim3(256), 0,
                       st, cache, slots, tokens, k, v);
    return status();
  });
}

Kv4Plan plan_kv4(int64_t seqs, int heads, int kv_heads, int head_size, int64_t capacity) {
  const int per = heads / kv_heads;
  const int64_t units = seqs * kv_heads * ((per + kRows - 1) / kRows);
  const int64_t steps = (capacity + 31) / 32;
  Kv4Plan plan;
  // Eight waves per CU are in flight either way.  Up to one block per CU they
  // are one block's, so that a long sequence is shared by half as many blocks
  // (1 x 131072 tokens, 8 heads: 38 us with 256 blocks of 8 waves, 42 with 512 of 4);
  // beyond, blocks of 4 waves waste less on short sequences (100 sequences of up
  // to 300 tokens, 8 heads: 10 against 16 us).
  plan.waves = units <= 256 ? 8 : 4;
  plan.blocks = plan.waves == 8 ? 256 : 512;
  // Four rounds of 8 waves.  Of a few thousand tokens fewer would serve as well or
  // better (1 x 4096, 8 heads: 15.2 us, 13.2 with 16 steps, 13.5 with 8; 1 x 16384 16.2,
  // 15.8, 15.8); longer or more sequences take the same either way.
  plan.least = 32;
  plan.slot = (per < kRows ? per : kRows) * head_size + 2 * kRows;
  // the runs beyond one per unit are at most `blocks`, and at most what the table's width allows
  const int64_t longest = (steps + plan.least - 1) / plan.least;
  plan.most = longest > 1 && units <= kKv4Counters && seqs <= 64 * kGroup ? kRuns : 1;
  plan.grid = units;
  if (plan.most > 1) plan.grid += units * (longest - 1) < plan.blocks ? units * (longest - 1) : plan.blocks;
  plan.workspace =
      plan.grid > units ? kKv4Counters * sizeof(uint32_t) + (size_t)plan.grid * plan.slot * sizeof(float) : 0;
  return plan;
}

template <typename B>
int launch_attention(const Kv4Params& p, const B& batch, int dtype, hipStream_t st) {
  return dispatch_layout(dtype, p.cache.head_size, p.cache.groups, [&](auto dt, auto d, auto g) -> int {
    constexpr int D = decltype(d)::value;
    if (p.plan.grid > INT32_MAX) return GRINQH_ERR_INVALID;
    auto kernel = p.plan.waves == 8 ? kv4_attention_kernel<decltype(dt), D, decltype(g)::value, 8, B>
                                    : kv4_attention_kernel<decltype(dt), D, decltype(g)::value, 4, B>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)p.plan.grid), dim3(64 * p.plan.waves), 0, st, p, batch);
    return status();
  });
}
int launch_kv4_attention(const Kv4Params& p, int dtype, hipStream_t st) {
  return launch_attention(p, OneRow{}, dtype, st);
}
int launch_kv4_attention_rows(const Kv4Params& p, const ChunkBatch& batch, int dtype, hipStream_t st) {
  return launch_attention(p, batch, dtype, st);
}

}  // namespace grinqh
