// Attention of chunks of new tokens over the 4-bit cache: packed rows, paged keys
// and values, causal, grouped heads.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j),  j <= i + (length - rows) of the sequence
//
// Rows of a block are (token, query head of one key/value head) pairs, so that all
// heads that share keys share the work of unpacking them: a tile of 64 tokens is
// loaded as it is kept, turned into fp16 by all threads together and left in LDS.
#include <cfloat>
#include <type_traits>

#include "attention_launch.h"
#include "grinqh_common.h"
#include "wave_scan.h"

namespace grinqh {

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4_t;

constexpr int kKeys = 64;         // tokens per tile
constexpr int kGroup = 4;         // sequences a lane looks at in a round of the plan
constexpr float kLow = -FLT_MAX;  // running reference before the first token (finite: -inf - -inf would be NaN)

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

// Sequence -1 stands for the rows in front of the first sequence, sequence `seqs` for
// those behind the last: they see no token, and their results are zeros.
struct Sequence {
  int row0, rows;  // tokens of the chunk
  int length;      // tokens in the cache that count
  bool bad;        // more than the page table covers
};
__device__ __forceinline__ int row_at(const ChunkParams& p, int i) {
  return (int)min((int64_t)max(p.ends[i], 0), p.tokens);
}
__device__ __forceinline__ Sequence sequence(const ChunkParams& p, int s) {
  Sequence q;
  q.row0 = s < 0 ? 0 : row_at(p, s);
  q.rows = max((s >= p.seqs ? (int)p.tokens : row_at(p, s + 1)) - q.row0, 0);
  q.length = 0;
  q.bad = false;
  if (s >= 0 && s < p.seqs) {
    const int64_t capacity = (int64_t)p.table_width << (p.sub_shift + 4);
    const int length = max(p.lengths[s], 0);
    q.bad = length > capacity;
    q.length = q.bad ? (int)capacity : length;
  }
  return q;
}

struct Share {
  Sequence q;
  int seq, head;    // key/value head
  int block;        // of rows, in the sequence
  int run, runs;
  int64_t id;       // place in the workspace of the unit's first run; the others stand `heads` apart
};

// Runs that each unit of a sequence is split into, `chunk` tiles each.
__device__ __forceinline__ int runs_of(const ChunkParams& p, int length, int chunk) {
  if (p.plan.most == 1) return 1;
  return min(max(((length + kKeys - 1) / kKeys + chunk - 1) / chunk, 1), p.plan.most);
}

// Every block plans by itself from the offsets and lengths, which only the device
// knows: units are blocks of rows and a key/value head, all tiles are shared out over
// plan.blocks, in runs of at least plan.least tiles, all runs of a sequence alike.
// With `joined` blocks stand for units, not runs.  False: past the last.
__device__ __forceinline__ bool find_share(const ChunkParams& p, int64_t id, bool joined, int lane, Share& out) {
  const int heads = p.cache.heads, per = p.heads / heads, block_rows = 32 * p.plan.waves;
  const int64_t at = id / heads;
  out.head = (int)(id - at * heads);
  auto blocks_of = [&](const Sequence& q) { return (int)(((int64_t)q.rows * per + block_rows - 1) / block_rows); };
  int chunk = 1;
  if (p.plan.most > 1) {
    float tiles = 0.f;
    for (int s0 = 0; s0 < p.seqs; s0 += 64 * kGroup)
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        const int s = s0 + 64 * i + lane;
        if (s < p.seqs) {
          const Sequence q = sequence(p, s);
          tiles += (float)blocks_of(q) * (float)((q.length + kKeys - 1) / kKeys);
        }
      }
    const float total =
        __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_scan(tiles)), 63));
    chunk = max(p.plan.least, (int)ceilf(fminf(total * (float)heads / (float)p.plan.blocks, 0x1p26f)));
  }
  int64_t before = 0, runs_before = 0;
  for (int s0 = -1; s0 <= p.seqs; s0 += 64) {
    const int s = s0 + lane;
    int blocks = 0, runs = 1;
    if (s <= p.seqs) {
      const Sequence q = sequence(p, s);
      blocks = blocks_of(q);
      runs = runs_of(p, q.length, chunk);
    }
    const int items = joined ? blocks : blocks * runs;
    const int upto = wave_scan(items), all = wave_scan(blocks * runs);
    const uint64_t after = __ballot(before + upto > at);
    if (after != 0) {
      const int owner = __builtin_ctzll(after);
      out.seq = s0 + owner;
      out.q = sequence(p, out.seq);
      out.runs = __builtin_amdgcn_readlane(runs, owner);
      const int rest = (int)(at - before) - __builtin_amdgcn_readlane(upto - items, owner);
      const int index = joined ? rest : rest / out.runs;
      out.run = joined ? 0 : rest - index * out.runs;
      // those with the most tokens first
      const int count = __builtin_amdgcn_readlane(blocks, owner);
      out.block = count - 1 - index;
      if (index < 0 || index >= count) return false;  // offsets that are not ascending
      out.id = (runs_before + __builtin_amdgcn_readlane(all - blocks * runs, owner) + (int64_t)index * out.runs) * heads +
               out.head;
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    runs_before += __builtin_amdgcn_readlane(all, 63);
  }
  return false;
}

// ---------------------------------------------------------------- unpacking

// 8 codes as fp16 pairs minimum + scale * code (rounded once).  A nibble under the
// exponent of 1024 is 1024 + code, one in the upper half of a byte 1024 + 16 code.
__device__ __forceinline__ u32x4_t unpack8(uint32_t w, f16x2_t scale, f16x2_t low) {
  const uint32_t u = w >> 8, base = 0x64006400u;
  const f16x2_t one = {(_Float16)-1024.f, (_Float16)-1024.f}, sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f},
                less = {(_Float16)-64.f, (_Float16)-64.f};
  auto pair = [&](uint32_t x, bool upper) {
    const f16x2_t c = __builtin_bit_cast(f16x2_t, x | base);
    const f16x2_t code = upper ? __builtin_elementwise_fma(c, sixteenth, less) : c + one;
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(code, scale, low));
  };
  return u32x4_t{pair(w & 0x000F000Fu, false), pair(w & 0x00F000F0u, true), pair(u & 0x000F000Fu, false),
                 pair(u & 0x00F000F0u, true)};
}
__device__ __forceinline__ u32x4_t limited8(u32x4_t x) {
  const f16x2_t most = (f16x2_t)((_Float16)65504.f);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(
                                            __builtin_elementwise_min(__builtin_bit_cast(f16x2_t, x[i]), most), -most));
  return x;
}
__device__ __forceinline__ f16x2_t both(uint32_t half) {
  return __builtin_bit_cast(f16x2_t, (half & 0xFFFFu) * 0x00010001u);
}
// a parameter that is NaN or infinite
__device__ __forceinline__ bool broken(uint32_t pair) {
  return (pair & 0x7C00u) == 0x7C00u || (pair & 0x7C000000u) == 0x7C000000u;
}
// Codes of this group may stand for more than fp16 holds (where a scale was rounded up).
__device__ __forceinline__ bool reaching(uint32_t pair) {
  return fmaf(15.f, fabsf(half_lo(pair)), fabsf(half_hi(pair))) > 65504.f;
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

// What a thread holds of a tile, as the cache keeps it.
template <int D, int WAVES>
struct Tile {
  static constexpr int WORDS = D / (8 * WAVES);              // of keys, and of values
  static constexpr int VEC = WORDS < 4 ? WORDS : 4;          // tokens of one chunk of the values
  static constexpr int PAIRS = WORDS < D / 32 ? WORDS : D / 32;
  uint32_t k[WORDS], kp[PAIRS];
  uint32_t v[WORDS / VEC][VEC], vp[WORDS / VEC][VEC];
  uint32_t own;  // the key's token: its values' parameters
  bool lost;     // its page is outside the cache
};

// ---------------------------------------------------------------- the kernel

template <bool BF, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, D > 128 ? 1 : 2) void chunk_attention_kernel(const ChunkParams p) {
  constexpr int STEPS = D / 16, MT = D / 32, W = D / 32, THREADS = 64 * WAVES;
  // A row of keys (values) is 16 (64) bytes longer than it need be: the 32 adjacent
  // keys' chunks of one read, and 4 adjacent values' 64 bytes, then lie in different banks.
  constexpr int KEY_ROW = 2 * D + 16, VALUE_ROW = 2 * D + 64;
  __shared__ __align__(16) uint8_t s_k[kKeys * KEY_ROW], s_v[kKeys * VALUE_ROW];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 31, half = lane >> 5;
  Share share;
  if (!find_share(p, blockIdx.x, false, lane, share)) return;
  const Sequence sq = share.q;
  const int per = p.heads / p.cache.heads;
  const int64_t rows = (int64_t)sq.rows * per;                      // of the sequence: (token, head)
  const int64_t row0 = ((int64_t)share.block * WAVES + wave) * 32;  // of this wave
  const bool live = row0 < rows;
  const int shift = sq.length - sq.rows;
  // this lane's row; past the last one it stands for the last and is not stored
  const int64_t row = min(row0 + n, rows - 1);
  const int token = (int)(row / per), head = share.head * per + (int)(row - (int64_t)token * per);
  const int seen = token + shift;  // last token it sees

  // tiles of the block's last row, and this run's share
  const int64_t last_row = min(((int64_t)share.block + 1) * 32 * WAVES, rows) - 1;
  const int tiles = max((int)(last_row / per) + shift + kKeys, 0) / kKeys;
  const int part = (tiles + share.runs - 1) / share.runs;
  const int first = min(share.run * part, tiles), last = min(first + part, tiles);
  // this wave's: up to what its last row sees; masked from where its first one ends
  const int wave_last = live ? (int)(min(row0 + 31, rows - 1) / per) + shift : -1;
  const int wave_seen = live ? (int)(row0 / per) + shift : 0;
  const int my_last = min(last, max(wave_last + kKeys, 0) / kKeys);

  // ---- a thread's share of a tile
  using T = Tile<D, WAVES>;
  constexpr int KEY_LANES = WAVES;  // threads per token's keys
  const int ktok = tid / KEY_LANES, kword = tid % KEY_LANES * T::WORDS;  // token of the tile, first word
  const int rec_of_tile = ktok >> 4;
  const int groups = p.cache.groups, record = kv4_record_bytes(D, groups);
  const int pair_shift = __builtin_ctz((unsigned)(D / groups)) - 5;  // words i of a group share parameters
  const int last_rec = max((sq.length - 1) >> 4, 0);
  const int32_t* table = p.table + (int64_t)share.seq * p.table_stride;
  auto page_of = [&](int tile) { return table[min(4 * tile + rec_of_tile, last_rec) >> p.sub_shift]; };
  auto load_tile = [&](T& t, int tile, int page) {
    t.lost = (uint32_t)page >= (uint64_t)p.cache.pages;
    const int rec = min(4 * tile + rec_of_tile, last_rec);
    const uint8_t* at = p.cache.p + ((((int64_t)(t.lost ? 0 : page) * p.cache.heads + share.head) << p.sub_shift) +
                                     (rec & (p.cache.sub - 1))) * record;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(at);
    load_words(t.k, w + (ktok & 15) * (D / 8) + kword);
#pragma unroll
    for (int i = 0; i < T::PAIRS; ++i) t.kp[i] = w[2 * D + (((kword + i) % W) >> pair_shift) * 16 + (ktok & 15)];
    const uint32_t* v = w + 2 * D + 16 * groups;
    t.own = v[2 * D + (ktok & 15)];
    const int x = tid % (16 * WAVES);
#pragma unroll
    for (int j = 0; j < T::WORDS / T::VEC; ++j) {
      const int id = x + 16 * WAVES * j, chunk = id % (D / 8), tok = id / (D / 8) * T::VEC;
      load_words(t.v[j], v + chunk * 16 + tok);
      load_words(t.vp[j], v + 2 * D + tok);
    }
  };
  // A token whose values are NaN (or lie outside the cache) gives zeros, and NaN as
  // its key: that reaches the rows that see it and no others, as the others' logits are masked.
  auto write_tile = [&](const T& t) {
    bool far = false;
    uint32_t kp[T::PAIRS];
#pragma unroll
    for (int i = 0; i < T::PAIRS; ++i) {
      kp[i] = t.lost || broken(t.own) ? 0x7E007E00u : t.kp[i];
      far |= reaching(kp[i]);
    }
    far = __any(far);
#pragma unroll
    for (int i = 0; i < T::WORDS; ++i) {
      const int word = kword + i, chunk = word / W + 4 * (word % W);
      const uint32_t pair = kp[i % T::PAIRS];
      u32x4_t x = unpack8(t.k[i], both(pair), both(pair >> 16));
      if (far) x = limited8(x);
      *reinterpret_cast<u32x4_t*>(s_k + ktok * KEY_ROW + chunk * 16) = x;
    }
    const int x0 = tid % (16 * WAVES), base = tid / (16 * WAVES) * 16;
#pragma unroll
    for (int j = 0; j < T::WORDS / T::VEC; ++j) {
      const int id = x0 + 16 * WAVES * j, chunk = id % (D / 8), tok = id / (D / 8) * T::VEC;
      uint32_t vp[T::VEC];
      far = false;
#pragma unroll
      for (int e = 0; e < T::VEC; ++e) {
        vp[e] = t.lost || broken(t.vp[j][e]) ? 0u : t.vp[j][e];
        far |= reaching(vp[e]);
      }
      far = __any(far);
#pragma unroll
      for (int e = 0; e < T::VEC; ++e) {
        u32x4_t x = unpack8(t.v[j][e], both(vp[e]), both(vp[e] >> 16));
        if (far) x = limited8(x);
        *reinterpret_cast<u32x4_t*>(s_v + (base + tok + e) * VALUE_ROW + chunk * 16) = x;
      }
    }
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
  auto read_key = [&](int b, int s) {
    return *reinterpret_cast<const u32x4_t*>(s_k + key_base + 32 * b * KEY_ROW + 32 * s);
  };
  auto read_value = [&](int t, int m) {
    u32x4_t a;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4_t)(s_v + value_base + (16 * t + 8 * u) * VALUE_ROW + 64 * m));
      const u32x2_t y = __builtin_bit_cast(u32x2_t, x);
      a[2 * u] = y[0];
      a[2 * u + 1] = y[1];
    }
    return a;
  };
  auto compute = [&](int tile) {
    f32x16_t S[2];
    float top = -__builtin_inff();
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      S[b] = (f32x16_t)(0.f);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) S[b] = mfma32x32x16(read_key(b, s), qf[s], S[b]);
    }
    if (tile * kKeys + kKeys - 1 > wave_seen) {
      // last token of this tile that the row sees, less the half's 4 (compared with constants)
      const int upto = seen - tile * kKeys - 4 * half;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (32 * b + (e & 3) + 8 * (e >> 2) > upto) S[b][e] = -__builtin_inff();
    }
    // S zs is exact in the exponent and M is not: the same factor for all tokens of a
    // row, but of more than 2^16 for logits past 2^28.  With `far` the product is rounded first.
    auto product_first = [&]() {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          S[b][e] *= unit;
          asm volatile("" : "+v"(S[b][e]));  // not contracted with the subtraction
        }
    };
    if (far) product_first();
    auto reach = [&]() {
      top = -__builtin_inff();
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, S[b][e]);
    };
    reach();
    if (__any(fmaf(top, zs, -M) > 8.f)) {
      float m = fmaxf(M, top * zs);
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      if (!far && __any(fabsf(m) > 0x1p24f && m != kLow)) {
        far = true;
        zs = 1.f;
        product_first();
        reach();
        m = fmaxf(M, top);
        m = fmaxf(m, __shfl_xor(m, 32, 64));
      }
      const float f = __builtin_amdgcn_exp2f(M - m);
      M = m;
      sum *= f;
#pragma unroll
      for (int t = 0; t < MT; ++t) O[t] *= f;
    }
    u32x4_t P[4];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(S[b][2 * i], zs, -M));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(S[b][2 * i + 1], zs, -M));
        sum += p0 + p1;
        P[2 * b + (i >> 2)][i & 3] = f16_pair(p0, p1);
      }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) O[m] = mfma32x32x16(read_value(t, m), P[t], O[m]);
  };

  T t;
  int page = 0;
  if (first < last) {
    load_tile(t, first, page_of(first));
    page = page_of(first + 1);
  }
  for (int tile = first; tile < last; ++tile) {
    __syncthreads();  // the tile before has been read
    write_tile(t);
    if (tile + 1 < last) {
      load_tile(t, tile + 1, page);
      page = page_of(tile + 2);
    }
    __syncthreads();
    if (tile < my_last) compute(tile);
  }
  if (!live) return;

  sum += __shfl_xor(sum, 32, 64);
  if (sq.bad) sum = __builtin_nanf("");
  const bool mine = row0 + n < rows;
  if (share.runs > 1) {
    const int r = wave * 32 + n;
    float* slot = p.partial + (share.id + (int64_t)share.run * p.cache.heads) * p.plan.slot;
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
    return;
  }
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

// Joins the runs of split units: 1024 results per block, 4 per thread.
template <bool BF, int D>
__global__ __launch_bounds__(256) void chunk_join_kernel(const ChunkParams p) {
  constexpr int ROWS = 1024 / D;
  const int block_rows = 32 * p.plan.waves, parts = block_rows / ROWS;
  const int lane = threadIdx.x & 63;
  Share share;
  if (!find_share(p, blockIdx.x / parts, true, lane, share) || share.runs == 1) return;
  if (share.id + (int64_t)(share.runs - 1) * p.cache.heads >= p.plan.grid) return;  // offsets that are not ascending
  const int per = p.heads / p.cache.heads;
  const int r = (int)(blockIdx.x % parts) * ROWS + threadIdx.x / (D / 4), c = threadIdx.x % (D / 4) * 4;
  const int64_t row = (int64_t)share.block * block_rows + r;
  if (row >= (int64_t)share.q.rows * per) return;
  const int token = (int)(row / per), head = share.head * per + (int)(row - (int64_t)token * per);
  const float* slot = p.partial + share.id * p.plan.slot;
  const int64_t step = (int64_t)p.cache.heads * p.plan.slot;
  float M = kLow, sum = 0.f;
  for (int i = 0; i < share.runs; ++i) M = fmaxf(M, slot[i * step + block_rows * D + r]);
  f32x4_t o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = 0; i < share.runs; ++i) {
    const float f = __builtin_amdgcn_exp2f(slot[i * step + block_rows * D + r] - M);
    sum = fmaf(f, slot[i * step + block_rows * (D + 1) + r], sum);
    const f32x4_t x = *reinterpret_cast<const f32x4_t*>(slot + i * step + r * D + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(f, x[e], o[e]);
  }
  const bool sees = token + share.q.length - share.q.rows >= 0;
  const float inv = sees || sum != sum ? 1.f / sum : 0.f;
  *reinterpret_cast<u32x2_t*>(p.out + (((int64_t)share.q.row0 + token) * p.heads + head) * D + c) =
      u32x2_t{result_pair<BF>(o[0] * inv, o[1] * inv), result_pair<BF>(o[2] * inv, o[3] * inv)};
}

}  // namespace

ChunkPlan plan_chunk(int64_t tokens, int64_t seqs, int heads, int kv_heads, int head_size, int64_t capacity) {
  const int per = heads / kv_heads;
  ChunkPlan plan;
  plan.waves = head_size > 128 ? 4 : 8;
  if (head_size <= 128 && tokens * per <= 64 * seqs) plan.waves = 2;
  const int64_t block_rows = 32 * plan.waves;
  // a partial block for every sequence and for the rows in front of them and behind
  const int64_t blocks = (tokens * per + block_rows - 1) / block_rows + seqs + 2;
  plan.units = blocks * kv_heads;
  plan.blocks = plan.waves == 2 ? 1024 : 256;
  plan.least = 4;
  const int64_t tiles = (capacity + kKeys - 1) / kKeys;
  plan.most = plan.units < plan.blocks && tiles > plan.least ? 64 : 1;
  plan.grid = plan.units;
  plan.slot = block_rows * (head_size + 2);
  plan.workspace = 0;
  if (plan.most > 1) {
    const int64_t longest = (tiles + plan.least - 1) / plan.least;
    plan.most = longest < plan.most ? (int)longest : plan.most;
    // a unit has at most one run more than its share of plan.blocks
    const int64_t more = plan.units * (plan.most - 1);
    plan.grid += more < plan.blocks ? more : plan.blocks;
    plan.workspace = (size_t)plan.grid * plan.slot * sizeof(float);
  }
  return plan;
}

int launch_chunk_attention(const ChunkParams& p, int dtype, hipStream_t st) {
  const int64_t joins = p.plan.units * 32 * p.plan.waves * p.cache.head_size / 1024;
  if (p.plan.grid > INT32_MAX || (p.plan.most > 1 && joins > INT32_MAX)) return GRINQH_ERR_INVALID;
  auto go = [&](auto bf, auto d) -> int {
    constexpr bool BF = decltype(bf)::value;
    constexpr int D = decltype(d)::value, WIDE = D > 128 ? 4 : 8;
    auto kernel = chunk_attention_kernel<BF, D, WIDE>;
    if constexpr (D <= 128)
      if (p.plan.waves == 2) kernel = chunk_attention_kernel<BF, D, 2>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)p.plan.grid), dim3(64 * p.plan.waves), 0, st, p);
    if (p.plan.most > 1)
      hipLaunchKernelGGL((chunk_join_kernel<BF, D>), dim3((uint32_t)joins), dim3(256), 0, st, p);
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
