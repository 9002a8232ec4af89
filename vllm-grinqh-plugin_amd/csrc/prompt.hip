// Attention over whole prompts: packed sequences, causal, grouped heads.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j),  j <= i + (keys - rows) of the sequence
//
// One pass over the keys with a running reference of the exponent.  S^T = K Q^T
// leaves a lane of v_mfma_f32_32x32x16 with one query row and 16 of 32 keys,
// which is the B operand of O^T = V^T P^T, so P never leaves its lane; keys
// and values go through LDS by direct loads, the values read back transposed
// (ds_read_b64_tr_b16).
//
// Bound by the matrix unit and the exponentials together: a tile of 64 keys and
// 32 rows of 128 channels takes 32 products of 32 cycles and some 130 VALU
// operations, 32 of them v_exp_f32 (8 cycles with two waves per SIMD, 16 with
// one).  One wave per SIMD issues a VALU operation every 6 cycles at most, two
// every 4-5 (measured), so a wave has 32 rows and a SIMD two waves (64 rows and one
// wave per SIMD would read LDS half as often, but took 826 us: accumulators moved
// between the register files).  One sequence of 8192 rows, 32 heads: 521 us, 1055
// TFLOP/s, where a library product of 8192^3 reaches 1400.  Heads of 256 channels
// need 445 registers (256 and 189 of the accumulators' file, with moves between the
// two in the loop), one wave per SIMD: 510 TFLOP/s.
//
// What a first pass cannot do is left to a second one over the block's keys, which
// blocks with NaN, infinite or very large inputs take: 2.0-2.6 times their time (3.5 with
// heads of 256 channels).
#include <cfloat>
#include <type_traits>

#include "attention_launch.h"
#include "grinqh_common.h"
#include "wave_scan.h"

namespace grinqh {

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4_t;
typedef __attribute__((address_space(3))) void* lds_t;

template <typename DT>
__device__ __forceinline__ f32x16_t mfma32x32x16(const u32x4_t& a, const u32x4_t& b, f32x16_t c) {
  if constexpr (DT::id == F16::id)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0,
                                                  0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
}

template <typename DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT::id == F16::id)
    return (uint32_t)f32_to_f16_bits(lo) | ((uint32_t)f32_to_f16_bits(hi) << 16);
  else
    return f32x2_to_bf16x2(lo, hi);
}

// Two results.  Weights are rounded for the second product and their sum is not,
// so that a mean of fp16 values next to the limit may pass it: it is limited.
// (What infinite and NaN accumulators become is put right in the second pass.)
template <typename DT>
__device__ __forceinline__ uint32_t pack_results(float lo, float hi) {
  const uint32_t w = pack2<DT>(lo, hi);
  if constexpr (DT::id != F16::id) return w;
  typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
  const f16x2_t most = (f16x2_t)((_Float16)65504.f);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(
                                          __builtin_elementwise_min(__builtin_bit_cast(f16x2_t, w), most), -most));
}

constexpr int kWaves = 4;
constexpr int kBlockRows = 32 * kWaves;
constexpr int kKeys = 64;       // keys per tile
// running reference before the first key (finite: -inf - -inf would be NaN; a row of
// logits below it is one for the second pass)
constexpr float kLow = -1e30f;
// A raised reference is so far (in powers of two) below the largest logit, and is raised again where a weight would
// pass 2^kRaise.  fp16's weights need that room below: beside a largest one of 1, those 17 nats lower are subnormal or
// zero, and where they are many thousands, of a token with a value near zero and all others, results were 3e-2 off.  From
// 2^7 on they are normal numbers down to 2^-21 of the largest, and off by 2^-32 of it below.  bf16 has the range.
template <typename DT>
constexpr float kRoom = DT::id == F16::id ? 7.f : 0.f;
template <typename DT>
constexpr float kRaise = kRoom<DT> + 8.f;

// A value that all lanes agree on, in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// One sequence's rows and keys.  Sequence `seqs` stands for the rows behind the
// last sequence: it has no keys, so its rows become zeros.
struct Sequence {
  int64_t row0, key0;
  int64_t rows, keys;
};
__device__ __forceinline__ int64_t offset_at(const int32_t* ends, int i, int64_t most) {
  return min(max((int64_t)ends[i], (int64_t)0), most);
}
__device__ __forceinline__ Sequence sequence(const PromptParams& p, int s) {
  Sequence q;
  q.row0 = offset_at(p.ends, s, p.q_tokens);
  if (s >= p.seqs) return {q.row0, 0, p.q_tokens - q.row0, 0};
  q.key0 = offset_at(p.key_ends, s, p.k_tokens);
  q.rows = max(offset_at(p.ends, s + 1, p.q_tokens) - q.row0, (int64_t)0);
  q.keys = max(offset_at(p.key_ends, s + 1, p.k_tokens) - q.key0, (int64_t)0);
  return q;
}

// Block `index` of the rows' blocks, those with the most keys first: level l
// holds the blocks whose last row sees about l * kBlockRows keys (at most one
// per sequence).  Returns the sequence, or -1 past the last block.
__device__ __forceinline__ int find_block(const PromptParams& p, int64_t index, int lane,
                                          Sequence& found, int64_t& block) {
  const int seqs = p.seqs + 1;
  // blocks of sequence s at level >= l: their indices b + before >= l
  auto count_of = [&](int s, int& blocks, int& before) {
    blocks = before = 0;
    if (s >= seqs) return;
    const Sequence q = sequence(p, s);
    blocks = (int)((q.rows + kBlockRows - 1) / kBlockRows);
    before = (int)(max(q.keys - q.rows, (int64_t)0) / kBlockRows);
  };
  int my_blocks, my_before;
  count_of(lane, my_blocks, my_before);
  auto at_least = [&](int level) {
    int sum = 0;
    for (int s = lane; s < seqs; s += 64) {
      int blocks = my_blocks, before = my_before;
      if (s >= 64) count_of(s, blocks, before);
      sum += min(max(blocks - max(level - before, 0), 0), blocks);
    }
    return wave_sum(sum);
  };
  if (index >= at_least(0)) return -1;
  int lo = 0, hi = 1;  // at_least(lo) > index >= at_least(hi)
  while (at_least(hi) > index) {
    lo = hi;
    hi *= 2;
  }
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at_least(mid) > index)
      lo = mid;
    else
      hi = mid;
  }
  int64_t rank = index - at_least(hi);  // among the blocks at level lo
  for (int s0 = 0; s0 < seqs; s0 += 64) {
    int blocks, before;
    count_of(s0 + lane, blocks, before);
    const int b = lo - before;
    const bool here = b >= 0 && b < blocks;
    const uint64_t mask = __ballot(here);
    const int n = __popcll(mask);
    if (rank < n) {
      uint64_t m = mask;
      for (int i = 0; i < (int)rank; ++i) m &= m - 1;
      const int s = s0 + __builtin_ctzll(m);
      found = sequence(p, s);
      block = lo - (int)(max(found.keys - found.rows, (int64_t)0) / kBlockRows);
      return s;
    }
    rank -= n;
  }
  return -1;
}

// Block = 4 waves x 32 query rows of one head.
template <typename DT, int D>
__global__ __launch_bounds__(64 * kWaves, D > 128 ? 1 : 2) void prompt_attention_kernel(const PromptParams p) {
  constexpr int STEPS = D / 16, MT = D / 32, CHUNKS = D / 8;
  constexpr int PER = 64 / CHUNKS;                      // keys per KiB
  constexpr int KEY_GROUP = 1024 + (D > 128 ? 32 : 64);  // bytes from one KiB of keys to the next
  constexpr int KEY_TILE = kKeys / PER * KEY_GROUP, VALUE_TILE = kKeys * D * 2;  // bytes
  // separate arrays, used by name: the compiler's wait for a tile that was loaded
  // straight into LDS is then not one for the tiles still on their way
  __shared__ __align__(1024) uint8_t s_k0[KEY_TILE], s_k1[KEY_TILE], s_v0[VALUE_TILE], s_v1[VALUE_TILE];
  __shared__ __align__(16) int s_first[3][D];  // first key whose value is NaN, +inf, -inf, by channel
  __shared__ int s_redo[kWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // heads of one key/value head run on one XCD (its L2 then holds their keys and values)
  int head;
  int64_t index;
  const int L = blockIdx.x;
  if (p.heads % 8 == 0) {
    const int per = p.heads / 8;
    head = (L % 8) * per + (L / 8) % per;
    index = L / 8 / per;
  } else {
    head = L % p.heads;
    index = L / p.heads;
  }
  // A head's first block: zeros for the rows in front of the first sequence, which
  // are few.  The others need not wait for ends[0].
  if (index == 0) {
    const int64_t chunks = offset_at(p.ends, 0, p.q_tokens) * CHUNKS;
    for (int64_t i = threadIdx.x; i < chunks; i += 64 * kWaves)
      *reinterpret_cast<u32x4_t*>(p.out + (i / CHUNKS * p.heads + head) * D + i % CHUNKS * 8) =
          u32x4_t{0u, 0u, 0u, 0u};
    return;
  }
  --index;

  // The block's rows, and what the second pass has to put right: values that are
  // NaN or infinite (kApart), logits too large for the weights' arithmetic (kFar).
  // Two copies of the code, so that the second pass costs the first no registers.
  constexpr int kApart = 1, kFar = 2;
  auto attend = [&](auto second, int lane, bool far) __attribute__((always_inline)) -> int {
    constexpr bool APART = decltype(second)::value;
    const int n = lane & 31, half = lane >> 5;
    Sequence sq;
    int64_t block;
    if (find_block(p, index, lane, sq, block) < 0) return 0;
    sq = {uniform(sq.row0), uniform(sq.key0), uniform(sq.rows), uniform(sq.keys)};
    block = uniform(block);
    const int kvh = head / (p.heads / p.kv_heads);
    const int row0 = (int)block * kBlockRows + wave * 32;  // of this wave, in the sequence
    const int rows = (int)sq.rows, shift = (int)(sq.keys - sq.rows), keys = (int)sq.keys;
    // keys that the block's last row sees
    const int block_keys = min(keys, min((int)(block + 1) * kBlockRows, rows) + shift);
    const int tiles = block_keys > 0 ? (block_keys + kKeys - 1) / kKeys : 0;
    const int wave_keys = row0 < rows ? min(keys, min(row0 + 32, rows) + shift) : 0;

    // queries: row n, channels 16 s + 8 half + e
    u32x4_t qf[STEPS];
    {
      const uint16_t* q = p.q.p + (sq.row0 + min(row0 + n, rows - 1)) * p.q.token + (int64_t)head * p.q.head + 8 * half;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) qf[s] = *reinterpret_cast<const u32x4_t*>(q + 16 * s);
    }

    // LDS position of 16-byte chunk c of key r.  Loads straight into LDS put 1 KiB
    // (PER keys) in a row, so what is read together is spread over the banks by
    // flipping bits of c, and for the keys by a gap after every KiB as well: the
    // keys' reads want 16 adjacent keys' chunks in 256 different bytes, the values'
    // transposed reads 4 adjacent keys' 64 bytes.  Few bits are flipped, so that
    // most of an address is an immediate offset.
    auto key_swz = [](int r) { return D == 64 ? (r >> 1) & 3 : D == 128 ? r & 3 : r & 1; };
    auto value_swz = [](int r) { return (D == 64 ? (r >> 1) & 1 : r & 3) << 2; };
    auto key_at = [](int r) { return r / PER * KEY_GROUP + r % PER * (2 * D); };
    const uint16_t* kbase = p.k.p + sq.key0 * p.k.token + (int64_t)kvh * p.k.head;
    const uint16_t* vbase = p.v.p + sq.key0 * p.v.token + (int64_t)kvh * p.v.head;
    // A wave loads PER keys at a time, 1 KiB; keys past the sequence's end come as
    // zeros (behind the buffer's end, as rows are at least D apart).
    const int load_row = wave * PER + lane / CHUNKS;
    static_assert(kWaves * PER % 8 == 0, "the flipped bits are the same for all loads of a lane");
    const int key_off = load_row * (int)p.k.token * 2 + (((lane % CHUNKS) ^ key_swz(load_row)) << 4);
    const int value_off = load_row * (int)p.v.token * 2 + (((lane % CHUNKS) ^ value_swz(load_row)) << 4);
    auto load_tile = [&](const uint16_t* base, int64_t stride, int off, int tile, uint8_t* to, int group) {
#pragma unroll
      for (int i = 0; i < kKeys / PER / kWaves; ++i) {
        const int r0 = tile * kKeys + i * kWaves * PER, live = min(kKeys, keys - r0);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t*>(base + (int64_t)r0 * stride), (short)0,
            live > 0 ? (int)(((live - 1) * stride + D) * 2) : 0, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_t)(to + (i * kWaves + wave) * group), 16, off, 0, 0, 0);
      }
    };

    f32x16_t O[MT];
    float M = APART && far ? -FLT_MAX : kLow, sum = 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m) O[m] = (f32x16_t)(0.f);
    const float c2 = p.scale * 1.44269504088896f;
    const int my_tiles = wave_keys > 0 ? (wave_keys + kKeys - 1) / kKeys : 0;

    // LDS reads.  Keys: row n of key block b, channels 16 s + 8 half + e.  Values,
    // transposed: channel 32 m + n, keys 16 t + 4 half + 0..3 and + 8.
    // The flipped bits make two bases (four for the values), the rest are offsets.
    int key_base[2], value_base[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) key_base[i] = key_at(n) + (((2 * i + half) ^ key_swz(n)) << 4);
    const int vrow = 4 * half + ((lane & 15) >> 2);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      value_base[i] = vrow * D * 2 + (((4 * i + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ value_swz(vrow)) << 4) +
                      8 * (lane & 1);
    auto read_key = [&](const uint8_t* kt, int b, int s) {
      return *reinterpret_cast<const u32x4_t*>(kt + key_base[s & 1] + key_at(32 * b) + 64 * (s >> 1));
    };
    auto read_value = [&](const uint8_t* vt, int t, int m) {
      u32x4_t a;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4_t)(vt + value_base[m & 3] + (16 * t + 8 * u) * D * 2 + 256 * (m >> 2)));
        const u32x2_t y = __builtin_bit_cast(u32x2_t, x);
        a[2 * u] = y[0];
        a[2 * u + 1] = y[1];
      }
      return a;
    };
    u32x4_t P[4];
    // The exponent of a weight.  S c2 is exact in here and M is not, which is the same
    // factor for all keys of a row, but of more than 2^16 for logits past 2^28: with
    // `far` M is in S's unit, and the difference is taken first.
    auto power = [&](float s) { return APART && far ? (s - M) * c2 : fmaf(s, c2, -M); };
    // Weights of two keys, pair q of key block b: in the tensors' type for the second
    // product, the only operand it takes at that rate.  Their sum is that of the
    // unrounded ones, so a result is off by a mean of the roundings (2^-8 and 2^-11 each
    // at most of what they weigh, to either side).
    auto weigh = [&](const f32x16_t (&S)[2], int b, int q) {
      const float p0 = __builtin_amdgcn_exp2f(power(S[b][2 * q]));
      const float p1 = __builtin_amdgcn_exp2f(power(S[b][2 * q + 1]));
      sum += p0 + p1;
      P[2 * b + (q >> 2)][q & 3] = pack2<DT>(p0, p1);
    };
    // Makes S of a tile ready for its weights: the mask where the tile reaches
    // past a row's last key, and the reference raised where a weight would pass
    // 2^kRaise (rarely after the first tiles: the accumulators are not rescaled for less).
    // With `far` it is the largest logit itself, whose steps are wider than the room.
    auto settle = [&](f32x16_t (&S)[2], float& top, int tile) {
      if (tile * kKeys + kKeys - 1 > row0 + shift) {
        // last key of this tile that the row sees, less the half's 4 (compared with constants)
        const int seen = row0 + n + shift - tile * kKeys - 4 * half;
        top = -__builtin_inff();
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (32 * b + (e & 3) + 8 * (e >> 2) > seen) S[b][e] = -__builtin_inff();
            top = fmaxf(top, S[b][e]);
          }
      }
      if (__any(power(top) > kRaise<DT>)) {
        float m = fmaxf(M, APART && far ? top : top * c2 - kRoom<DT>);
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const float f = __builtin_amdgcn_exp2f(APART && far ? (M - m) * c2 : M - m);
        M = m;
        sum *= f;
#pragma unroll
        for (int t = 0; t < MT; ++t) O[t] *= f;
      }
    };

    // One tile: its weights and its part of O, and the products of the next tile,
    // slot by slot: every slot gives the matrix unit one product and the vector unit
    // a share of the exponentials (those of keys 0..31 under the next tile's
    // products, those of keys 32..63 under the first values'), with LDS reads AHEAD
    // slots before their use (1: 571 us, 2: 539, 3: 533 at one sequence of 8192 rows,
    // 32 heads of 128).
    constexpr int KSLOTS = 2 * STEPS, VSLOTS = 4 * MT, AHEAD = 3;
    auto step = [&](f32x16_t (&S)[2], f32x16_t (&N)[2], const uint8_t* kt, const uint8_t* vt, float& top) {
      u32x4_t f[AHEAD + 1];
      auto read = [&](int at) {  // the A operand of slot `at`
        f[at % (AHEAD + 1)] = at < KSLOTS ? read_key(kt, at / STEPS, at % STEPS)
                                          : read_value(vt, (at - KSLOTS) / MT, (at - KSLOTS) % MT);
      };
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) read(k);
      int done = 0;
#pragma unroll
      for (int k = 0; k < KSLOTS; ++k) {
        const int b = k / STEPS, s = k % STEPS;
        read(k + AHEAD);
        N[b] = mfma32x32x16<DT>(f[k % (AHEAD + 1)], qf[s], s == 0 ? (f32x16_t)(0.f) : N[b]);
#pragma unroll
        for (; done < (k + 1) * 8 / KSLOTS; ++done) weigh(S, 0, done);
        __builtin_amdgcn_sched_barrier(0);
      }
      done = 0;
      int seen = 0;
      top = -__builtin_inff();
#pragma unroll
      for (int k = 0; k < VSLOTS; ++k) {
        const int t = k / MT, m = k % MT;
        if (k + AHEAD < VSLOTS) read(KSLOTS + k + AHEAD);
        O[m] = mfma32x32x16<DT>(f[(KSLOTS + k) % (AHEAD + 1)], P[t], O[m]);
        if (k < VSLOTS / 2) {
#pragma unroll
          for (; done < (k + 1) * 8 / (VSLOTS / 2); ++done) weigh(S, 1, done);
        } else {
#pragma unroll
          for (; seen < (k + 1 - VSLOTS / 2) * 16 / (VSLOTS / 2); ++seen)
            top = fmaxf(fmaxf(top, N[seen >> 3][2 * (seen & 7)]), N[seen >> 3][2 * (seen & 7) + 1]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    // A value that is NaN or infinite must not reach the rows that do not see its
    // key, but their weight of zero times it is NaN; and a row that sees it must not
    // get NaN for an infinity because its weight rounds to zero.  Such results send
    // the block through its keys a second time: with APART the tiles are stripped of
    // these values, which keep their place in s_first: key j is seen by the rows from
    // j - shift on, so that the first key of each kind and channel decides.
    auto strip = [&](uint8_t* vt, int tile) {
      constexpr uint32_t kInf = DT::id == F16::id ? 0x7C00u : 0x7F80u;
      int at = 64 * wave + lane;
      asm volatile("" : "+v"(at));  // addresses are computed here, not kept through the products
#pragma unroll 1
      for (; at < VALUE_TILE / 16; at += 64 * kWaves) {
        const int r = at / CHUNKS, c = (at % CHUNKS) ^ value_swz(r);
        u32x4_t* place = reinterpret_cast<u32x4_t*>(vt) + at;
        u32x4_t w = *place;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t x = (w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
          if ((x & kInf) == kInf) {
            atomicMin(&s_first[(x & 0x7FFFu) > kInf ? 0 : 1 + (int)(x >> 15)][8 * c + e], tile * kKeys + r);
            w[e >> 1] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
          }
        }
        *place = w;
      }
    };

    // Keys run one tile ahead of the values: while tile j is weighed, S of tile
    // j + 1 is computed and the keys of j + 2 and the values of j + 1 are loaded.
    // After the wave's last tile S is computed from whatever LDS holds, and not used:
    // a second form of the step would cost the registers of a second O.
    f32x16_t Sa[2], Sb[2];
    float top;
    if constexpr (APART)
#pragma unroll 1
      for (int i = 64 * wave + lane; i < 3 * D; i += 64 * kWaves) s_first[0][i] = INT32_MAX;
    if (tiles > 0) {
      load_tile(kbase, p.k.token, key_off, 0, s_k0, KEY_GROUP);
      load_tile(vbase, p.v.token, value_off, 0, s_v0, 1024);
      if (tiles > 1) load_tile(kbase, p.k.token, key_off, 1, s_k1, KEY_GROUP);
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's shares are in LDS
      __syncthreads();
      if (my_tiles > 0) {
        top = -__builtin_inff();
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          Sa[b] = (f32x16_t)(0.f);
#pragma unroll
          for (int s = 0; s < STEPS; ++s) Sa[b] = mfma32x32x16<DT>(read_key(s_k0, b, s), qf[s], Sa[b]);
#pragma unroll
          for (int e = 0; e < 16; ++e) top = fmaxf(top, Sa[b][e]);
        }
        settle(Sa, top, 0);
      }
    }
    // k, v: where tile j is; v_next: the values' other slot
    auto turn = [&](int j, uint8_t* k, uint8_t* v, uint8_t* v_next) {
      __builtin_amdgcn_s_waitcnt(0x0f70);
      __syncthreads();
      if constexpr (APART) {
        strip(v, j);
        __syncthreads();
      }
      if (j + 2 < tiles) load_tile(kbase, p.k.token, key_off, j + 2, k, KEY_GROUP);
      if (j + 1 < tiles) load_tile(vbase, p.v.token, value_off, j + 1, v_next, 1024);
    };
    int j = 0;
    for (; j + 1 < my_tiles; j += 2) {
      turn(j, s_k0, s_v0, s_v1);
      step(Sa, Sb, s_k1, s_v0, top);
      settle(Sb, top, j + 1);
      turn(j + 1, s_k1, s_v1, s_v0);
      step(Sb, Sa, s_k0, s_v1, top);
      if (j + 2 < my_tiles) settle(Sa, top, j + 2);
    }
    if (j < my_tiles) {
      turn(j, s_k0, s_v0, s_v1);
      step(Sa, Sb, s_k1, s_v0, top);
      ++j;
    }
    for (; j < tiles; ++j)  // the other waves' tiles
      turn(j, (j & 1) ? s_k1 : s_k0, (j & 1) ? s_v1 : s_v0, (j & 1) ? s_v0 : s_v1);

    const float l = sum + __shfl_xor(sum, 32, 64);
    const int row = row0 + n;
    const float inv = l != 0.f ? 1.f / l : 0.f;  // a row that sees no key gives zeros
    float odd = 0.f;  // NaN if an accumulator is NaN or infinite
    uint16_t* o = p.out + ((sq.row0 + row) * p.heads + head) * D + 4 * half;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        u32x2_t w =
            u32x2_t{pack_results<DT>(O[m][e] * inv, O[m][e + 1] * inv),
                    pack_results<DT>(O[m][e + 2] * inv, O[m][e + 3] * inv)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          odd = fmaf(O[m][e + i], 0.f, odd);
          if constexpr (APART) {
            const int channel = 32 * m + 2 * e + 4 * half + i, seen = row + shift;
            const bool nan = s_first[0][channel] <= seen, up = s_first[1][channel] <= seen,
                       down = s_first[2][channel] <= seen;
            const bool finite = fabsf(O[m][e + i]) < __builtin_inff();
            float x = finite ? to_f32<DT>((uint16_t)(w[i >> 1] >> (16 * (i & 1)))) : O[m][e + i] * inv;
            if (up) x += __builtin_inff();
            if (down) x -= __builtin_inff();
            if (nan) x = __builtin_nanf("");
            if (!finite || nan || up || down)
              w[i >> 1] = i & 1 ? (w[i >> 1] & 0xFFFFu) | ((uint32_t)from_f32<DT>(x) << 16)
                                : (w[i >> 1] & 0xFFFF0000u) | from_f32<DT>(x);
          }
        }
        if (row < rows) *reinterpret_cast<u32x2_t*>(o + 32 * m + 2 * e) = w;
      }
    if (APART || tiles == 0) return 0;
    // A row's largest weight is 2^kRoom or more, where its exponent was right.
    const bool lost = l < 0.5f * (float)(1 << (int)kRoom<DT>) && row < rows && row + shift >= 0;
    int mine = 0;
    if (__any(odd != odd || lost)) mine = __any(lost || fabsf(M) > 0x1p24f && M != kLow) ? kApart | kFar : kApart;
    if (lane == 0) s_redo[wave] = mine;
    __syncthreads();
    int redo = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) redo |= s_redo[w];
    return redo;
  };
  const int redo = attend(std::false_type{}, threadIdx.x & 63, false);
  if (redo == 0) return;
  int none = 0;
  asm volatile("" : "+s"(index), "+s"(head), "+s"(none));  // nothing is kept from the first pass
  attend(std::true_type{}, __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, none)),
         (__builtin_amdgcn_readfirstlane(redo) & kFar) != 0);
}

}  // namespace

int launch_prompt_attention(const PromptParams& p, int dtype, hipStream_t st) {
  auto go = [&](auto kernel) -> int {
    // a partial block for every sequence and for the rows behind them, one for the rows in front
    const int64_t blocks = ((p.q_tokens + kBlockRows - 1) / kBlockRows + p.seqs + 1) * p.heads;
    if (blocks > INT32_MAX) return GRINQH_ERR_INVALID;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(64 * kWaves), 0, st, p);
    return hipGetLastError() == hipSuccess ? GRINQH_OK : GRINQH_ERR_HIP;
  };
  const bool bf16 = dtype == GRINQH_DTYPE_BF16;
  switch (p.head_size) {
    case 64: return bf16 ? go(prompt_attention_kernel<BF16, 64>) : go(prompt_attention_kernel<F16, 64>);
    case 128: return bf16 ? go(prompt_attention_kernel<BF16, 128>) : go(prompt_attention_kernel<F16, 128>);
    case 256: return bf16 ? go(prompt_attention_kernel<BF16, 256>) : go(prompt_attention_kernel<F16, 256>);
  }
  return GRINQH_ERR_INVALID;
}

}  // namespace grinqh
