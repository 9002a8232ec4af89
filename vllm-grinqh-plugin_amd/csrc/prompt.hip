// Attention over whole prompts: packed sequences, causal, grouped heads.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j),  j <= i + (keys - rows) of the sequence
//
// One pass over the keys with a running reference of the exponent.  S^T = K Q^T
// leaves a lane of v_mfma_f32_32x32x16 with one query row and 16 of 32 keys,
// which is the B operand of O^T = V^T P^T, so P never leaves its lane; keys
// and values go through LDS, the values read back transposed.
#include <type_traits>

#include "attention_launch.h"
#include "grinqh_common.h"

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

constexpr int kWaves = 4;
constexpr int kKeys = 64;       // keys per tile
constexpr float kLow = -1e30f;  // running reference before the first key (finite: -inf - -inf would be NaN)

// Sum over the wave, in every lane.
__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return v;
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
// holds the blocks whose last row sees about l * rows_per_block keys (at most one
// per sequence).  Returns the sequence, or -1 past the last block.
__device__ __forceinline__ int find_block(const PromptParams& p, int rows_per_block, int64_t index, int lane,
                                          Sequence& found, int64_t& block) {
  const int seqs = p.seqs + 1;
  // blocks of sequence s at level >= l: their indices b + before >= l
  auto count_of = [&](int s, int& blocks, int& before) {
    blocks = before = 0;
    if (s >= seqs) return;
    const Sequence q = sequence(p, s);
    blocks = (int)((q.rows + rows_per_block - 1) / rows_per_block);
    before = (int)(max(q.keys - q.rows, (int64_t)0) / rows_per_block);
  };
  int my_blocks, my_before, most = 0;
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
  for (int s = lane; s < seqs; s += 64) {
    int blocks = my_blocks, before = my_before;
    if (s >= 64) count_of(s, blocks, before);
    if (blocks > 0) most = max(most, blocks + before);
  }
  most = wave_max(most);
  if (index >= at_least(0)) return -1;
  int lo = 0, hi = most;  // at_least(lo) > index >= at_least(hi)
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
    // level 0 also holds every block below it (there are none: before >= 0)
    const int b = lo - before;
    const bool here = b >= 0 && b < blocks;
    const uint64_t mask = __ballot(here);
    const int n = __popcll(mask);
    if (rank < n) {
      uint64_t m = mask;
      for (int i = 0; i < (int)rank; ++i) m &= m - 1;
      const int s = s0 + __builtin_ctzll(m);
      found = sequence(p, s);
      block = lo - (int)(max(found.keys - found.rows, (int64_t)0) / rows_per_block);
      return s;
    }
    rank -= n;
  }
  return -1;
}

// Block = 4 waves x 32 * NQ query rows of one head.
template <typename DT, int D, int NQ>
__global__ __launch_bounds__(64 * kWaves, 1) void prompt_attention_kernel(const PromptParams p) {
  constexpr int ROWS = kWaves * 32 * NQ, STEPS = D / 16, MT = D / 32, CHUNKS = D / 8;
  constexpr int TILE = kKeys * D * 2;  // bytes of a tile of keys, or of values
  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 63, n = lane & 31, half = lane >> 5;
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
  Sequence sq;
  int64_t block;
  if (find_block(p, ROWS, index, lane, sq, block) < 0) return;
  const int kvh = head / (p.heads / p.kv_heads);
  const int row0 = (int)block * ROWS + wave * 32 * NQ;  // of this wave, in the sequence
  const int rows = (int)sq.rows, shift = (int)(sq.keys - sq.rows), keys = (int)sq.keys;
  // keys that the block's last row sees
  const int block_keys = min(keys, min((int)(block + 1) * ROWS, rows) + shift);
  const int tiles = block_keys > 0 ? (block_keys + kKeys - 1) / kKeys : 0;
  const int wave_keys = row0 < rows ? min(keys, min(row0 + 32 * NQ, rows) + shift) : 0;

  // queries: row n of each 32, channels 16 s + 8 half + e
  u32x4_t qf[NQ][STEPS];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int64_t row = sq.row0 + min(row0 + 32 * i + n, rows - 1);
    const uint16_t* q = p.q.p + row * p.q.token + (int64_t)head * p.q.head + 8 * half;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) qf[i][s] = *reinterpret_cast<const u32x4_t*>(q + 16 * s);
  }

  // LDS position of 16-byte chunk c of key r: c with bits flipped by the key, so
  // that the 8 keys (4 key rows x 2 for the transposed read) that are read
  // together lie in different banks
  auto swz = [](int r) { return ((r & 3) << 2 | (r >> 2 & 3)) & (CHUNKS - 1); };
  const uint16_t* kbase = p.k.p + sq.key0 * p.k.token + (int64_t)kvh * p.k.head;
  const uint16_t* vbase = p.v.p + sq.key0 * p.v.token + (int64_t)kvh * p.v.head;
  auto load_tile = [&](int tile, int slot) {
    const int k0 = tile * kKeys, live = min(kKeys, keys - k0);
    auto one = [&](const uint16_t* base, int64_t stride, uint8_t* to) {
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint16_t*>(base + (int64_t)k0 * stride), (short)0, (int)(((live - 1) * stride + D) * 2),
          0x00020000);
      constexpr int PER = 64 / CHUNKS;  // keys per load of a wave (1 KiB)
#pragma unroll
      for (int i = 0; i < kKeys / PER / kWaves; ++i) {
        const int r0 = (i * kWaves + wave) * PER, r = r0 + lane / CHUNKS;
        const int c = (lane % CHUNKS) ^ swz(r);
        const uint32_t off = r < live ? (uint32_t)(r * stride * 2 + c * 16) : 0xFFFFFFFFu;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_t)(to + r0 * D * 2), 16, (int)off, 0, 0, 0);
      }
    };
    one(kbase, p.k.token, smem + slot * 2 * TILE);
    one(vbase, p.v.token, smem + slot * 2 * TILE + TILE);
  };

  f32x16_t O[NQ][MT];
  float M[NQ], sum[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    M[i] = kLow;
    sum[i] = 0.f;
#pragma unroll
    for (int m = 0; m < MT; ++m) O[i][m] = (f32x16_t)(0.f);
  }
  const float c2 = p.scale * 1.44269504088896f;

  if (tiles > 0) load_tile(0, 0);
  for (int tile = 0; tile < tiles; ++tile) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's share of the tile is in LDS
    __syncthreads();
    if (tile + 1 < tiles) load_tile(tile + 1, (tile + 1) & 1);
    if (tile * kKeys >= wave_keys) continue;
    const uint8_t* kt = smem + (tile & 1) * 2 * TILE;
    const uint8_t* vt = kt + TILE;
    f32x16_t S[NQ][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int i = 0; i < NQ; ++i) S[i][b] = (f32x16_t)(0.f);
      const int r = 32 * b + n;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(kt + r * D * 2 + (((2 * s + half) ^ swz(r)) << 4));
#pragma unroll
        for (int i = 0; i < NQ; ++i) S[i][b] = mfma32x32x16<DT>(a, qf[i][s], S[i][b]);
      }
    }
    u32x4_t P[NQ][4];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int seen = row0 + 32 * i + n + shift - tile * kKeys;  // last key of this tile that the row sees
      if (tile * kKeys + kKeys - 1 > row0 + 32 * i + shift) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (32 * b + (e & 3) + 8 * (e >> 2) + 4 * half > seen) S[i][b][e] = -__builtin_inff();
      }
      float top = S[i][0][0];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, S[i][b][e]);
      if (__any(fmaf(top, c2, -M[i]) > 8.f)) {
        float m = fmaxf(M[i], top * c2);
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const float f = __builtin_amdgcn_exp2f(M[i] - m);
        M[i] = m;
        sum[i] *= f;
#pragma unroll
        for (int t = 0; t < MT; ++t) O[i][t] *= f;
      }
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(S[i][b][e], c2, -M[i]));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(S[i][b][e + 1], c2, -M[i]));
          sum[i] += p0 + p1;
          P[i][2 * b + (e >> 3)][(e & 7) >> 1] = pack2<DT>(p0, p1);
        }
    }
    // values, transposed: row (channel) n, keys 16 t + 4 half + 0..3 and + 8
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        u32x4_t a;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int r = 16 * t + 8 * u + 4 * half + ((lane & 15) >> 2);
          const int byte = 64 * m + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
          const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_s16x4_t)(vt + r * D * 2 + (((byte >> 4) ^ swz(r)) << 4) + (byte & 15)));
          const u32x2_t y = __builtin_bit_cast(u32x2_t, x);
          a[2 * u] = y[0];
          a[2 * u + 1] = y[1];
        }
#pragma unroll
        for (int i = 0; i < NQ; ++i) O[i][m] = mfma32x32x16<DT>(a, P[i][t], O[i][m]);
      }
  }

#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const float l = sum[i] + __shfl_xor(sum[i], 32, 64);
    const int row = row0 + 32 * i + n;
    if (row >= rows) continue;
    const float inv = l != 0.f ? 1.f / l : 0.f;  // a row that sees no key gives zeros
    uint16_t* o = p.out + ((sq.row0 + row) * p.heads + head) * D + 4 * half;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<u32x2_t*>(o + 32 * m + 2 * e) =
            u32x2_t{pack2<DT>(O[i][m][e] * inv, O[i][m][e + 1] * inv),
                    pack2<DT>(O[i][m][e + 2] * inv, O[i][m][e + 3] * inv)};
  }
}

}  // namespace

int launch_prompt_attention(const PromptParams& p, int dtype, hipStream_t st) {
  auto go = [&](auto dt, auto d, auto nq) -> int {
    constexpr int D = decltype(d)::value, NQ = decltype(nq)::value, ROWS = kWaves * 32 * NQ;
    auto kernel = prompt_attention_kernel<decltype(dt), D, NQ>;
    const int lds = 4 * kKeys * D * 2;
    const int64_t blocks = ((p.q_tokens + ROWS - 1) / ROWS + p.seqs) * p.heads;
    if (blocks > INT32_MAX) return GRINQH_ERR_INVALID;
    if (lds > 64 * 1024)
      if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds) !=
          hipSuccess)
        return GRINQH_ERR_HIP;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(64 * kWaves), lds, st, p);
    return hipGetLastError() == hipSuccess ? GRINQH_OK : GRINQH_ERR_HIP;
  };
  auto sized = [&](auto dt) -> int {
    switch (p.head_size) {
      case 64: return go(dt, std::integral_constant<int, 64>{}, std::integral_constant<int, 1>{});
      case 128: return go(dt, std::integral_constant<int, 128>{}, std::integral_constant<int, 1>{});
      case 256: return go(dt, std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{});
    }
    return GRINQH_ERR_INVALID;
  };
  return dtype == GRINQH_DTYPE_BF16 ? sized(BF16{}) : sized(F16{});
}

}  // namespace grinqh
