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
#include <type_traits>

#include "attention_launch.h"
#include "grinqh_common.h"

namespace grinqh {

namespace {

constexpr float kLimit = 65504.f;  // largest finite fp16

__device__ __forceinline__ uint32_t f16_pair(float lo, float hi) {
  return (uint32_t)f32_to_f16_bits(lo) | ((uint32_t)f32_to_f16_bits(hi) << 16);
}
__device__ __forceinline__ float half_lo(uint32_t w) { return f16_bits_to_f32((uint16_t)w); }
__device__ __forceinline__ float half_hi(uint32_t w) { return f16_bits_to_f32((uint16_t)(w >> 16)); }

// ---------------------------------------------------------------- store, load

// Codes and (scale, minimum) of one lane's 8 channels; the WIDTH adjacent lanes
// of a group share the parameters.  A NaN becomes +inf in the maximum, which
// no finite input reaches, and makes the group's parameters NaN.
template <typename DT, int WIDTH>
__device__ __forceinline__ uint32_t quantize8(const u32x4_t& in, uint32_t& params) {
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = to_f32<DT>((uint16_t)(in[e >> 1] >> (16 * (e & 1))));
  bool nan = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    nan = nan || x[e] != x[e];
    x[e] = fminf(fmaxf(x[e], -kLimit), kLimit);
  }
  float mn = x[0], mx = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    mn = fminf(mn, x[e]);
    mx = fmaxf(mx, x[e]);
  }
  if (nan) mx = __builtin_inff();
#pragma unroll
  for (int o = 1; o < WIDTH; o <<= 1) {
    mn = fminf(mn, __shfl_xor(mn, o, 64));
    mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  }
  if (mx > kLimit) {
    params = 0x7E007E00u;  // NaN, NaN
    return 0;
  }
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
    out[p] = (uint32_t)from_f32<DT>(a) | ((uint32_t)from_f32<DT>(b) << 16);
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

constexpr int kWaves = 4;       // per block
constexpr int kRows = 16;       // query heads of one key/value head per block
constexpr float kLow = -1e30f;  // running reference before the first token (finite: -inf - -inf would be NaN)

// What one wave holds of 32 tokens (two records).
template <int D, int G>
struct Tokens {
  uint32_t k[2][D / 32];
  u32x4_t kp[2][G];
  u32x4_t v[2][D < 128 ? 1 : D / 128];
  u32x4_t vp[2];
};

template <int D, int G>
__device__ __forceinline__ void load_tokens(Tokens<D, G>& t, int r, const uint8_t* __restrict__ rec, int lane) {
  const int n = lane & 15, quad = lane >> 4;
  constexpr int W = D / 32;
  const uint8_t* kb = rec + n * (D / 2) + quad * (D / 8);
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
#pragma unroll
  for (int g = 0; g < G; ++g) t.kp[r][g] = *reinterpret_cast<const u32x4_t*>(rec + 8 * D + 64 * g + 16 * quad);
  const uint8_t* vb = rec + 8 * D + 64 * G;
  if constexpr (D < 128) {
    t.v[r][0] = *reinterpret_cast<const u32x4_t*>(vb + (n & 7) * 64 + 16 * quad);
  } else {
#pragma unroll
    for (int i = 0; i < D / 128; ++i)
      t.v[r][i] = *reinterpret_cast<const u32x4_t*>(vb + (n + 16 * i) * 64 + 16 * quad);
  }
  t.vp[r] = *reinterpret_cast<const u32x4_t*>(rec + 16 * D + 64 * G + 16 * quad);
}

// Block = one sequence, one key/value head (up to 16 of its query heads) and
// one run of tokens; its waves take 32-token steps in turn, each with a softmax
// of its own, joined at the end (and with other blocks' by kv4_join_kernel).
//
// S^T = K Q^T leaves a lane with one query row and 8 of the 32 tokens, which
// is the B operand of O^T = V^T P^T: nothing crosses lanes in the loop.  With
// value = m + s c:  o = sum_t (p_t s_t) c_t + sum_t p_t m_t, so P carries the
// value scale and the minimum is one sum per row.
//
// The exponent's reference M is raised only when a weight p s passes 2^8
// (checked for all lanes at once), so the accumulators are rarely rescaled;
// M includes the value scale, which keeps the fp16 weights in range whatever
// the values' size.  Queries are brought to 2^13 <= max < 2^14 by a power of two
// (exact), so fp16 holds them for both types and the nibbles that come out
// 16-fold can be undone on the query's side.
template <typename DT, int D, int G>
__global__ __launch_bounds__(64 * kWaves) void kv4_attention_kernel(const Kv4Params p) {
  constexpr int R = kv4_record_bytes(D, G), W = D / 32, M_TILES = D < 128 ? 1 : D / 128, SLOTS = D < 128 ? 4 : 8;
  __shared__ float s_o[kWaves][kRows][D + 4];
  __shared__ float s_m[kWaves][kRows], s_l[kWaves][kRows], s_off[kWaves][kRows];
  const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = p.heads / p.cache.heads, tiles = (per + kRows - 1) / kRows;
  int id = blockIdx.x;
  const int split = id % p.plan.splits;
  id /= p.plan.splits;
  const int tile = id % tiles;
  id /= tiles;
  const int kvh = id % p.cache.heads, seq = id / p.cache.heads;
  const int h0 = kvh * per + tile * kRows, rows = min(kRows, per - tile * kRows);

  const int64_t capacity = (int64_t)p.table_width * p.cache.sub * 16;
  int length = max(p.lengths[seq], 0);
  bool bad = (int64_t)length > capacity;
  if (bad) length = (int)capacity;
  const int steps = (length + 31) >> 5;
  const int first = split * p.plan.chunk;
  const int last = split + 1 == p.plan.splits ? steps : min(steps, first + p.plan.chunk);
  if (split > 0 && first >= steps) return;

  // queries: row n, channels 32 s + 8 quad + e
  u32x4_t qf[W];
  float qsum[G], qs;
  {
    const uint16_t* q = p.q.p + (int64_t)seq * p.q.token + (int64_t)(h0 + min(n, rows - 1)) * p.q.head;
    float x[W][8];
    float mx = 0.f;
#pragma unroll
    for (int s = 0; s < W; ++s) {
      const u32x4_t in = *reinterpret_cast<const u32x4_t*>(q + 32 * s + 8 * quad);
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
    qs = ldexpf(p.scale * 1.44269504088896f, 24 - ex);  // logits in powers of two
  }

  f32x4_t O[M_TILES][SLOTS];
#pragma unroll
  for (int i = 0; i < M_TILES; ++i)
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) O[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float M = kLow, L = 0.f, off = 0.f;

  const int32_t* table = p.table + (int64_t)seq * p.table_stride;
  const int last_rec = max((length - 1) >> 4, 0);
  auto record = [&](int step, int r) -> const uint8_t* {
    const int rec = min(2 * step + r, last_rec);
    int page = table[rec / p.cache.sub];
    if ((uint32_t)page >= (uint64_t)p.cache.pages) {
      bad = true;
      page = 0;
    }
    return p.cache.p + (((int64_t)page * p.cache.heads + kvh) * p.cache.sub + (rec & (p.cache.sub - 1))) * R;
  };

  for (int step = first + wave; step < last; step += kWaves) {
    Tokens<D, G> t;
    load_tokens<D, G>(t, 0, record(step, 0), lane);
    load_tokens<D, G>(t, 1, record(step, 1), lane);

    float z[8], vs[8], vm[8];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        z[4 * r + i] = 0.f;
        vs[4 * r + i] = half_lo(t.vp[r][i]);
        vm[4 * r + i] = half_hi(t.vp[r][i]);
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = g * (W / G); s < (g + 1) * (W / G); ++s) {
          const uint32_t w = t.k[r][s], u = w >> 8;
          const u32x4_t a = u32x4_t{w & 0x000F000Fu, w & 0x00F000F0u, u & 0x000F000Fu, u & 0x00F000F0u};
          acc = mfma16x16x32<F16>(a, qf[s], acc);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          z[4 * r + i] += fmaf(acc[i], half_lo(t.kp[r][g][i]), half_hi(t.kp[r][g][i]) * qsum[g]);
      }
    }
    if (32 * step + 32 > length) {  // tokens past the end: whatever the record holds must not count
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (32 * step + 16 * (e >> 2) + 4 * quad + (e & 3) >= length) {
          z[e] = -__builtin_inff();
          vs[e] = 0.f;
          vm[e] = 0.f;
        }
    }
    float pe[8], pw[8];
    auto weights = [&]() {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pe[e] = __builtin_amdgcn_exp2f(fmaf(z[e], qs, -M));
        pw[e] = pe[e] * vs[e];
      }
    };
    weights();
    float top = 0.f, top_e = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      top = fmaxf(top, pw[e]);
      top_e = fmaxf(top_e, pe[e]);
    }
    if (__any(top > 256.f || top_e > 0x1p60f)) {
      float m = M;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, fmaf(z[e], qs, __log2f(fmaxf(vs[e], 0x1p-24f))));
      m = fmaxf(m, __shfl_xor(m, 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float f = __builtin_amdgcn_exp2f(M - m);
      M = m;
      L *= f;
      off *= f;
#pragma unroll
      for (int i = 0; i < M_TILES; ++i)
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) O[i][j] *= f;
      weights();
    }
    u32x4_t pf;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      L += pe[e];
      off = fmaf(pe[e], vm[e], off);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) pf[i] = f16_pair(pw[2 * i], pw[2 * i + 1]);

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
    for (int j = 0; j < SLOTS; ++j)
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
        s_o[wave][n][channel] = O[mt][j][i] * unit;
      }
  __syncthreads();
  for (int at = threadIdx.x; at < rows * D; at += 64 * kWaves) {
    const int row = at / D, d = at % D;
    float m = s_m[0][row];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s_m[w][row]);
    float sum = 0.f, val = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(s_m[w][row] - m);
      sum = fmaf(f, s_l[w][row], sum);
      val = fmaf(f, s_o[w][row][d] + s_off[w][row], val);
    }
    const int64_t out_row = (int64_t)seq * p.heads + h0 + row;
    if (p.plan.splits == 1) {
      p.out[out_row * D + d] = from_f32<DT>(length > 0 || sum != sum ? val / sum : 0.f);
    } else {
      float* to = p.partial + (out_row * p.plan.splits + split) * (D + 2);
      to[d] = val;
      if (d == 0) {
        to[D] = m;
        to[D + 1] = sum;
      }
    }
  }
}

// Joins the runs of one query row: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.
template <typename DT, int D>
__global__ __launch_bounds__(D) void kv4_join_kernel(const Kv4Params p) {
  const int64_t row = blockIdx.x;
  const int seq = (int)(row / p.heads), d = threadIdx.x;
  const int64_t capacity = (int64_t)p.table_width * p.cache.sub * 16;
  const int64_t length = min((int64_t)max(p.lengths[seq], 0), capacity);
  const int steps = (int)((length + 31) >> 5);
  const int runs = max(1, min(p.plan.splits, (steps + p.plan.chunk - 1) / p.plan.chunk));
  const float* part = p.partial + row * p.plan.splits * (D + 2);
  float m = kLow;
  for (int i = 0; i < runs; ++i) m = fmaxf(m, part[(int64_t)i * (D + 2) + D]);
  float sum = 0.f, val = 0.f;
  for (int i = 0; i < runs; ++i) {
    const float* x = part + (int64_t)i * (D + 2);
    const float f = __builtin_amdgcn_exp2f(x[D] - m);
    sum = fmaf(f, x[D + 1], sum);
    val = fmaf(f, x[d], val);
  }
  p.out[row * D + d] = from_f32<DT>(length > 0 || sum != sum ? val / sum : 0.f);
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

Kv4Plan plan_kv4(int64_t seqs, int heads, int kv_heads, int head_size, int64_t max_length) {
  constexpr int64_t kBlocks = 1024;
  const int64_t steps = max_length > 32 ? (max_length + 31) / 32 : 1;
  const int64_t base = seqs * kv_heads * ((heads / kv_heads + kRows - 1) / kRows);
  int64_t want = kBlocks / (base < 1 ? 1 : base);
  want = want < 1 ? 1 : want;
  int64_t chunk = (steps + want - 1) / want;
  chunk = (chunk + kWaves - 1) / kWaves * kWaves;
  Kv4Plan plan;
  plan.chunk = (int)chunk;
  plan.splits = (int)((steps + chunk - 1) / chunk);
  plan.workspace = plan.splits > 1 ? (size_t)seqs * heads * plan.splits * (head_size + 2) * sizeof(float) : 0;
  return plan;
}

int launch_kv4_attention(const Kv4Params& p, int dtype, hipStream_t st) {
  return dispatch_layout(dtype, p.cache.head_size, p.cache.groups, [&](auto dt, auto d, auto g) -> int {
    constexpr int D = decltype(d)::value;
    using DT = decltype(dt);
    const int tiles = (p.heads / p.cache.heads + kRows - 1) / kRows;
    const int64_t blocks = (int64_t)p.seqs * p.cache.heads * tiles * p.plan.splits;
    if (blocks > INT32_MAX || (int64_t)p.seqs * p.heads > INT32_MAX) return GRINQH_ERR_INVALID;
    hipLaunchKernelGGL((kv4_attention_kernel<DT, D, decltype(g)::value>), dim3((uint32_t)blocks), dim3(64 * kWaves), 0,
                       st, p);
    if (p.plan.splits > 1)
      hipLaunchKernelGGL((kv4_join_kernel<DT, D>), dim3((uint32_t)(p.seqs * p.heads)), dim3(D), 0, st, p);
    return status();
  });
}

}  // namespace grinqh
