// Sparse attention's selection: the mean key of every page in 8 bits, and the
// pages whose mean keys promise a query the largest logits.
//
// Summary: int8 [pages][heads][D + 16], D codes, their fp32 step, 12 unused bytes.
// With m the mean of a page's keys and 2^E <= max |m| < 2^(E + 1): step = 2^(E - 6),
// code = round(m / step) within +-127; a page of zeros has step 0.  Queries get
// codes the same way, a step per head.  A page's score is the largest of its
// heads' products codes(q).codes(m), times both steps: whole numbers below 2^22
// times powers of two, so nothing is rounded and the selection does not depend on
// the order of any sum.  The means are sums in 64 bits that are exact too: what a code
// stands for is a multiple of 2^-24 below 2^17, and 4096 tokens of it fit 53 bits; longer
// pages' sums are rounded, in the order of the lanes, which is always the same.
//
// All are bound by latency: of a page's records (summaries: 32 tokens' pages 4.7 us, 4
// prompts of 2048 tokens 7.4 us, 0.8 TB/s), of the search for the last selected score.
// 64 sequences of 8192 tokens, pages of 16, 8 key/value heads of 128: 16 us, 38 MB of
// summaries; one of 131072 tokens, 9.4 MB: 5 us for the scores, 14 for the search.
#include <cfloat>
#include <type_traits>

#include "attention_launch.h"
#include "grinqh_common.h"
#include "wave_scan.h"

namespace grinqh {

namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float half_lo(uint32_t w) { return f16_bits_to_f32((uint16_t)w); }
__device__ __forceinline__ float half_hi(uint32_t w) { return f16_bits_to_f32((uint16_t)(w >> 16)); }

__device__ __forceinline__ double shfl_xor_f64(double v, int mask) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)b, mask, 64);
  const uint32_t hi = (uint32_t)__shfl_xor((int)(uint32_t)(b >> 32), mask, 64);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// ---------------------------------------------------------------- summaries

// A wave per page and head.  A lane has a quarter of a token's words per record (word
// (chunk % 4) * (D / 32) + chunk / 4, so quarter q has the chunks q + 4 i) and sums
// its D / 4 channels over the records; the 16 lanes of a quarter then add
// up, each keeping its share of the channels (half as many exchanged at every step).
template <int D>
__device__ __forceinline__ void summarize_page(const SummarizeParams& p, int64_t page, int head, int tokens, int lane) {
  constexpr int I = D / 32, N = 8 * I;
  const int groups = p.cache.groups, token = lane >> 2, quarter = lane & 3;
  const int record = kv4_record_bytes(D, groups);
  const uint8_t* base = p.cache.p + (page * p.cache.heads + head) * p.cache.sub * record;
  double sum[N], low[I];
#pragma unroll
  for (int i = 0; i < N; ++i) sum[i] = 0.;
#pragma unroll
  for (int i = 0; i < I; ++i) low[i] = 0.;
  for (int r = 0; 16 * r < tokens; ++r) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(base + (int64_t)r * record);
    uint32_t word[I], pair[I];
#pragma unroll
    for (int i = 0; i < I; i += 2) {
      const u32x2_t x = *reinterpret_cast<const u32x2_t*>(w + token * (D / 8) + quarter * I + i);
      word[i] = x[0];
      word[i + 1] = x[1];
    }
    const bool live = 16 * r + token < tokens;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      pair[i] = w[2 * D + i * groups / I * 16 + token];
      if (!live) pair[i] = 0;  // whatever the record holds behind the last token must not count
    }
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const double s = (double)half_lo(pair[i]);
      low[i] += (double)half_hi(pair[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int nib = 4 * (e / 2 + 4 * (e % 2));
        sum[8 * i + e] = fma(s, (double)((word[i] >> nib) & 15u), sum[8 * i + e]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) sum[i] += low[i / 8];
  // lane bits 5..2 pick the halves
#pragma unroll
  for (int step = 0; step < 4; ++step) {
    const int mask = 32 >> step, half = N >> (step + 1);
    const bool upper = lane & mask;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const double send = upper ? sum[i] : sum[i + half], keep = upper ? sum[i + half] : sum[i];
      sum[i] = keep + shfl_xor_f64(send, mask);
    }
  }
  constexpr int MINE = N / 16;
  const int first = (token & 8 ? N / 2 : 0) + (token & 4 ? N / 4 : 0) + (token & 2 ? N / 8 : 0) + (token & 1 ? N / 16 : 0);
  double mean[MINE];
  int top = 0;  // biased exponent of the largest
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    mean[i] = sum[i] / (double)tokens;
    if (!(fabs(mean[i]) < (double)FLT_MAX)) mean[i] = 0.;  // NaN keys
    top = max(top, (int)(__builtin_bit_cast(uint64_t, mean[i]) >> 52 & 0x7FF));
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = max(top, __shfl_xor(top, o, 64));
  const int exponent = top - 1023 - 6;
  int8_t* out = p.summary + (page * p.cache.heads + head) * summary_bytes(D);
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int c = top == 0 ? 0 : (int)fmin(fmax(rint(ldexp(mean[i], -exponent)), -127.), 127.);
    codes |= ((uint32_t)c & 0xFFu) << (8 * i);
  }
  const int channel = 8 * (quarter + 4 * (first / 8)) + first % 8;
  if constexpr (MINE == 1) out[channel] = (int8_t)codes;
  if constexpr (MINE == 2) *reinterpret_cast<uint16_t*>(out + channel) = (uint16_t)codes;
  if constexpr (MINE == 4) *reinterpret_cast<uint32_t*>(out + channel) = codes;
  if (lane == 0) *reinterpret_cast<float*>(out + D) = top == 0 ? 0.f : ldexpf(1.f, exponent);
}

// All waves look at all sequences, 64 at a time, and take the pages and heads in turn.
template <int D>
__global__ __launch_bounds__(256) void kv4_summarize_kernel(const SummarizeParams p) {
  const int lane = threadIdx.x & 63, shift = p.sub_shift + 4;
  const uint32_t waves = gridDim.x * 4;
  uint32_t next = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // of units: page, head
  uint32_t before = 0;
  const uint32_t heads = (uint32_t)p.cache.heads;
  for (int s0 = 0; s0 < p.seqs; s0 += 64) {
    const int s = s0 + lane;
    int length = 0, first = 0, pages = 0;
    if (s < p.seqs) {
      length = (int)min((int64_t)max(p.lengths[s], 0), (int64_t)p.table_width << shift);
      const int start = max(p.starts[s], 0);
      first = start >> shift;
      if (length > start) pages = (int)(((int64_t)length + (1 << shift) - 1) >> shift) - first;
    }
    const uint32_t upto = before + (uint32_t)wave_scan(pages) * heads;
    const uint32_t end = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    for (; next < end; next += waves) {
      const int owner = __builtin_ctzll(__ballot(upto > next));
      const uint32_t unit = next - (uint32_t)__builtin_amdgcn_readlane((int)(upto - (uint32_t)pages * heads), owner);
      const int place = __builtin_amdgcn_readlane(first, owner) + (int)(unit / heads);
      const int tokens = min(__builtin_amdgcn_readlane(length, owner) - (place << shift), 1 << shift);
      const int page = p.table[(int64_t)(s0 + owner) * p.table_stride + place];
      if ((uint32_t)page < (uint64_t)p.cache.pages) summarize_page<D>(p, page, (int)(unit % heads), tokens, lane);
    }
    before = end;
  }
}

// ---------------------------------------------------------------- scores

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kLeast = -(1 << 20);  // exponent of a head of zeros

// A query's value in fp32, limited to what is finite, NaN as 0.
template <typename DT>
__device__ __forceinline__ float query_value(uint16_t h) {
  const float x = to_f32<DT>(h);
  return x != x ? 0.f : fminf(fmaxf(x, -FLT_MAX), FLT_MAX);
}

// A sequence and key/value head.
struct Unit {
  int seq, head;
  int length, pages;  // limited to the table
  bool bad;           // the length is past the table
};
__device__ __forceinline__ Unit unit_of(const SelectParams& p, uint32_t id) {
  Unit u;
  u.seq = (int)(id / (uint32_t)p.kv_heads);
  u.head = (int)(id - (uint32_t)u.seq * (uint32_t)p.kv_heads);
  const int capacity = p.table_width << p.page_shift, held = max(p.lengths[u.seq], 0);
  u.bad = held > capacity;
  u.length = min(held, capacity);
  u.pages = (int)(((int64_t)u.length + (1 << p.page_shift) - 1) >> p.page_shift);
  return u;
}

// The codes and exponents of 16 query heads of a group, made once per block.
template <int D>
struct Queries {
  __align__(16) int8_t code[16][D];
  int exponent[16];
  int most;
};
// 32 threads per head.  Heads past the group's last stand for it.
template <typename DT, int D>
__device__ __forceinline__ int query_row(const SelectParams& p, const Unit& u, int tile, float (&x)[D / 32]) {
  constexpr int N = D / 32;
  const int per = p.heads / p.kv_heads, row = min(16 * tile + (int)threadIdx.x / 32, per - 1);
  const uint16_t* q = p.q.p + (int64_t)u.seq * p.q.token + (int64_t)(u.head * per + row) * p.q.head +
                      threadIdx.x % 32 * N;
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(q + i);
    x[i] = query_value<DT>((uint16_t)w);
    x[i + 1] = query_value<DT>((uint16_t)(w >> 16));
    top = fmaxf(top, fmaxf(fabsf(x[i]), fabsf(x[i + 1])));
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  return top > 0.f ? ilogbf(top) : kLeast;
}
template <int D>
__device__ __forceinline__ void store_query(Queries<D>& sh, const float (&x)[D / 32], int exponent) {
  constexpr int N = D / 32;
#pragma unroll
  for (int i = 0; i < N; ++i)
    sh.code[threadIdx.x / 32][threadIdx.x % 32 * N + i] =
        (int8_t)(int)fminf(fmaxf(rintf(ldexpf(x[i], 6 - max(exponent, -200))), -127.f), 127.f);
  if (threadIdx.x % 32 == 0) sh.exponent[threadIdx.x / 32] = exponent;
}

// Scores of the pages base .. end - 1 of a unit by the whole block, a wave 16 TILES
// at a time; put(place, score, first round).  Rows of the matrix products are query
// heads, columns pages, so that a lane ends up with 4 heads' products of one page.
template <typename DT, int D, int TILES, typename F>
__device__ __forceinline__ void score_pages(const SelectParams& p, const Unit& u, int base, int end, Queries<D>& sh,
                                            F&& put) {
  constexpr int J = D / 64, R = summary_bytes(D);
  const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = p.heads / p.kv_heads, tiles = (per + 15) / 16;
  const int32_t* table = p.table + (int64_t)u.seq * p.table_stride;
  float x[D / 32];
  int mine = query_row<DT, D>(p, u, 0, x);
  int most = kLeast;
  if (tiles > 1) {
    if (threadIdx.x == 0) sh.most = kLeast;
    __syncthreads();
    for (int t = 0; t < tiles; ++t) {
      float y[D / 32];
      const int e = query_row<DT, D>(p, u, t, y);
      if (threadIdx.x % 32 == 0) atomicMax(&sh.most, e);
    }
    __syncthreads();
    most = sh.most;
  }
  for (int tile = 0; tile < tiles; ++tile) {
    if (tile > 0) {
      mine = query_row<DT, D>(p, u, tile, x);
      __syncthreads();  // the codes before have been read
    }
    store_query<D>(sh, x, mine);
    bool ready = false;
    i32x4_t codes[J];
    float f[4];
    for (int at = base + wave * 16 * TILES; at < end || !ready; at += kWaves * 16 * TILES) {
      int index[TILES];
      i32x4_t means[TILES][J];
      float step[TILES];
      if (at < end) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) index[t] = table[min(at + 16 * t + n, u.pages - 1)];
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          const bool bad = (uint32_t)index[t] >= (uint64_t)p.pages;
          const int8_t* rec = p.summary + ((bad ? 0 : (int64_t)index[t]) * p.kv_heads + u.head) * R;
#pragma unroll
          for (int j = 0; j < J; ++j) means[t][j] = *reinterpret_cast<const i32x4_t*>(rec + 64 * j + 16 * quad);
          step[t] = *reinterpret_cast<const float*>(rec + D);
          if (bad) index[t] = -1;
        }
      }
      if (!ready) {  // after the loads have left
        ready = true;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < J; ++j) codes[j] = *reinterpret_cast<const i32x4_t*>(&sh.code[n][64 * j + 16 * quad]);
        if (tiles == 1) {
          most = sh.exponent[n];
#pragma unroll
          for (int o = 8; o >= 1; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = ldexpf(1.f, max(sh.exponent[4 * quad + i] - most, -40));
        if (at >= end) break;
      }
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        i32x4_t acc = i32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < J; ++j) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(codes[j], means[t][j], acc, 0, 0, 0);
        float best = fmaxf(fmaxf((float)acc[0] * f[0], (float)acc[1] * f[1]),
                           fmaxf((float)acc[2] * f[2], (float)acc[3] * f[3]));
        best = fmaxf(best, __shfl_xor(best, 16, 64));
        best = fmaxf(best, __shfl_xor(best, 32, 64));
        // a page outside the cache scores highest, and so does one whose summary was never made and holds
        // anything: scores are finite
        float score = best * step[t] + 0.f;  // -0 as 0
        if (index[t] < 0 || !(fabsf(score) <= FLT_MAX)) score = FLT_MAX;
        if (quad == 0 && at + 16 * t + n < end) put(at + 16 * t + n, score, tile == 0);
      }
    }
  }
}

// Wide tables: 256 pages per block, the scores to the workspace.
constexpr int kScorePages = 256;
template <typename DT, int D>
__global__ __launch_bounds__(kThreads) void kv4_score_kernel(const SelectParams p) {
  __shared__ Queries<D> sh;
  const uint32_t parts = (uint32_t)(p.table_width + kScorePages - 1) / kScorePages, id = blockIdx.x / parts;
  const int base = (int)(blockIdx.x - id * parts) * kScorePages;
  const Unit u = unit_of(p, id);
  if (u.pages <= p.count || base >= u.pages) return;  // all are selected
  float* out = p.scores + (int64_t)id * p.table_width;
  score_pages<DT, D, kScorePages / 16 / kWaves>(
      p, u, base, min(base + kScorePages, u.pages), sh,
      [&](int place, float score, bool first) { out[place] = first ? score : fmaxf(out[place], score); });
}

// ---------------------------------------------------------------- the largest scores

// The count - 2 highest scored of a block's pages beside those that are always
// selected (forced), equal ones from the front: put(page, place) in ascending order. A
// thread has PER adjacent pages, their scores in registers; PER == 0: any number, read
// again in every round.
//
// A histogram over the scores' range finds in which of 2048 parts the last selected one
// lies; of up to 64 in that part a wave finds it directly. More (equal scores, or
// one far from the rest) take it digit by digit, 11 bits of the scores' order as whole
// numbers at a time.
constexpr int kBins = 2048;
__device__ __forceinline__ uint32_t ordered(float score) {
  const uint32_t b = __float_as_uint(score);
  return b >> 31 ? ~b : b | 0x80000000u;
}
template <int THREADS>
struct TopShared {
  uint32_t bin[kBins];
  uint32_t wave[2][THREADS / 64];
  uint32_t range[2][2];
  uint32_t found[3];  // bin, number above it, number in it
  uint32_t some[64], number;
};
__device__ __forceinline__ float ordered_inverse(uint32_t k) {
  return __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~k);
}
template <int THREADS, int PER, typename K, typename F>
__device__ __forceinline__ void select_top(TopShared<THREADS>& sh, int count, int pages, int span, K&& score_at,
                                           F&& put) {
  constexpr int WAVES = THREADS / 64, BINS = kBins / THREADS;
  constexpr int kForced = 1 << 20, kNone = -1;  // instead of a part
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), first = tid * span;
  auto each = [&](auto&& f) __attribute__((always_inline)) {
    if constexpr (PER > 0) {
#pragma unroll
      for (int j = 0; j < PER; ++j) f(j);
    } else {
      for (int j = 0; j < span; ++j) f(j);
    }
  };
  auto special = [&](int j) {
    return first + j >= pages ? kNone : first + j == 0 || first + j == pages - 1 ? kForced : 0;
  };
  // minimum and maximum of the block's scores, as whole numbers
  auto range = [&](float low, float high, int round, uint32_t& lo, uint32_t& hi) __attribute__((always_inline)) {
    low = wave_reduce(low, [](float a, float b) { return fminf(a, b); });
    high = wave_reduce(high, [](float a, float b) { return fmaxf(a, b); });
    if (lane == 0) {
      atomicMin(&sh.range[round][0], ordered(low));
      atomicMax(&sh.range[round][1], ordered(high));
    }
    __syncthreads();
    lo = sh.range[round][0];
    hi = sh.range[round][1];
  };
  // the sum over the waves before this one
  auto waves_before = [&](const uint32_t* sums) {
    const uint32_t v = wave_scan(lane < WAVES ? sums[lane] : 0u);
    return wave == 0 ? 0u : (uint32_t)__builtin_amdgcn_readlane((int)v, wave - 1);
  };
  for (int i = tid; i < kBins; i += THREADS) sh.bin[i] = 0;
  if (tid == 0) {
    sh.number = 0;
    sh.range[0][0] = sh.range[1][0] = 0xFFFFFFFFu;
    sh.range[0][1] = sh.range[1][1] = 0;
  }
  __syncthreads();
  float low = FLT_MAX, high = -FLT_MAX;
  each([&](int j) {
    const bool in = special(j) == 0;
    low = in ? fminf(low, score_at(j)) : low;
    high = in ? fmaxf(high, score_at(j)) : high;
  });
  uint32_t lo, hi;
  range(low, high, 0, lo, hi);
  low = ordered_inverse(lo);
  high = ordered_inverse(hi);
  uint32_t need = (uint32_t)(count - 2);  // still to be found among those of part `at`
  // After the threads have counted into the bins: the one with the need-th from the top; the bins are cleared.
  auto find_bin = [&]() __attribute__((always_inline)) {
    __syncthreads();
    uint32_t bin[BINS], sum = 0;  // this thread's bins from the top
#pragma unroll
    for (int i = 0; i < BINS; ++i) {
      const int at = kBins - 1 - (tid * BINS + i);
      sum += bin[i] = sh.bin[at];
      sh.bin[at] = 0;
    }
    const uint32_t inside = wave_scan(sum);
    if (lane == 63) sh.wave[0][wave] = inside;
    __syncthreads();
    uint32_t over = inside - sum + waves_before(sh.wave[0]);
#pragma unroll
    for (int i = 0; i < BINS; ++i) {
      if (over < need && over + bin[i] >= need) {
        sh.found[0] = kBins - 1 - (tid * BINS + i);
        sh.found[1] = over;
        sh.found[2] = bin[i];
      }
      over += bin[i];
    }
    __syncthreads();
    need -= sh.found[1];
  };
  const float width = high - low, inv = (float)(kBins - 1) / width;
  const bool parts = need > 0 && width > 0.f && width <= FLT_MAX && inv <= FLT_MAX;
  // rounding keeps the order, so that a part's scores are all between its neighbours'
  auto part_now = [&](int j) {
    const int s = special(j);
    return s != 0 || !parts ? s : min((int)((score_at(j) - low) * inv), kBins - 1);
  };
  int kept[PER > 0 ? PER : 1];
  if constexpr (PER > 0) {
#pragma unroll
    for (int j = 0; j < PER; ++j) kept[j] = part_now(j);
  }
  auto part = [&](int j) { return PER > 0 ? kept[PER > 0 ? j : 0] : part_now(j); };
  int at = 0;
  bool many = need > 0;  // more than a wave finds at once
  uint32_t bar = 0;      // of part `at`: those above it, and the first `need` equal to it
  if (parts) {
    each([&](int j) {
      const int b = part(j);
      if (b >= 0 && b < kBins) atomicAdd(&sh.bin[b], 1u);
    });
    find_bin();
    at = (int)sh.found[0];
    const int number = (int)sh.found[2];
    many = number > 64;
    if (!many) {
      each([&](int j) {
        if (part(j) == at) sh.some[atomicAdd(&sh.number, 1u)] = ordered(score_at(j));
      });
      __syncthreads();
      // every wave by itself
      const uint32_t k = lane < number ? sh.some[lane] : 0;
      uint32_t above = 0, equal = 0;
      for (int i = 0; i < number; ++i) {
        const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)k, i);
        above += other > k;
        equal += other == k;
      }
      const int owner = __builtin_ctzll(__ballot(lane < number && above < need && above + equal >= need));
      bar = (uint32_t)__builtin_amdgcn_readlane((int)k, owner);
      need -= (uint32_t)__builtin_amdgcn_readlane((int)above, owner);
    }
  }
  if (many) {
    float least = FLT_MAX, most = -FLT_MAX;  // not low and high, which the parts are reckoned from
    each([&](int j) {
      if (part(j) != at) return;
      least = fminf(least, score_at(j));
      most = fmaxf(most, score_at(j));
    });
    range(least, most, 1, lo, hi);
    while (lo < hi) {
      const int shift = max(32 - __builtin_clz(hi - lo) - 11, 0);
      each([&](int j) {
        if (part(j) != at) return;
        const uint32_t k = ordered(score_at(j));
        if (k >= lo && k <= hi) atomicAdd(&sh.bin[(k - lo) >> shift], 1u);
      });
      find_bin();
      lo += sh.found[0] << shift;
      hi = min(hi, lo + ((1u << shift) - 1));
    }
    bar = lo;
  }
  // selected for sure, and as far as `need` reaches
  const bool middle = count > 2;
  auto sure_now = [&](int j) {
    const int b = part(j);
    return b == kForced || (middle && (b > at || (b == at && ordered(score_at(j)) > bar)));
  };
  auto level_now = [&](int j) { return middle && part(j) == at && ordered(score_at(j)) == bar; };
  uint32_t sures = 0, levels = 0;  // a bit for each of PER pages
  uint32_t mine = 0, equal = 0;
  each([&](int j) {
    const bool s = sure_now(j), l = level_now(j);
    mine += s;
    equal += l;
    sures |= (uint32_t)s << (j & 31);
    levels |= (uint32_t)l << (j & 31);
  });
  const uint32_t upto = wave_scan(mine), upto_equal = wave_scan(equal);
  __syncthreads();
  if (lane == 63) {
    sh.wave[0][wave] = upto;
    sh.wave[1][wave] = upto_equal;
  }
  __syncthreads();
  uint32_t above = upto - mine + waves_before(sh.wave[0]), before = upto_equal - equal + waves_before(sh.wave[1]);
  each([&](int j) {
    const bool s = PER > 0 ? sures >> (j & 31) & 1 : sure_now(j), l = PER > 0 ? levels >> (j & 31) & 1 : level_now(j);
    if (s || (l && before < need)) put(j, (int)(above + min(before, need)));
    above += s;
    before += l;
  });
}

// What is known without scores.  True: nothing is left to do.
__device__ __forceinline__ bool select_all(const SelectParams& p, const Unit& u, int32_t* out, int threads) {
  const int32_t* table = p.table + (int64_t)u.seq * p.table_stride;
  if (u.head == 0 && threadIdx.x == 0)  // a length past the table stays one
    p.new_lengths[u.seq] = u.bad ? INT32_MAX
                                 : u.pages > p.count ? u.length - ((u.pages - p.count) << p.page_shift) : u.length;
  if (u.pages > p.count) return false;
  for (int i = threadIdx.x; i < p.count; i += threads) out[i] = i < u.pages ? table[i] : -1;
  return true;
}

// A block per sequence and key/value head; scores from the workspace.
template <int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void kv4_top_kernel(const SelectParams p) {
  __shared__ TopShared<THREADS> sh;
  const Unit u = unit_of(p, blockIdx.x);
  int32_t* out = p.selected + (int64_t)blockIdx.x * p.count;
  if (select_all(p, u, out, THREADS)) return;
  const int32_t* table = p.table + (int64_t)u.seq * p.table_stride;
  const float* scores = p.scores + (int64_t)blockIdx.x * p.table_width;
  const int span = PER > 0 ? PER : (u.pages + THREADS - 1) / THREADS, first = threadIdx.x * span;
  float mine[PER > 0 ? PER : 1];
  int index[PER > 0 ? PER : 1];  // loaded here, all at once
  if constexpr (PER > 0) {
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      mine[j] = scores[min(first + j, u.pages - 1)];
      index[j] = table[min(first + j, u.pages - 1)];
    }
  }
  select_top<THREADS, PER>(
      sh, p.count, u.pages, span, [&](int j) { return PER > 0 ? mine[PER > 0 ? j : 0] : scores[first + j]; },
      [&](int j, int place) { out[place] = PER > 0 ? index[PER > 0 ? j : 0] : table[first + j]; });
}

// Both in one launch, up to 1024 pages. As two (1, 8, 64 sequences, 8 key/value heads of
// 128, us): 512 pages 8.1, 8.2, 16.0 in one and 8.7, 9.0, 19.8 in two; 1024: 10.9, 11.1, 26
// and 8.8, 9.3, 30; 2047: 17.2, 18.7, 47 and 9.2, 11.4, 38. The second of the two has 2, 8 or any
// number of pages per thread (2047 pages with 8: 12.8, 15.0, 44).
constexpr int kSelectPages = 1024;
template <typename DT, int D>
__global__ __launch_bounds__(kThreads, 4) void kv4_select_kernel(const SelectParams p) {
  constexpr int PER = kSelectPages / kThreads;
  __shared__ __align__(16) float s_score[kSelectPages];
  __shared__ Queries<D> s_query;
  __shared__ TopShared<kThreads> sh;
  const Unit u = unit_of(p, blockIdx.x);
  int32_t* out = p.selected + (int64_t)blockIdx.x * p.count;
  if (select_all(p, u, out, kThreads)) return;
  const int32_t* table = p.table + (int64_t)u.seq * p.table_stride;
  const int first = threadIdx.x * PER;
  int index[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) index[j] = table[min(first + j, u.pages - 1)];
  score_pages<DT, D, (D > 128 ? 2 : 4)>(p, u, 0, u.pages, s_query, [&](int place, float score, bool first) {
    s_score[place] = first ? score : fmaxf(s_score[place], score);
  });
  __syncthreads();
  float mine[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) mine[j] = s_score[min(first + j, u.pages - 1)];
  select_top<kThreads, PER>(sh, p.count, u.pages, PER, [&](int j) { return mine[j]; },
                            [&](int j, int place) { out[place] = index[j]; });
}

int status() { return hipGetLastError() == hipSuccess ? GRINQH_OK : GRINQH_ERR_HIP; }

}  // namespace

int launch_kv4_summarize(const SummarizeParams& p, hipStream_t st) {
  // a wave per page and head of the whole table, but at most 16 per CU: the rest are taken in turn
  const int64_t units = (int64_t)p.seqs * p.table_width * p.cache.heads;
  const uint32_t blocks = (uint32_t)((units < 4096 ? units : 4096) + 3) / 4;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, st, p);
    return status();
  };
  switch (p.cache.head_size) {
    case 64: return go(kv4_summarize_kernel<64>);
    case 128: return go(kv4_summarize_kernel<128>);
    case 256: return go(kv4_summarize_kernel<256>);
  }
  return GRINQH_ERR_INVALID;
}

bool kv4_select_fits(int table_width) { return table_width <= kSelectPages; }

int launch_kv4_select(const SelectParams& p, int dtype, hipStream_t st) {
  const int64_t heads = (int64_t)p.seqs * p.kv_heads;
  const dim3 units((uint32_t)heads);
  const bool bf16 = dtype == GRINQH_DTYPE_BF16;
  auto sized = [&](auto&& go) {
    switch (p.head_size) {
      case 64: go(std::integral_constant<int, 64>{}); break;
      case 128: go(std::integral_constant<int, 128>{}); break;
      case 256: go(std::integral_constant<int, 256>{}); break;
    }
    return status();
  };
  if (kv4_select_fits(p.table_width))
    return sized([&](auto d) {
      constexpr int D = decltype(d)::value;
      auto kernel = bf16 ? kv4_select_kernel<BF16, D> : kv4_select_kernel<F16, D>;
      hipLaunchKernelGGL(kernel, units, dim3(kThreads), 0, st, p);
    });
  if (p.table_width > p.count) {  // otherwise all pages are selected
    const int64_t blocks = heads * ((p.table_width + kScorePages - 1) / kScorePages);
    if (blocks > INT32_MAX) return GRINQH_ERR_INVALID;
    const int s = sized([&](auto d) {
      constexpr int D = decltype(d)::value;
      auto kernel = bf16 ? kv4_score_kernel<BF16, D> : kv4_score_kernel<F16, D>;
      hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(kThreads), 0, st, p);
    });
    if (s != GRINQH_OK) return s;
  }
  if (p.table_width <= 2048)
    hipLaunchKernelGGL((kv4_top_kernel<1024, 2>), units, dim3(1024), 0, st, p);
  else if (p.table_width <= 8192)
    hipLaunchKernelGGL((kv4_top_kernel<1024, 8>), units, dim3(1024), 0, st, p);
  else
    hipLaunchKernelGGL((kv4_top_kernel<1024, 0>), units, dim3(1024), 0, st, p);
  return status();
}

}  // namespace grinqh
