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
// stands for is a multiple of 2^-24 below 2^17, and 4096 tokens of it fit 53 bits.
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

constexpr int kLeast = -(1 << 20);  // exponent of a head of zeros

// A row of a query in fp32, limited to what is finite, NaN as 0.
template <typename DT>
__device__ __forceinline__ float query_value(uint16_t h) {
  const float x = to_f32<DT>(h);
  return x != x ? 0.f : fminf(fmaxf(x, -FLT_MAX), FLT_MAX);
}

// A wave: 64 pages of one sequence and key/value head, 16 at a time.  Rows of the
// matrix products are query heads, columns pages, so that a lane ends up
// with 4 heads' products of one page.
constexpr int kScorePages = 64;
template <typename DT, int D>
__global__ __launch_bounds__(256) void kv4_score_kernel(const SelectParams p) {
  constexpr int J = D / 64, R = summary_bytes(D), TILES = kScorePages / 16;
  const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
  const int parts = (p.table_width + kScorePages - 1) / kScorePages;
  const int64_t unit = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t sh = unit / parts;
  const int base = (int)(unit - sh * parts) * kScorePages;
  const int seq = (int)(sh / p.kv_heads), head = (int)(sh - (int64_t)seq * p.kv_heads);
  if (seq >= p.seqs) return;
  const int64_t length = min((int64_t)max(p.lengths[seq], 0), (int64_t)p.table_width << p.page_shift);
  const int pages = (int)((length + (1 << p.page_shift) - 1) >> p.page_shift);
  if (pages <= p.count || base >= pages) return;  // all are selected
  const int per = p.heads / p.kv_heads;

  // the pages' codes: their loads leave before the queries are looked at
  int index[TILES];
  i32x4_t means[TILES][J];
  float step[TILES];
  const int32_t* table = p.table + (int64_t)seq * p.table_stride;
#pragma unroll
  for (int t = 0; t < TILES; ++t) index[t] = table[min(base + 16 * t + n, pages - 1)];
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const bool bad = (uint32_t)index[t] >= (uint64_t)p.pages;
    const int8_t* rec = p.summary + ((bad ? 0 : (int64_t)index[t]) * p.kv_heads + head) * R;
#pragma unroll
    for (int j = 0; j < J; ++j) means[t][j] = *reinterpret_cast<const i32x4_t*>(rec + 64 * j + 16 * quad);
    step[t] = *reinterpret_cast<const float*>(rec + D);
    if (bad) index[t] = -1;
  }
  auto row_of = [&](int tile) {
    return p.q.p + (int64_t)seq * p.q.token + (int64_t)(head * per + min(16 * tile + n, per - 1)) * p.q.head + 16 * quad;
  };
  float x[J][16];
  auto load_row = [&](int tile) -> int {  // returns the row's exponent
    const uint16_t* q = row_of(tile);
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(q + 64 * j + 8 * h);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[j][8 * h + e] = query_value<DT>((uint16_t)(w[e >> 1] >> (16 * (e & 1))));
          top = fmaxf(top, fabsf(x[j][8 * h + e]));
        }
      }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    return top > 0.f ? ilogbf(top) : kLeast;
  };
  const int tiles = (per + 15) / 16;
  int most = kLeast, mine = 0;
  for (int t = tiles - 1; t >= 0; --t) {
    mine = load_row(t);
    most = max(most, mine);
  }
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
  float best[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) best[t] = -__builtin_inff();
  for (int tile = 0;;) {
    i32x4_t codes[J];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t c = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = fminf(fmaxf(rintf(ldexpf(x[j][4 * w + e], 6 - max(mine, -200))), -127.f), 127.f);
          c |= ((uint32_t)(int)v & 0xFFu) << (8 * e);
        }
        codes[j][w] = (int)c;
      }
    const float factor = ldexpf(1.f, max(mine - most, -40));
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __shfl(factor, 4 * quad + i, 64);
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      i32x4_t acc = i32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < J; ++j) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(codes[j], means[t][j], acc, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) best[t] = fmaxf(best[t], (float)acc[i] * f[i]);
    }
    if (++tile >= tiles) break;
    mine = load_row(tile);
  }
  float* out = p.scores + sh * p.table_width + base;
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    best[t] = fmaxf(best[t], __shfl_xor(best[t], 16, 64));
    best[t] = fmaxf(best[t], __shfl_xor(best[t], 32, 64));
    const float score = index[t] < 0 ? __builtin_inff() : best[t] * step[t];
    if (quad == 0 && base + 16 * t + n < pages) out[16 * t + n] = score;
  }
}

// ---------------------------------------------------------------- the largest scores

// A block per sequence and key/value head.  The count - 2 largest scores between
// the first page and the last are found digit by digit, 11 bits at a time: a histogram
// of what is left of the range, and the digit in which the last selected one lies.
// The range starts from the smallest and the largest score, so that the first
// histogram already spreads (digits of the plain numbers would put nearly all
// scores into a few places, one after the other).  KEYS > 0: scores are kept in LDS.
constexpr int kBins = 2048;
template <int THREADS, int KEYS>
__global__ __launch_bounds__(THREADS) void kv4_top_kernel(const SelectParams p) {
  constexpr int WAVES = THREADS / 64, PER = kBins / THREADS;
  __shared__ uint32_t s_key[KEYS > 0 ? KEYS : 1];
  __shared__ uint32_t s_bin[kBins];
  __shared__ uint32_t s_wave[2][WAVES];
  __shared__ uint32_t s_found[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int seq = blockIdx.x / p.kv_heads, head = blockIdx.x - seq * p.kv_heads;
  const int64_t capacity = (int64_t)p.table_width << p.page_shift, held = max(p.lengths[seq], 0);
  const int length = (int)min(held, capacity);
  const int n = (int)(((int64_t)length + (1 << p.page_shift) - 1) >> p.page_shift);
  const int32_t* table = p.table + (int64_t)seq * p.table_stride;
  int32_t* out = p.selected + (int64_t)blockIdx.x * p.count;
  if (head == 0 && tid == 0)  // a length past the table stays one
    p.new_lengths[seq] = held > capacity ? INT32_MAX : n > p.count ? length - ((n - p.count) << p.page_shift) : length;
  if (n <= p.count) {
    for (int i = tid; i < p.count; i += THREADS) out[i] = i < n ? table[i] : -1;
    return;
  }
  const float* scores = p.scores + (int64_t)blockIdx.x * p.table_width;
  auto ordered = [&](int i) {  // scores' order as whole numbers'
    const uint32_t b = __float_as_uint(scores[i] + 0.f);  // -0 as 0
    return b >> 31 ? ~b : b | 0x80000000u;
  };
  auto key = [&](int i) { return KEYS > 0 ? s_key[i] : ordered(i); };

  uint32_t lo = 0xFFFFFFFFu, hi = 0;
  for (int i = 1 + tid; i < n - 1; i += THREADS) {
    const uint32_t k = ordered(i);
    if constexpr (KEYS > 0) s_key[i] = k;
    lo = min(lo, k);
    hi = max(hi, k);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    lo = min(lo, (uint32_t)__shfl_xor((int)lo, o, 64));
    hi = max(hi, (uint32_t)__shfl_xor((int)hi, o, 64));
  }
  if (lane == 0) {
    s_wave[0][wave] = lo;
    s_wave[1][wave] = hi;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    lo = min(lo, s_wave[0][w]);
    hi = max(hi, s_wave[1][w]);
  }
  uint32_t need = (uint32_t)(p.count - 2);  // still to be found within lo..hi
  // selected: keys above `above`, and the first `need` of those equal to `equal`
  while (need > 0 && lo < hi) {
    const int shift = max(32 - __builtin_clz(hi - lo) - 11, 0);
    for (int i = tid; i < kBins; i += THREADS) s_bin[i] = 0;
    __syncthreads();
    for (int i = 1 + tid; i < n - 1; i += THREADS) {
      const uint32_t k = key(i);
      if (k >= lo && k <= hi) atomicAdd(&s_bin[(k - lo) >> shift], 1u);
    }
    __syncthreads();
    uint32_t bin[PER], sum = 0;  // this thread's bins from the top
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += bin[i] = s_bin[kBins - 1 - (tid * PER + i)];
    uint32_t upto = wave_scan(sum);
    if (lane == 63) s_wave[0][wave] = upto;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      if (w < wave) upto += s_wave[0][w];
    if (upto >= need && upto - sum < need) {
      uint32_t over = upto - sum;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (over + bin[i] >= need) {
          s_found[0] = kBins - 1 - (tid * PER + i);
          s_found[1] = over;
          s_found[2] = bin[i];
          break;
        }
        over += bin[i];
      }
    }
    __syncthreads();
    const uint32_t at = s_found[0];
    need -= s_found[1];
    const uint32_t first = lo + (at << shift);
    const bool whole = s_found[2] == need;  // all of this digit's
    hi = min(hi, first + ((1u << shift) - 1));
    lo = first;
    if (whole) {
      need = 0;
      --lo;  // keys above it are selected
      hi = lo;
    }
  }
  // Now lo == hi but for need == 0 from the start: the first `need` keys equal to `lo`, and all above.
  const uint32_t bar = p.count == 2 ? 0xFFFFFFFFu : lo;
  const int span = ((n + 64 * WAVES - 1) / (64 * WAVES)) * 64, begin = wave * span, end = min(begin + span, n);
  auto kind = [&](int i) {  // 2: above the bar, 1: at it
    if (i >= end) return 0;
    if (i == 0 || i == n - 1) return 2;
    const uint32_t k = key(i);
    return k > bar ? 2 : k == bar ? 1 : 0;
  };
  uint32_t sure = 0, ties = 0;
  for (int i = begin; i < end; i += 64) {
    const int k = kind(i + lane);
    sure += __popcll(__ballot(k == 2));
    ties += __popcll(__ballot(k == 1));
  }
  __syncthreads();
  if (lane == 0) {
    s_wave[0][wave] = sure;
    s_wave[1][wave] = ties;
  }
  __syncthreads();
  sure = ties = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w)
    if (w < wave) {
      sure += s_wave[0][w];
      ties += s_wave[1][w];
    }
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  for (int i = begin; i < end; i += 64) {
    const int k = kind(i + lane);
    const uint64_t s = __ballot(k == 2), t = __ballot(k == 1);
    const uint32_t tie = ties + __popcll(t & below);
    const uint32_t place = sure + __popcll(s & below) + min(tie, need);
    if (k == 2 || (k == 1 && tie < need)) out[place] = table[i + lane];
    sure += __popcll(s);
    ties += __popcll(t);
  }
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

int launch_kv4_select(const SelectParams& p, int dtype, hipStream_t st) {
  const int64_t heads = (int64_t)p.seqs * p.kv_heads;
  if (p.table_width > p.count) {  // otherwise all pages are selected
    const int64_t waves = heads * ((p.table_width + kScorePages - 1) / kScorePages);
    if ((waves + 3) / 4 > INT32_MAX) return GRINQH_ERR_INVALID;
    const dim3 grid((uint32_t)((waves + 3) / 4));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, p); };
    const bool bf16 = dtype == GRINQH_DTYPE_BF16;
    switch (p.head_size) {
      case 64: bf16 ? go(kv4_score_kernel<BF16, 64>) : go(kv4_score_kernel<F16, 64>); break;
      case 128: bf16 ? go(kv4_score_kernel<BF16, 128>) : go(kv4_score_kernel<F16, 128>); break;
      case 256: bf16 ? go(kv4_score_kernel<BF16, 256>) : go(kv4_score_kernel<F16, 256>); break;
      default: return GRINQH_ERR_INVALID;
    }
    const int s = status();
    if (s != GRINQH_OK) return s;
  }
  const dim3 grid((uint32_t)heads);
  if (p.table_width <= 2048)
    hipLaunchKernelGGL((kv4_top_kernel<256, 2048>), grid, dim3(256), 0, st, p);
  else if (p.table_width <= 16384)
    hipLaunchKernelGGL((kv4_top_kernel<1024, 16384>), grid, dim3(1024), 0, st, p);
  else
    hipLaunchKernelGGL((kv4_top_kernel<1024, 0>), grid, dim3(1024), 0, st, p);
  return status();
}

}  // namespace grinqh
