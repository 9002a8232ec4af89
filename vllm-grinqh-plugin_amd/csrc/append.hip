// Room for new tokens: free pages into the page table, the tokens' slots.
//
//   need_s = pages(len_s + n_s) - pages(len_s);  page k of all needed ones = free[count - 1 - k]
//   token i of sequence s: position len_s + i, slot = page * page size + place
//
// Bound by latency: lengths, counts, one page index, each loaded after the other.
// So it is one launch in which every block scans all sequences by itself (256 at
// a time) and writes its own 256 tokens' results and its share of the new pages;
// a token of a new page takes the index from the list of free pages, as the table's
// entry may not be written yet.  Nothing that a block reads is written in the launch.
// 32 sequences of 1 token: 3.0 us; 256 of 33 tokens: 3.8 us.  A call with its outputs takes the
// host 12.8 us, which is what calls one after the other take.
#include "attention_launch.h"
#include "wave_scan.h"

namespace grinqh {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

// Inclusive sum over the block; total in all threads.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* s_sum, uint32_t& total) {
  const int wave = threadIdx.x >> 6;
  v = wave_scan(v);
  if ((threadIdx.x & 63) == 63) s_sum[wave] = v;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) v += s_sum[w];
    total += s_sum[w];
  }
  __syncthreads();
  return v;
}

// The last i with first[i] <= x, first[0] <= x: of equal ones the last, which is the one that holds x.
__device__ __forceinline__ int holder(const uint32_t* first, uint32_t x) {
  int at = 0;
#pragma unroll
  for (int step = kThreads / 2; step >= 1; step >>= 1)
    if (first[at + step] <= x) at += step;
  return at;
}

__global__ __launch_bounds__(kThreads) void kv4_append_kernel(const AppendParams p) {
  __shared__ uint32_t s_row[kThreads], s_rank[kThreads];  // first row and first new page of a sequence
  __shared__ int s_len[kThreads], s_place[kThreads];      // tokens held, place of its first new page
  __shared__ uint32_t s_sum[kWaves];
  const int tid = threadIdx.x, page = 1 << p.page_shift;
  const uint32_t id = blockIdx.x * kThreads + tid, ids = gridDim.x * kThreads;
  const int free_count = min(max(*p.free_count, 0), p.free_size);
  const auto page_of = [&](uint32_t rank) {
    return rank < (uint32_t)free_count ? p.free_pages[free_count - 1 - (int)rank] : -1;
  };
  uint32_t rows = 0, rank = 0;  // of the sequences so far
  bool done = id >= (uint32_t)p.tokens;
  uint32_t next = id;  // this thread's next new page
  if (id == 0) p.ends[0] = 0;
  for (int s0 = 0; s0 < p.seqs; s0 += kThreads) {
    const int s = s0 + tid;
    const int len = s < p.seqs ? max(p.lengths[s], 0) : 0;
    // at most p.tokens < 2^23 each: the sum of a block fits 32 bits
    const uint32_t count = s < p.seqs ? (uint32_t)min(max(p.counts[s], 0), p.tokens) : 0u;
    uint32_t total_rows, total_rank;
    const uint32_t sum = rows + block_scan(count, s_sum, total_rows);
    const uint32_t begin = min(sum - count, (uint32_t)p.tokens), upto = min(sum, (uint32_t)p.tokens);
    const int64_t after = (int64_t)len + (upto - begin);
    const int64_t place = ((int64_t)len + page - 1) >> p.page_shift;
    const int64_t end = min((after + page - 1) >> p.page_shift, (int64_t)p.table_width);
    const uint32_t need = (uint32_t)max(end - place, (int64_t)0);
    const uint32_t rank_upto = rank + block_scan(need, s_sum, total_rank);
    s_row[tid] = begin;
    s_rank[tid] = rank_upto - need;
    s_len[tid] = len;
    s_place[tid] = (int)place;
    __syncthreads();
    const uint32_t rows_end = min(rows + total_rows, (uint32_t)p.tokens), rank_end = rank + total_rank;
    if (!done && id < rows_end) {
      const int i = holder(s_row, id);
      const int64_t position = (int64_t)s_len[i] + (id - s_row[i]);
      const int64_t at = position >> p.page_shift;
      int index = -1;
      if (at < p.table_width)
        index = at >= s_place[i] ? page_of(s_rank[i] + (uint32_t)(at - s_place[i]))
                                 : p.table[(int64_t)(s0 + i) * p.table_stride + at];
      p.slots[id] = index >= 0 ? ((int64_t)index << p.page_shift) + (position & (page - 1)) : -1;
      p.positions[id] = (int)min(position, (int64_t)INT32_MAX);
      done = true;
    }
    for (; next < rank_end; next += ids) {
      const int i = holder(s_rank, next);
      p.table[(int64_t)(s0 + i) * p.table_stride + s_place[i] + (next - s_rank[i])] = page_of(next);
    }
    if ((s0 / kThreads) % gridDim.x == blockIdx.x && s < p.seqs) {
      p.ends[s + 1] = (int)upto;
      p.new_lengths[s] = (int)min(after, (int64_t)INT32_MAX);
    }
    rows = rows_end;
    rank = rank_end;
    __syncthreads();
  }
  if (!done) {  // rows behind the last sequence
    p.slots[id] = -1;
    p.positions[id] = 0;
  }
  if (id == 0) *p.new_free_count = max(free_count - (int)min(rank, (uint32_t)INT32_MAX), 0);
}

}  // namespace

int launch_kv4_append(const AppendParams& p, hipStream_t st) {
  const int blocks = p.tokens > 0 ? (p.tokens + kThreads - 1) / kThreads : 1;
  hipLaunchKernelGGL(kv4_append_kernel, dim3((uint32_t)blocks), dim3(kThreads), 0, st, p);
  return hipGetLastError() == hipSuccess ? GRINQH_OK : GRINQH_ERR_HIP;
}

}  // namespace grinqh
