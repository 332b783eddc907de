// page_table.hip — hands out and takes back the pages of a paged cache on the
// GPU: block tables, slots and positions of a batch's next tokens from the
// requests' lengths (gfx950).
//
// The pages and tokens of request b follow from exclusive prefix sums over
// the batch.  Every workgroup forms them itself (a few loads a thread and two
// barriers) instead of waiting for another launch; it keeps the sums at the
// first request of each of its threads in LDS.  A token then finds its
// request by a binary search over these and a walk within one thread's share
// (none up to kThreads requests).  Latency is all that counts here: a decode
// step's call is one workgroup and one launch (64 sequences: 6.3 us, most of it
// the launch and three dependent loads; 512 sequences of up to 127 tokens each:
// 10.4 us, and 6.6 to take the pages of 171 back).
#include "sa_device.hpp"
#include "sa_internal.hpp"

namespace sa {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kItems = 4;  // tokens a thread before another workgroup is worth its scan

// What a launch writes: the outputs that may lie over the inputs (the new
// lengths and the free count) come after every read of those.
enum Finish : int32_t {
  kTables = 0,    // everything else
  kLengths = 1,   // those alone, one workgroup
  kOneGroup = 2,  // both, one workgroup: a barrier between them
  kSeparate = 3,  // both: the outputs do not lie over the inputs
};

struct Sums {
  int64_t tokens;
  int64_t pages;
};

struct Scan {
  int32_t tokens[kThreads + 1];  // sums before each thread's first request; the totals at the end
  int32_t pages[kThreads + 1];
  Sums wave[kWaves];
  int32_t bad;
  int32_t ok;
};

// Exclusive prefix over the workgroup of each thread's (tokens, pages), and
// the totals; 64-bit, so that no total of a batch wraps.
__device__ inline Sums scan_sums(Scan& s, Sums mine, Sums& total) {
  const int lane = threadIdx.x % kWave;
  const int wave = threadIdx.x / kWave;
  Sums run = mine;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int64_t t = __shfl_up(run.tokens, d);
    const int64_t p = __shfl_up(run.pages, d);
    if (lane >= d) run.tokens += t, run.pages += p;
  }
  if (lane == kWave - 1) s.wave[wave] = run;
  __syncthreads();
  Sums before{0, 0};
  total = Sums{0, 0};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const Sums x = s.wave[w];
    if (w < wave) before.tokens += x.tokens, before.pages += x.pages;
    total.tokens += x.tokens, total.pages += x.pages;
  }
  return Sums{before.tokens + run.tokens - mine.tokens, before.pages + run.pages - mine.pages};
}

__device__ inline int64_t pages_of(int64_t tokens) { return (tokens + kPageTokens - 1) / kPageTokens; }

// The share (thread) of item x, given the sums before each share: the last
// share whose sum is <= x and that holds an item.
__device__ inline int share_of(const int32_t* before, int64_t x) {
  int lo = 0, hi = kThreads;  // before[lo] <= x < before[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (before[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

struct Reserve {
  int32_t* table;
  const int32_t* seq_len;
  const int32_t* new_tokens;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t* query_start;
  int32_t* slots;
  int32_t* positions;
  int32_t* seq_len_out;
  int32_t* free_count_out;
  int32_t* status;
  int64_t num_pages;
  int32_t batch;
  int32_t table_stride;
  int32_t max_tokens;
  int32_t finish;  // one of Finish
};

__device__ inline Sums wants(const Reserve& p, int64_t len, int64_t n) {
  return Sums{n, pages_of(len + n) - pages_of(len)};
}

__global__ __launch_bounds__(kThreads) void reserve_kernel(const Reserve p) {
  __shared__ Scan s;
  const int tid = threadIdx.x;
  const int share = (p.batch + kThreads - 1) / kThreads;
  const int first = min(tid * share, p.batch);
  const int last = min(first + share, p.batch);
  if (tid == 0) s.bad = 0;
  __syncthreads();

  Sums mine{0, 0};
  int bad = 0;
  for (int b = first; b < last; ++b) {
    const int64_t len = p.seq_len[b], n = p.new_tokens[b];
    if (len < 0 || n < 0 || len + n > INT32_MAX)
      bad |= kStatusBadLength;
    else if (n > 0 && pages_of(len + n) > p.table_stride)
      bad |= kStatusCapacity;
    else {
      const Sums w = wants(p, len, n);
      mine.tokens += w.tokens, mine.pages += w.pages;
    }
  }
  if (bad) atomicOr(&s.bad, bad);
  Sums total;
  const Sums before = scan_sums(s, mine, total);  // its barrier orders s.bad too
  const int64_t count = p.free_count[0];
  s.tokens[tid] = static_cast<int32_t>(min<int64_t>(before.tokens, INT32_MAX));
  s.pages[tid] = static_cast<int32_t>(min<int64_t>(before.pages, INT32_MAX));
  int why = s.bad;
  if (count < 0 || count > p.num_pages) why |= kStatusBadLength;
  else if (total.pages > count) why |= kStatusCapacity;
  if (total.tokens > p.max_tokens) why |= kStatusCapacity;
  const bool ok = why == 0;
  if (tid == 0) {
    s.tokens[kThreads] = static_cast<int32_t>(min<int64_t>(total.tokens, INT32_MAX));
    s.pages[kThreads] = static_cast<int32_t>(min<int64_t>(total.pages, INT32_MAX));
    if (!ok && blockIdx.x == 0 && p.finish != kLengths) flag_status(p.status, why);
  }
  __syncthreads();

  if (p.finish != kLengths) {
    const int64_t start = static_cast<int64_t>(blockIdx.x) * kThreads + tid;
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    if (blockIdx.x == 0) {  // where each request's tokens start
      int64_t at = before.tokens;
      for (int b = first; b < last; ++b) {
        p.query_start[b] = ok ? static_cast<int32_t>(at) : 0;
        if (ok) at += p.new_tokens[b];
      }
      if (tid == 0) p.query_start[p.batch] = ok ? static_cast<int32_t>(total.tokens) : 0;
    }
    if (ok) {
      for (int64_t x = start; x < total.pages; x += step) {  // the pages handed out, in the requests' order
        int b = share_of(s.pages, x) * share;
        int64_t at = s.pages[b / share];
        int64_t len = p.seq_len[b];
        int64_t w = wants(p, len, p.new_tokens[b]).pages;
        while (x >= at + w) {
          at += w;
          ++b;
          len = p.seq_len[b];
          w = wants(p, len, p.new_tokens[b]).pages;
        }
        p.table[static_cast<int64_t>(b) * p.table_stride + pages_of(len) + (x - at)] = p.free_pages[count - 1 - x];
      }
    }
    for (int64_t x = start; x < p.max_tokens; x += step) {
      int32_t slot = -1, position = -1;
      if (ok && x < total.tokens) {
        const int sh = share_of(s.tokens, x);
        int b = sh * share;
        int64_t at = s.tokens[sh];
        int64_t page_at = s.pages[sh];
        int64_t len = p.seq_len[b], n = p.new_tokens[b];
        while (x >= at + n) {
          at += n;
          page_at += wants(p, len, n).pages;
          ++b;
          len = p.seq_len[b];
          n = p.new_tokens[b];
        }
        position = static_cast<int32_t>(len + (x - at));
        const int64_t block = position / kPageTokens;
        const int64_t held = pages_of(len);
        const int64_t page = block < held ? p.table[static_cast<int64_t>(b) * p.table_stride + block]
                                          : p.free_pages[count - 1 - page_at - (block - held)];
        if (page >= 0 && page < p.num_pages)
          slot = static_cast<int32_t>(page * kPageTokens + position % kPageTokens);
        else
          flag_status(p.status, kStatusBadPage);
      }
      p.slots[x] = slot;
      if (p.positions) p.positions[x] = position;
    }
  }
  if (p.finish == kTables || (p.finish == kSeparate && blockIdx.x != 0)) return;
  if (p.finish == kOneGroup) __syncthreads();  // every lane has read the lengths, which may be written in place
  for (int b = first; b < last; ++b)
    p.seq_len_out[b] = ok ? static_cast<int32_t>(static_cast<int64_t>(p.seq_len[b]) + p.new_tokens[b]) : p.seq_len[b];
  if (tid == 0) p.free_count_out[0] = static_cast<int32_t>(ok ? count - total.pages : count);
}

struct Release {
  const int32_t* table;
  const int32_t* seq_len;
  int32_t* sealed;
  const int32_t* finished;
  int32_t* free_pages;
  const int32_t* free_count;
  int32_t* seq_len_out;
  int32_t* free_count_out;
  int32_t* status;
  int64_t num_pages;
  int32_t batch;
  int32_t table_stride;
  int32_t finish;
};

__global__ __launch_bounds__(kThreads) void release_kernel(const Release p) {
  __shared__ Scan s;
  const int tid = threadIdx.x;
  const int share = (p.batch + kThreads - 1) / kThreads;
  const int first = min(tid * share, p.batch);
  const int last = min(first + share, p.batch);
  if (tid == 0) s.bad = 0;
  __syncthreads();
  Sums mine{0, 0};
  int bad = 0;
  for (int b = first; b < last; ++b) {
    if (!p.finished[b]) continue;
    const int64_t n = pages_of(p.seq_len[b]);
    if (p.seq_len[b] < 0 || n > p.table_stride)
      bad = kStatusBadLength;
    else
      mine.pages += n;
  }
  if (bad) atomicOr(&s.bad, bad);
  Sums total;
  const Sums before = scan_sums(s, mine, total);
  const int64_t count = p.free_count[0];
  s.pages[tid] = static_cast<int32_t>(min<int64_t>(before.pages, INT32_MAX));
  int why = s.bad;
  if (count < 0) why |= kStatusBadLength;
  else if (count + total.pages > p.num_pages) why |= kStatusCapacity;
  const bool ok = why == 0;
  if (tid == 0) {
    s.pages[kThreads] = static_cast<int32_t>(min<int64_t>(total.pages, INT32_MAX));
    if (!ok && blockIdx.x == 0 && p.finish != kLengths) flag_status(p.status, why);
  }
  __syncthreads();
  if (p.finish != kLengths && ok) {
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t x = static_cast<int64_t>(blockIdx.x) * kThreads + tid; x < total.pages; x += step) {
      const int sh = share_of(s.pages, x);
      int b = sh * share;
      int64_t at = s.pages[sh];
      int64_t n = p.finished[b] ? pages_of(p.seq_len[b]) : 0;
      while (x >= at + n) {
        at += n;
        ++b;
        n = p.finished[b] ? pages_of(p.seq_len[b]) : 0;
      }
      const int32_t page = p.table[static_cast<int64_t>(b) * p.table_stride + (x - at)];
      if (page < 0 || page >= p.num_pages) flag_status(p.status, kStatusBadPage);
      p.free_pages[count + x] = page;
    }
  }
  if (p.finish == kTables || (p.finish == kSeparate && blockIdx.x != 0)) return;
  if (p.finish == kOneGroup) __syncthreads();
  for (int b = first; b < last; ++b) {
    const bool gone = ok && p.finished[b];
    p.seq_len_out[b] = gone ? 0 : p.seq_len[b];
    if (gone) p.sealed[b] = 0;
  }
  if (tid == 0) p.free_count_out[0] = static_cast<int32_t>(ok ? count + total.pages : count);
}

// One workgroup takes `items` by itself up to kItems a thread; with more of
// them, outputs in place wait for a second launch, which the first one's reads
// precede.
template <class K, class P>
hipError_t launch(K kernel, P p, int64_t items, bool in_place, hipStream_t stream) {
  const int64_t groups = (items + kThreads * kItems - 1) / (kThreads * kItems);
  p.finish = groups <= 1 ? kOneGroup : in_place ? kTables : kSeparate;
  const dim3 grid(static_cast<uint32_t>(groups < 1 ? 1 : groups < 256 ? groups : 256));
  hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.finish != kTables) return e;
  p.finish = kLengths;
  hipLaunchKernelGGL(kernel, dim3(1), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_reserve_tokens(const ReserveLaunch& a, hipStream_t stream) {
  Reserve p{};
  p.table = a.table;
  p.seq_len = a.seq_len;
  p.new_tokens = a.new_tokens;
  p.free_pages = a.free_pages;
  p.free_count = a.free_count;
  p.query_start = a.query_start;
  p.slots = a.slots;
  p.positions = a.positions;
  p.seq_len_out = a.seq_len_out;
  p.free_count_out = a.free_count_out;
  p.status = a.status;
  p.num_pages = a.num_pages;
  p.batch = a.batch;
  p.table_stride = a.table_stride;
  p.max_tokens = a.max_tokens;
  return launch(reserve_kernel, p, a.max_tokens, a.in_place, stream);
}

hipError_t launch_release_sequences(const ReleaseLaunch& a, hipStream_t stream) {
  Release p{};
  p.table = a.table;
  p.seq_len = a.seq_len;
  p.sealed = a.sealed;
  p.finished = a.finished;
  p.free_pages = a.free_pages;
  p.free_count = a.free_count;
  p.seq_len_out = a.seq_len_out;
  p.free_count_out = a.free_count_out;
  p.status = a.status;
  p.num_pages = a.num_pages;
  p.batch = a.batch;
  p.table_stride = a.table_stride;
  // pages that may go back: the batch's share of the pool, at most its tables
  const int64_t tables = static_cast<int64_t>(a.batch) * a.table_stride;
  return launch(release_kernel, p, tables < a.num_pages ? tables : a.num_pages, a.in_place, stream);
}

}  // namespace sa
