// kv4_store.hip — writes tokens into the 4-bit pages, reads them back, and
// keeps the block representatives of such a cache (gfx950).
//
// A lane handles 8 channels of one row, so a group of 32 channels is a quad of
// lanes whose minimum and maximum meet by DPP; a wave covers 512 / D tokens of
// one head, adjacent waves adjacent heads, so the reads of k and v are whole
// rows and the codes of 4 adjacent tokens fill the record's lines together.
// 16384 tokens, 8 heads of 128, BF16: the store takes 27 us (3.3 TB/s, bound by
// the 400 vector instructions of a wave's 8 values of k and of v), the load 18.5
// (4.8 TB/s, bound by memory).  A workgroup for all of a page, so that no line
// is written from two dies, made the store slower (36 against 33 us).
// Append + seal of one token for 64 sequences: 7.1 us, the chain length ->
// table -> record -> mean.
#include "kv4_format.hpp"
#include "sa_internal.hpp"

namespace sa {
namespace {

using namespace kv4;

constexpr int kThreads = 256;

struct Rows {
  uint8_t* pool;
  void* k;
  void* v;
  const int32_t* slots;
  int32_t* status;
  int64_t num_pages;
  int64_t k_stride;  // elements between tokens
  int64_t v_stride;
  int32_t tokens;
  int32_t kv_heads;
  int32_t type;
};

// A negative slot is a row without a place: it is passed over.  Null records
// mean the same to the callers.
template <int D>
__device__ inline uint8_t* slot_record(const Rows& p, int64_t token, int head, int& t) {
  const int32_t slot = p.slots[token];
  if (slot < 0) return nullptr;
  const int64_t page = slot / kPageTokens;
  if (page >= p.num_pages) {
    flag_status(p.status, kStatusBadPage);
    return nullptr;
  }
  t = slot % kPageTokens;
  return p.pool + (page * p.kv_heads + head) * Format<D>::kRecord;
}

// Work item of a wave: (tokens [first, first + 512 / D), head), head fastest.
template <int D>
__device__ inline bool item_of(const Rows& p, int64_t& token, int& head, int& o) {
  constexpr int kLanes = D / 8;
  constexpr int kTokens = kWave / kLanes;
  const int lane = threadIdx.x % kWave;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / kWave) + threadIdx.x / kWave;
  head = static_cast<int>(item % p.kv_heads);
  token = item / p.kv_heads * kTokens + lane / kLanes;
  o = lane % kLanes;
  return token < p.tokens;
}

template <int D>
__global__ __launch_bounds__(kThreads) void store_kernel(const Rows p) {
  int64_t token;
  int head, o, t = 0;
  if (!item_of<D>(p, token, head, o)) return;  // whole rows leave together: a quad keeps its 4 lanes
  uint8_t* rec = slot_record<D>(p, token, head, t);
  if (!rec) return;
  float k[8], v[8];
  load8(p.k, token * p.k_stride + head * D + o * 8, p.type, k);
  load8(p.v, token * p.v_stride + head * D + o * 8, p.type, v);
  store_key<D>(rec, t, o, quantise(k));
  store_value<D>(rec, t, o, quantise(v));
}

template <int D>
__global__ __launch_bounds__(kThreads) void load_kernel(const Rows p) {
  int64_t token;
  int head, o, t = 0;
  if (!item_of<D>(p, token, head, o)) return;
  const uint8_t* rec = slot_record<D>(p, token, head, t);
  if (!rec) return;
  float x[8];
  load_key<D>(rec, t, o, x);
  store8(p.k, token * p.k_stride + head * D + o * 8, p.type, x);
  load_value<D>(rec, t, o, x);
  store8(p.v, token * p.v_stride + head * D + o * 8, p.type, x);
}

// ---- append + seal ---------------------------------------------------------------

struct Cache {
  uint8_t* pool;
  const int32_t* table;
  int32_t* seq_len;
  int32_t* sealed;
  int32_t* generation;
  float* reps;
  int32_t* status;
  const void* k;
  const void* v;
  int64_t num_pages;
  int64_t k_stride;
  int64_t v_stride;
  int32_t batch;
  int32_t table_stride;
  int32_t kv_heads;
  int32_t rep_heads;
  int32_t rep_stride;
  int32_t local_tokens;
  int32_t type;
};

__device__ inline int64_t table_page(const Cache& p, int b, int64_t logical) {
  if (logical < 0 || logical >= p.table_stride) return -1;
  const int64_t page = p.table[static_cast<int64_t>(b) * p.table_stride + logical];
  return (page >= 0 && page < p.num_pages) ? page : -1;
}

// The sum of a block's 32 keys over a wave: lane (octet o = lane % (D/8),
// share = lane / (D/8)) adds the tokens of its share in order, then the
// shares meet; every lane of an octet gets the sums of its 8 channels.
template <int D>
__device__ inline void block_key_sum(const uint8_t* rec, int lane, float (&sum)[8]) {
  constexpr int kLanes = D / 8;
  constexpr int kShares = kWave / kLanes;
  constexpr int kTokens = kPageTokens / kShares;
  const int o = lane % kLanes;
  const int share = lane / kLanes;
#pragma unroll
  for (int n = 0; n < 8; ++n) sum[n] = 0.0f;
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    float x[8];
    load_key<D>(rec, share * kTokens + i, o, x);
#pragma unroll
    for (int n = 0; n < 8; ++n) sum[n] += x[n];
  }
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    if constexpr (kLanes <= 8) sum[n] = xor_sum<8>(sum[n]);
    if constexpr (kLanes <= 16) sum[n] = xor_sum<16>(sum[n]);
    sum[n] = xor_sum<32>(sum[n]);
  }
}

// One workgroup a sequence: its token's rows, then (in a step that fills a
// block) a wave a KV head for the representative.
template <int D>
__global__ __launch_bounds__(kThreads) void append_seal_kernel(const Cache p) {
  constexpr int kLanes = D / 8;
  const int b = blockIdx.x;
  const int tid = threadIdx.x;
  const int wave = tid / kWave;
  const int lane = tid % kWave;
  const int64_t len = p.seq_len[b];
  int64_t s = p.sealed[b];
  if (len < 0 || s < 0 || s * kPageTokens > len) {
    if (tid == 0) flag_status(p.status, kStatusBadLength);
    return;
  }
  const int64_t page = table_page(p, b, len / kPageTokens);
  if (page < 0) {
    if (tid == 0) flag_status(p.status, kStatusCapacity);
    return;
  }
  const int t = static_cast<int>(len % kPageTokens);
  for (int e = tid; e < p.kv_heads * kLanes; e += kThreads) {  // kThreads is a multiple of kLanes: quads stay whole
    const int head = e / kLanes;
    const int o = e % kLanes;
    uint8_t* rec = p.pool + (page * p.kv_heads + head) * Format<D>::kRecord;
    float k[8], v[8];
    load8(p.k, b * p.k_stride + head * D + o * 8, p.type, k);
    load8(p.v, b * p.v_stride + head * D + o * 8, p.type, v);
    store_key<D>(rec, t, o, quantise(k));
    store_value<D>(rec, t, o, quantise(v));
  }
  __syncthreads();  // the seal may read the row just written by other waves; every wave has read the lengths
  if (tid == 0) p.seq_len[b] = static_cast<int32_t>(len + 1);

  int added = 0;
  while (len + 1 >= (s + 1) * kPageTokens + p.local_tokens) {
    const int64_t block = s < p.rep_stride ? table_page(p, b, s) : -1;
    if (block < 0) {
      if (tid == 0) flag_status(p.status, kStatusCapacity);
      break;
    }
    const int group = p.rep_heads / p.kv_heads;
    for (int head = wave; head < p.kv_heads; head += kThreads / kWave) {
      float sum[8];
      block_key_sum<D>(p.pool + (block * p.kv_heads + head) * Format<D>::kRecord, lane, sum);
      if (lane < kLanes) {
        for (int j = 0; j < group; ++j) {
          float* rep = p.reps + ((static_cast<int64_t>(b) * p.rep_heads + head * group + j) * D + lane * 8) * p.rep_stride + s;
#pragma unroll
          for (int n = 0; n < 8; ++n) rep[static_cast<int64_t>(n) * p.rep_stride] = sum[n] / kPageTokens;
        }
      }
    }
    ++s;
    ++added;
  }
  if (tid == 0 && added) {
    p.sealed[b] = static_cast<int32_t>(s);
    if (p.generation) p.generation[b] += added;
  }
}

// The bulk seal after a prompt: workgroup (chunk of kSealBlocks blocks, KV
// head, sequence).  The means of a chunk are turned through LDS, so that a
// channel's row of the representatives is written as a whole 128-byte line.
constexpr int kSealBlocks = 32;

template <int D>
__global__ __launch_bounds__(kThreads) void seal_kernel(const Cache p) {
  constexpr int kLanes = D / 8;
  __shared__ float mean[D][kSealBlocks + 1];
  const int b = blockIdx.z;
  const int head = blockIdx.y;
  const int wave = threadIdx.x / kWave;
  const int lane = threadIdx.x % kWave;
  const int64_t len = p.seq_len[b];
  const int64_t sealed = p.sealed[b];
  if (len < 0 || sealed < 0 || sealed * kPageTokens > len) return;  // advance_seal_kernel flags it
  const int64_t end = (len - p.local_tokens) / kPageTokens;          // (a negative difference seals nothing)
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kSealBlocks;
  const int64_t from = first > sealed ? first : sealed;
  int64_t to = first + kSealBlocks < end ? first + kSealBlocks : end;
  if (to > p.rep_stride) to = p.rep_stride;
  if (from >= to) return;
  for (int64_t s = from + wave; s < to; s += kThreads / kWave) {
    const int64_t page = table_page(p, b, s);
    if (page < 0) continue;  // the block stays unsealed (advance_seal_kernel)
    float sum[8];
    block_key_sum<D>(p.pool + (page * p.kv_heads + head) * Format<D>::kRecord, lane, sum);
    if (lane < kLanes) {
#pragma unroll
      for (int n = 0; n < 8; ++n) mean[lane * 8 + n][s - first] = sum[n] / kPageTokens;
    }
  }
  __syncthreads();
  const int group = p.rep_heads / p.kv_heads;
  for (int e = threadIdx.x; e < D * kSealBlocks; e += kThreads) {
    const int d = e / kSealBlocks;
    const int64_t s = first + e % kSealBlocks;
    if (s < from || s >= to || table_page(p, b, s) < 0) continue;
    for (int j = 0; j < group; ++j)
      p.reps[((static_cast<int64_t>(b) * p.rep_heads + head * group + j) * D + d) * p.rep_stride + s] =
          mean[d][s - first];
  }
}

// One wave a sequence advances its counters over the blocks that have a page
// and a place for their representative; the first one without stops it.
__global__ __launch_bounds__(kWave) void advance_seal_kernel(const Cache p) {
  const int b = blockIdx.x;
  const int lane = threadIdx.x;
  const int64_t len = p.seq_len[b];
  const int64_t sealed = p.sealed[b];
  if (len < 0 || sealed < 0 || sealed * kPageTokens > len) {
    if (lane == 0) flag_status(p.status, kStatusBadLength);
    return;
  }
  const int64_t end = (len - p.local_tokens) / kPageTokens;
  int64_t s = sealed;
  bool stopped = false;
  while (s < end && !stopped) {  // the same in every lane
    const int64_t at = s + lane;
    const bool bad = at < end && (at >= p.rep_stride || table_page(p, b, at) < 0);
    const uint64_t mask = __ballot(bad);
    if (mask) {
      s += __builtin_ctzll(mask);
      stopped = true;
    } else {
      s = s + kWave < end ? s + kWave : end;
    }
  }
  if (lane != 0) return;
  if (stopped) flag_status(p.status, kStatusCapacity);
  if (s > sealed) {
    p.sealed[b] = static_cast<int32_t>(s);
    if (p.generation) p.generation[b] += static_cast<int32_t>(s - sealed);
  }
}

template <class F>
hipError_t for_head_dim(int head_dim, F&& f) {
  if (head_dim == 64) f(std::integral_constant<int, 64>{});
  if (head_dim == 128) f(std::integral_constant<int, 128>{});
  if (head_dim == 256) f(std::integral_constant<int, 256>{});
  return hipGetLastError();
}

Cache cache_of(const Kv4SealLaunch& a) {
  Cache p{};
  p.pool = a.pool;
  p.table = a.table;
  p.seq_len = a.seq_len;
  p.sealed = a.sealed;
  p.generation = a.generation;
  p.reps = a.reps;
  p.status = a.status;
  p.k = a.k;
  p.v = a.v;
  p.num_pages = a.num_pages;
  p.k_stride = a.k_stride;
  p.v_stride = a.v_stride;
  p.batch = a.batch;
  p.table_stride = a.table_stride;
  p.kv_heads = a.kv_heads;
  p.rep_heads = a.rep_heads;
  p.rep_stride = a.rep_stride;
  p.local_tokens = a.local_tokens;
  p.type = a.type;
  return p;
}

}  // namespace

hipError_t launch_kv4_rows(const Kv4RowsLaunch& a, hipStream_t stream) {
  Rows p{};
  p.pool = a.pool;
  p.k = a.k;
  p.v = a.v;
  p.slots = a.slots;
  p.status = a.status;
  p.num_pages = a.num_pages;
  p.k_stride = a.k_stride;
  p.v_stride = a.v_stride;
  p.tokens = a.tokens;
  p.kv_heads = a.kv_heads;
  p.type = a.type;
  return for_head_dim(a.head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    constexpr int kTokens = kWave / (D / 8);
    const int64_t items = (static_cast<int64_t>(a.tokens) + kTokens - 1) / kTokens * a.kv_heads;
    const dim3 grid(static_cast<uint32_t>((items + kThreads / kWave - 1) / (kThreads / kWave)));
    if (a.load)
      hipLaunchKernelGGL(load_kernel<D>, grid, dim3(kThreads), 0, stream, p);
    else
      hipLaunchKernelGGL(store_kernel<D>, grid, dim3(kThreads), 0, stream, p);
  });
}

hipError_t launch_kv4_append_seal(const Kv4SealLaunch& a, hipStream_t stream) {
  const Cache p = cache_of(a);
  return for_head_dim(a.head_dim, [&](auto d) {
    hipLaunchKernelGGL(append_seal_kernel<decltype(d)::value>, dim3(a.batch), dim3(kThreads), 0, stream, p);
  });
}

hipError_t launch_kv4_seal(const Kv4SealLaunch& a, hipStream_t stream) {
  const Cache p = cache_of(a);
  const int blocks = a.table_stride < a.rep_stride ? a.table_stride : a.rep_stride;
  const dim3 grid((blocks + kSealBlocks - 1) / kSealBlocks, a.kv_heads, a.batch);
  const hipError_t e = for_head_dim(a.head_dim, [&](auto d) {
    hipLaunchKernelGGL(seal_kernel<decltype(d)::value>, grid, dim3(kThreads), 0, stream, p);
  });
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(advance_seal_kernel, dim3(a.batch), dim3(kWave), 0, stream, p);
  return hipGetLastError();
}

}  // namespace sa
