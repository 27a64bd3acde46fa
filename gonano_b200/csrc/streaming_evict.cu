// Eviction from a paged cache by accumulated attention weight (gn_cache_evict): which keys stay, and their move.
//
// Bound: HBM, the kept rows read and written once (16 D bytes a key) and 4 bytes of weight a key.
#include <algorithm>

#include "streaming_tc.cuh"

namespace gn {

namespace {

struct Evict {
  gn_evict_params p;
  int32_t* kept; int32_t* new_lens; float* mass_out;   // new_lens null: written at the end, over the lengths that all kernels read
  int vec;
};
// Weight as an integer that orders like it: equal values (both zeros too) alike, NaN below everything.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (isnan(x)) return 0u;
  const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ int evict_len(const gn_evict_params& p, int r) { return min(max(p.context_lens[r], 0), p.max_context); }
__device__ __forceinline__ int64_t slot_of(const gn_evict_params& p, const int32_t* table, int width, int r, int hk, int j) {
  const int page = table[(int64_t)r * width + j / p.page_size];
  if ((unsigned)page >= (unsigned)p.pages) return -1;
  return (((int64_t)page * p.n_kv_head + hk) * p.page_size + j % p.page_size) * p.head_dim;
}

constexpr int kSelect = 1024, kWarpsS = kSelect / 32;
constexpr int kCached = 49152;

// A CTA per (row, kv head).  The threshold (the smallest kept order key among those that are neither sinks nor recent) by three radix
// passes of 11, 11 and 10 bits; the digit of a warp's first key is added once for all that share it (weights are often alike: keys
// nobody looked at hold 0).  Then every warp takes a run of keys, counts what it keeps, and writes the indices behind those of the warps before it: two
// passes, no order left to chance.  Of the keys equal to the threshold the first ones are kept.  Up to kCached keys are read from memory
// once and kept as order keys in shared memory.  Bound: the latency of its passes; 22 us for 32 rows of 8704 keys.
__global__ void __launch_bounds__(kSelect) evict_select_kernel(const __grid_constant__ Evict e, int cached) {
  extern __shared__ uint32_t cache[];
  pdl_trigger();
  const gn_evict_params& p = e.p;
  const int hk = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = evict_len(p, r), keep = min(n, p.budget), lo = p.sinks, hi = n - p.recent;
  const int64_t head = (int64_t)r * p.n_kv_head + hk;
  const float* mass = p.mass + head * p.mass_stride;
  int32_t* kept = e.kept + head * p.budget;
  __shared__ int hist[2048];
  __shared__ int sums[kWarpsS], ties_s[kWarpsS];
  __shared__ uint32_t prefix_s;
  __shared__ int want_s;
  const int wanted = n <= p.budget ? 0 : p.budget - p.sinks - p.recent;   // of the middle
  uint32_t prefix = 0;
  int want = wanted;
  if (wanted > 0 && cached) {
#pragma unroll 4
    for (int j = lo + tid; j < hi; j += kSelect) cache[j] = order_key(mass[j]);
    __syncthreads();
  }
  auto key_at = [&](int j) { return cached ? cache[j] : order_key(mass[j]); };   // of the middle
  if (wanted > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
      hist[tid] = 0; hist[tid + 1024] = 0;
      __syncthreads();
#pragma unroll 4
      for (int j0 = lo; j0 < hi; j0 += kSelect) {
        const int j = j0 + tid;
        const uint32_t k = j < hi ? key_at(j) : 0u;
        const bool in = j < hi && (pass == 0 || (k >> (pass == 1 ? 21 : 10)) == prefix);
        const uint32_t digit = in ? (k >> shift) & (uint32_t)(bins - 1) : 0xffffffffu;
        const uint32_t most = __shfl_sync(0xffffffffu, digit, 0), same = __ballot_sync(0xffffffffu, in && digit == most);
        if (in && digit != most) atomicAdd(&hist[digit], 1);
        else if (in && lane == __ffs(same) - 1) atomicAdd(&hist[digit], __popc(same));
      }
      __syncthreads();
      // the digit at which the count from above reaches `want`: thread t holds bins 2t' and 2t' + 1 counted from the top
      const int b1 = 2047 - 2 * tid, b0 = b1 - 1, h1 = hist[b1], h0 = hist[b0];
      int before = h1 + h0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) { const int y = __shfl_up_sync(0xffffffffu, before, d); if (lane >= d) before += y; }
      if (lane == 31) sums[warp] = before;
      __syncthreads();
      const int base = __reduce_add_sync(0xffffffffu, lane < warp ? sums[lane] : 0);
      const int above1 = base + before - h1 - h0, above0 = above1 + h1;   // keys of larger digits
      if (above1 < want && want <= above1 + h1) { prefix_s = (pass == 0 ? 0u : prefix << (pass == 1 ? 11 : 10)) | (uint32_t)b1; want_s = want - above1; }
      if (above0 < want && want <= above0 + h0) { prefix_s = (pass == 0 ? 0u : prefix << (pass == 1 ? 11 : 10)) | (uint32_t)b0; want_s = want - above0; }
      __syncthreads();
      prefix = prefix_s; want = want_s;
      __syncthreads();
    }
  }
  // all keys above `prefix` stay, and the first `want` of those equal to it
  const int run = ((n + kWarpsS - 1) / kWarpsS + 31) & ~31, j0 = min(n, warp * run), j1 = min(n, j0 + run);
  auto look = [&](int j, bool& take, bool& tie) {
    take = tie = false;
    if (j >= j1) return;
    if (n <= p.budget || j < lo || j >= hi) take = true;
    else if (wanted > 0) { const uint32_t k = key_at(j); take = k > prefix; tie = k == prefix; }
  };
  int sure = 0, equal = 0;
#pragma unroll 4
  for (int j = j0; j < j1; j += 32) {
    bool take, tie;
    look(j + lane, take, tie);
    sure += __popc(__ballot_sync(0xffffffffu, take));
    equal += __popc(__ballot_sync(0xffffffffu, tie));
  }
  if (lane == 0) { sums[warp] = sure; ties_s[warp] = equal; }
  __syncthreads();
  // kept and equal keys before this warp's
  int ties = __reduce_add_sync(0xffffffffu, lane < warp ? ties_s[lane] : 0);
  int at = __reduce_add_sync(0xffffffffu, lane < warp ? sums[lane] : 0) + min(ties, want);
  for (int j = j0; j < j1; j += 32) {
    bool take, tie;
    look(j + lane, take, tie);
    const uint32_t tied = __ballot_sync(0xffffffffu, tie), below = (1u << lane) - 1u;
    if (tie) take = ties + __popc(tied & below) < want;
    ties += __popc(tied);
    const uint32_t taken = __ballot_sync(0xffffffffu, take);
    if (take) {
      const int to = at + __popc(taken & below);
      kept[to] = j + lane;
      if (e.mass_out) e.mass_out[head * p.budget + to] = mass[j + lane];
    }
    at += __popc(taken);
  }
  for (int i = keep + tid; i < p.budget; i += kSelect) { kept[i] = -1; if (e.mass_out) e.mass_out[head * p.budget + i] = 0.0f; }
  if (hk == 0 && tid == 0 && e.new_lens) e.new_lens[r] = keep;
}

// A row's kept keys to slots that may be its own: the slots are filled in ascending order, KEYS at a time, every read of a group before its
// writes: slot i <= kept[i], so a group writes only what it or earlier groups have read.  256 threads do a (row, kv head)'s channels c0 .. c0 + 31.
template <int KEYS>
__device__ __forceinline__ void move_row(const Evict& e, int hk, int r, float* pages, int c0, int64_t (&from)[KEYS], int64_t (&to)[KEYS]) {
  const gn_evict_params& p = e.p;
  const int tid = threadIdx.x, keep = min(evict_len(p, r), p.budget);
  const int32_t* kept = e.kept + ((int64_t)r * p.n_kv_head + hk) * p.budget;
  for (int i0 = 0; i0 < keep; i0 += KEYS) {
    __syncthreads();
    if (tid < KEYS) {
      const int i = i0 + tid;
      from[tid] = i < keep ? slot_of(p, p.page_table, p.table_width, r, hk, kept[i]) : -1;
      to[tid] = i < keep ? slot_of(p, p.new_table, p.new_width, r, hk, i) : -1;
    }
    __syncthreads();
    if (e.vec) {   // 8 threads carry a key's 32 channels
      const int c = c0 + (tid & 7) * 4;
      const bool in = c < p.head_dim;
      float4 x[KEYS / 32];
#pragma unroll
      for (int u = 0; u < KEYS / 32; ++u) {
        const int k = (tid >> 3) + u * 32;
        x[u] = make_float4(0, 0, 0, 0);
        if (in && from[k] >= 0) x[u] = *reinterpret_cast<const float4*>(pages + from[k] + c);
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < KEYS / 32; ++u) {
        const int k = (tid >> 3) + u * 32;
        if (in && to[k] >= 0) *reinterpret_cast<float4*>(pages + to[k] + c) = x[u];
      }
    } else {
      const int c = c0 + (tid & 31);
      const bool in = c < p.head_dim;
      float x[KEYS / 8];
#pragma unroll
      for (int u = 0; u < KEYS / 8; ++u) { const int k = (tid >> 5) + u * 8; x[u] = in && from[k] >= 0 ? pages[from[k] + c] : 0.0f; }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < KEYS / 8; ++u) { const int k = (tid >> 5) + u * 8; if (in && to[k] >= 0) pages[to[k] + c] = x[u]; }
    }
  }
}

// In place (new_table is page_table): a CTA per (32 channels, kv head, row x {key, value}).  With the selection 53 us for 32 rows of up to 8704 keys to
// 2048 (on other pages 49), 113 for 64 x 2 of 4096 to 2048 (104), 12 for 8 x 2 of 384 to 128 (14).
__global__ void __launch_bounds__(256) evict_move_kernel(const __grid_constant__ Evict e) {
  pdl_wait();
  __shared__ int64_t from[256], to[256];
  const int r = blockIdx.z >> 1, n = evict_len(e.p, r);
  if (n > e.p.budget) move_row(e, blockIdx.y, r, (blockIdx.z & 1) ? e.p.value_pages : e.p.key_pages, blockIdx.x * 32, from, to);   // else nothing moves
}

// To other pages: every kept key on its own.  A CTA per (64 kept keys, kv head, row x {key, value}); with 16-byte accesses
// `lanes` threads carry a row, all reads of a thread before its writes.  Bound: HBM; 24 us for 32 rows of 2048 keys (67 MB read and written, 5.6 TB/s).
__global__ void __launch_bounds__(256) evict_copy_kernel(const __grid_constant__ Evict e, int lanes) {
  pdl_wait();
  const gn_evict_params& p = e.p;
  const int hk = blockIdx.y, r = blockIdx.z >> 1, i0 = blockIdx.x * 64;
  const int keep = min(evict_len(p, r), p.budget);
  if (i0 >= keep) return;
  const int32_t* kept = e.kept + ((int64_t)r * p.n_kv_head + hk) * p.budget;
  float* pages = (blockIdx.z & 1) ? p.value_pages : p.key_pages;
  __shared__ int64_t from[64], to[64];
  // A row that keeps a page of its own in its column (new_table may be a copy of page_table's first columns) goes in order, by the first blocks
  int own = 0;
  for (int c = threadIdx.x; (int64_t)c * p.page_size < keep; c += 256) own |= p.new_table[(int64_t)r * p.new_width + c] == p.page_table[(int64_t)r * p.table_width + c];
  if (__syncthreads_or(own)) {
    for (int c0 = blockIdx.x * 32; c0 < p.head_dim; c0 += (keep + 63) / 64 * 32) move_row(e, hk, r, pages, c0, from, to);
    return;
  }
  if (threadIdx.x < 64) {
    const int i = i0 + threadIdx.x;
    from[threadIdx.x] = i < keep ? slot_of(p, p.page_table, p.table_width, r, hk, kept[i]) : -1;
    to[threadIdx.x] = i < keep ? slot_of(p, p.new_table, p.new_width, r, hk, i) : -1;
  }
  __syncthreads();
  if (e.vec) {
    const int mine = threadIdx.x / lanes, ch = (threadIdx.x % lanes) * 4, step = 256 / lanes;
    for (int c = ch; c < p.head_dim; c += lanes * 4)
      for (int k0 = mine; k0 < 64; k0 += 4 * step) {
        float4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int k = k0 + u * step;
          x[u] = make_float4(0, 0, 0, 0);
          if (k < 64 && from[k] >= 0) x[u] = *reinterpret_cast<const float4*>(pages + from[k] + c);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int k = k0 + u * step;
          if (k < 64 && to[k] >= 0) *reinterpret_cast<float4*>(pages + to[k] + c) = x[u];
        }
      }
  } else {
    for (int i = threadIdx.x; i < 64 * p.head_dim; i += 256) {
      const int k = i / p.head_dim, c = i % p.head_dim;
      if (to[k] >= 0) pages[to[k] + c] = from[k] >= 0 ? pages[from[k] + c] : 0.0f;
    }
  }
}

__global__ void __launch_bounds__(256) evict_lens_kernel(const __grid_constant__ Evict e, int32_t* new_lens) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r < e.p.rows) new_lens[r] = min(evict_len(e.p, r), e.p.budget);
}

}  // namespace

int stream_evict(const gn_evict_params& p, int32_t* kept, int32_t* new_lens, float* mass_out, cudaStream_t st) {
  const bool over = new_lens == p.context_lens;
  Evict e{p, kept, over ? nullptr : new_lens, mass_out, 0};
  e.vec = p.head_dim % 4 == 0 && ((reinterpret_cast<uintptr_t>(p.key_pages) | reinterpret_cast<uintptr_t>(p.value_pages)) & 15) == 0;
  const int cached = p.max_context <= kCached;
  static std::atomic<uint64_t> ready{0};
  GN_TRY(prepare_kernel(ready, reinterpret_cast<const void*>(evict_select_kernel), kCached * (int)sizeof(uint32_t), kSelect, 0));
  evict_select_kernel<<<dim3(p.n_kv_head, p.rows), kSelect, cached ? p.max_context * sizeof(uint32_t) : 0, st>>>(e, cached);
  GN_LAUNCH_CHECK();
  const int most = std::min(p.budget, p.max_context);
  if (most == 0) {
    // nothing moves
  } else if (p.new_table == p.page_table) {
    GN_CUDA(launch_pdl(evict_move_kernel, dim3(ceil_div(p.head_dim, 32), p.n_kv_head, 2 * p.rows), dim3(256), 0, st, e));
  } else {
    int lanes = 1;
    while (lanes < 32 && lanes * 4 < p.head_dim) lanes *= 2;
    GN_CUDA(launch_pdl(evict_copy_kernel, dim3(ceil_div(most, 64), p.n_kv_head, 2 * p.rows), dim3(256), 0, st, e, lanes));
  }
  if (over) {
    evict_lens_kernel<<<ceil_div(p.rows, 256), 256, 0, st>>>(e, new_lens);
    GN_LAUNCH_CHECK();
  }
  return GN_OK;
}

}  // namespace gn
