// Streaming attention (include/gonano_cuda.h): what its kernels share.
#pragma once
#include "common.cuh"

namespace gn {

// Division of 0 <= n < 2^31 by a number that a launch fixes: the high half of n m, m = floor(2^(31 + s) / d) + 1, 2^(s - 1) < d <= 2^s.
// (The error of m, below 2^-31 of it, moves n m / 2^(31 + s) by less than 1 / d, so the floor is exact.)
struct FastDiv {
  uint32_t d = 1, m = 0; int s = 0;
  FastDiv() = default;
  explicit FastDiv(int64_t by) : d((uint32_t)by) {
    while ((1ll << s) < by) ++s;
    m = s == 0 ? 0u : (uint32_t)((1ull << (31 + s)) / d + 1);
  }
#ifdef __CUDACC__
  __device__ __forceinline__ int of(int n) const { return s == 0 ? n : (int)(__umulhi((uint32_t)n, m) >> (s - 1)); }
#endif
};

// The rows (sequences) of a call, padded batch or paged cache, as the kernels see them.
struct StreamRows {
  int rows = 0, Hq = 0, Hkv = 0, G = 0, D = 0, window = -1, sinks = 0;
  FastDiv by_G, by_page;
  float scale = 1.0f;
  gn_view q{}, k{}, v{};            // k, v: padded batch
  // padded batch: `seq` tokens a row, lengths nullable
  int seq = 0;
  const int32_t* lengths = nullptr;
  // paged cache
  bool is_paged = false;
  float* pages_k = nullptr; float* pages_v = nullptr;
  const int32_t* table = nullptr; const int32_t* starts = nullptr; const int32_t* lens = nullptr;
  int tokens = 0, max_query = 0, max_context = 0, page_size = 1, pages = 0, width = 0;
  bool paged() const { return is_paged; }   // not by the pages' address: a workspace may be asked for before there are pages, and an empty pool has none
};

// Few new tokens a row over a paged cache (streaming_decode.cu): max_query * G <= 16.  Appends, attends and gathers the mass.
int64_t stream_decode_bytes(const StreamRows& s, bool mass);
int stream_decode(const StreamRows& s, const gn_view& nk, const gn_view& nv, const gn_view& out, float* lse, const float* mass, float* mass_out, void* workspace,
                  cudaStream_t st);

// Eviction (streaming_evict.cu), arguments checked.
int stream_evict(const gn_evict_params& p, int32_t* kept, int32_t* new_lens, float* mass_out, cudaStream_t st);

#ifdef __CUDACC__
struct RowSpan { int q_begin, q_len, ctx; };   // the row's first token, its new tokens, its keys

template <bool PAGED>
__device__ __forceinline__ RowSpan row_span(const StreamRows& s, int r) {
  if (!PAGED) {
    const int n = s.lengths ? min(max(s.lengths[r], 0), s.seq) : s.seq;
    return {0, n, n};
  }
  // offsets and lengths are device data: cut to what the buffers hold
  const int b = min(max(s.starts[r], 0), s.tokens), e = min(max(s.starts[r + 1], b), s.tokens);
  return {b, min(e - b, s.max_query), min(max(s.lens[r], 0), s.max_context)};
}
// Key j of row r, kv head hk; null when its page does not exist.
template <bool PAGED>
__device__ __forceinline__ int64_t key_offset(const StreamRows& s, const gn_view& view, int r, int hk, int j) {
  if (!PAGED) return (int64_t)r * view.batch_stride + (int64_t)hk * view.head_stride + (int64_t)j * view.token_stride;
  const int at = s.by_page.of(j), page = s.table[(int64_t)r * s.width + at];
  if ((unsigned)page >= (unsigned)s.pages) return -1;
  return (((int64_t)page * s.Hkv + hk) * s.page_size + j - at * s.page_size) * s.D;
}
template <bool PAGED>
__device__ __forceinline__ int64_t token_offset(const gn_view& view, int r, int h, int token) {
  return (PAGED ? 0 : (int64_t)r * view.batch_stride) + (int64_t)h * view.head_stride + (int64_t)token * view.token_stride;
}
// lse and other per-(token, head) numbers: [batch, heads, seq] or [tokens, heads]
template <bool PAGED>
__device__ __forceinline__ int64_t stat_offset(const StreamRows& s, int r, int h, int token) {
  return PAGED ? (int64_t)token * s.Hq + h : ((int64_t)r * s.Hq + h) * s.seq + token;
}
__device__ __forceinline__ bool sees(const StreamRows& s, int pos, int j) {
  return j <= pos && (s.window < 0 || pos - j <= s.window || j < s.sinks);
}
#endif

}  // namespace gn
