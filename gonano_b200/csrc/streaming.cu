// Streaming attention: the C entry points, their checks, and the copy of new tokens to their pages.
#include <algorithm>
#include <cmath>

#include "streaming_tc.cuh"

namespace gn {

namespace {

// A warp per (row, new token, kv head): the new token's key and value go to its slot.
__global__ void __launch_bounds__(128) stream_append_kernel(StreamRows s, gn_view nk, gn_view nv) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * 4 + warp, hk = blockIdx.y, r = blockIdx.z;
  const RowSpan sp = row_span<true>(s, r);
  if (t >= sp.q_len) return;
  const int pos = sp.ctx - sp.q_len + t;
  if (pos < 0) return;
  const int64_t to = key_offset<true>(s, s.k, r, hk, pos);
  if (to < 0) return;
  const float* a = nk.data + token_offset<true>(nk, r, hk, sp.q_begin + t); const float* b = nv.data + token_offset<true>(nv, r, hk, sp.q_begin + t);
  for (int c = lane; c < s.D; c += 32) { s.pages_k[to + c] = a[c]; s.pages_v[to + c] = b[c]; }
}
// A call without new tokens: every key keeps the weight that it has.
__global__ void __launch_bounds__(256) stream_keep_mass_kernel(StreamRows s, const float* mass, float* mass_out) {
  const int key = blockIdx.x * 256 + threadIdx.x, hk = blockIdx.y, r = blockIdx.z;
  if (key >= min(s.lens[r], s.max_context)) return;
  const int64_t at = ((int64_t)r * s.Hkv + hk) * s.width * s.page_size + key;
  mass_out[at] = mass ? mass[at] : 0.0f;
}
// ------------------------------------------------------------------ checks
int on_this_device(const void* p, const char* what) {
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) { cudaGetLastError(); set_error("no CUDA device available: %s", cudaGetErrorString(err)); return GN_ERR_CUDA; }
  cudaPointerAttributes at;
  err = cudaPointerGetAttributes(&at, p);
  if (err != cudaSuccess) { cudaGetLastError(); set_error("%s: %s", what, cudaGetErrorString(err)); return GN_ERR_CUDA; }
  GN_REQUIRE(at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged, "%s: not device memory", what);
  if (at.type == cudaMemoryTypeDevice && at.device != device) {
    set_error("%s: memory of device %d, but device %d is current", what, at.device, device);
    return GN_ERR_UNSUPPORTED;
  }
  return GN_OK;
}
// An output's elements must not share memory: sorted by stride, every dimension steps over the whole of the one inside it.
bool apart(const gn_view& v, int64_t batch, int64_t heads, int64_t tokens, int64_t dim) {
  int64_t n[3] = {batch, heads, tokens}, st[3] = {v.batch_stride, v.head_stride, v.token_stride};
  int order[3] = {0, 1, 2};
  std::sort(order, order + 3, [&](int a, int b) { return st[a] < st[b]; });
  int64_t extent = dim;
  for (int i : order) {
    if (n[i] <= 1) continue;
    if (st[i] < extent) return false;
    extent = st[i] * (n[i] - 1) + extent;
  }
  return true;
}
// Whether two pieces of memory have a byte in common.
bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a && b && a_bytes > 0 && b_bytes > 0 && x < y + b_bytes && y < x + a_bytes;
}
bool strides_ok(const gn_view& v) { return v.batch_stride >= 0 && v.head_stride >= 0 && v.token_stride >= 0; }

constexpr int kFar = 1 << 30;   // no sequence is longer: wider windows and more sinks are cut to it, so that sums with positions stay in 32 bits

int sink_rows(const gn_sink_params* p, StreamRows* s) {
  GN_REQUIRE(p, "attention_sink: null parameters");
  GN_REQUIRE(p->batch >= 0 && p->seq >= 0 && p->n_kv_head > 0 && p->n_head > 0 && p->n_head % p->n_kv_head == 0,
             "attention_sink: batch %d, seq %d, %d heads on %d kv heads", p->batch, p->seq, p->n_head, p->n_kv_head);
  GN_REQUIRE(p->head_dim > 0 && p->head_dim <= 128, "attention_sink: head_dim %d outside [1, 128]", p->head_dim);
  GN_REQUIRE(p->batch <= 32767 && p->n_head <= 65535, "attention_sink: more than 32767 sequences or 65535 heads");
  GN_REQUIRE(p->sinks >= 0 && std::isfinite(p->scale), "attention_sink: bad sinks or scale");
  GN_REQUIRE(strides_ok(p->query) && strides_ok(p->key) && strides_ok(p->value), "attention_sink: negative stride");
  GN_REQUIRE((int64_t)p->seq * (p->n_head / p->n_kv_head) < (1ll << 30), "attention_sink: seq x heads of a group exceeds 2^30");
  s->rows = p->batch; s->Hq = p->n_head; s->Hkv = p->n_kv_head; s->G = p->n_head / p->n_kv_head; s->by_G = FastDiv(s->G); s->D = p->head_dim;
  s->window = std::min(p->window, kFar); s->sinks = std::min(p->sinks, kFar); s->scale = p->scale; s->q = p->query; s->k = p->key; s->v = p->value; s->seq = p->seq; s->lengths = p->lengths;
  return GN_OK;
}
int sink_pointers(const gn_sink_params* p) {
  GN_REQUIRE(p->query.data && p->key.data && p->value.data, "attention_sink: null tensor");
  GN_TRY(on_this_device(p->query.data, "attention_sink: query")); GN_TRY(on_this_device(p->key.data, "attention_sink: key"));
  GN_TRY(on_this_device(p->value.data, "attention_sink: value"));
  if (p->lengths) GN_TRY(on_this_device(p->lengths, "attention_sink: lengths"));
  return GN_OK;
}
int workspace_ok(const void* w, int64_t have, int64_t need, const char* what) {
  if (need == 0) return GN_OK;
  GN_REQUIRE(w && have >= need, "%s: workspace of %lld bytes, %lld needed", what, (long long)(w ? have : 0), (long long)need);
  GN_REQUIRE((reinterpret_cast<uintptr_t>(w) & 15) == 0, "%s: workspace not 16-byte aligned", what);
  return on_this_device(w, what);
}
int64_t sink_bytes(const StreamRows& s, int backward) { return backward ? stream_tc_backward_bytes(s) : stream_tc_forward_bytes(s); }
// New tokens over a paged cache: up to 16 query rows a kv head (as many as that kernel holds) run on the kernel that streams the cache once, more
// on the tensor cores, which pack the keys first (3 times the cache's bytes) but take 128 rows for one reading.  Both at 16 rows (4 tokens, 4 heads
// on 1, 128 channels): 1 x 300 keys 29 and 35 us, 1 x 8704 41 and 51, 32 x 8704 98 and 215, 128 x 300 33 and 53; at 8 rows 32 x 8704 takes 82 and 211.
bool paged_on_tensor_cores(const StreamRows& s) { return (int64_t)s.max_query * s.G > 16; }
int64_t paged_bytes(const StreamRows& s, bool mass) { return !paged_on_tensor_cores(s) ? stream_decode_bytes(s, mass) : stream_tc_forward_bytes(s) + (mass ? stream_tc_mass_bytes(s) : 0); }

int paged_rows(const gn_paged_params* p, StreamRows* s) {
  GN_REQUIRE(p, "attention_paged: null parameters");
  GN_REQUIRE(p->rows >= 0 && p->tokens >= 0 && p->max_query >= 0 && p->n_kv_head > 0 && p->n_head > 0 && p->n_head % p->n_kv_head == 0,
             "attention_paged: rows %d, tokens %d, max_query %d, %d heads on %d kv heads", p->rows, p->tokens, p->max_query, p->n_head, p->n_kv_head);
  GN_REQUIRE(p->head_dim > 0 && p->head_dim <= 128, "attention_paged: head_dim %d outside [1, 128]", p->head_dim);
  GN_REQUIRE(p->rows <= 32767 && p->n_head <= 65535, "attention_paged: more than 32767 rows or 65535 heads");
  GN_REQUIRE(p->page_size > 0 && p->pages >= 0 && p->table_width >= 0 && (int64_t)p->table_width * p->page_size <= kFar,
             "attention_paged: pages %d of %d keys, table of %d", p->pages, p->page_size, p->table_width);
  GN_REQUIRE((int64_t)p->pages * p->n_kv_head < (1ll << 31) / p->page_size, "attention_paged: more than 2^31 slots of keys");
  GN_REQUIRE(p->max_context >= 0 && (int64_t)p->max_context <= (int64_t)p->table_width * p->page_size, "attention_paged: max_context %d, but a row of the table holds %lld keys",
             p->max_context, (long long)p->table_width * p->page_size);
  GN_REQUIRE((int64_t)p->max_query * (p->n_head / p->n_kv_head) < (1ll << 30), "attention_paged: max_query x heads of a group exceeds 2^30");
  GN_REQUIRE(p->sinks >= 0 && std::isfinite(p->scale), "attention_paged: bad sinks or scale");
  GN_REQUIRE(strides_ok(p->query) && strides_ok(p->new_key) && strides_ok(p->new_value), "attention_paged: negative stride");
  s->rows = p->rows; s->Hq = p->n_head; s->Hkv = p->n_kv_head; s->G = p->n_head / p->n_kv_head; s->by_G = FastDiv(s->G); s->D = p->head_dim;
  s->window = std::min(p->window, kFar); s->sinks = std::min(p->sinks, kFar); s->scale = p->scale; s->q = p->query;
  s->is_paged = true; s->pages_k = p->key_pages; s->pages_v = p->value_pages; s->table = p->page_table; s->starts = p->query_starts; s->lens = p->context_lens;
  s->tokens = p->tokens; s->max_query = std::min(p->max_query, p->tokens); s->max_context = p->max_context; s->page_size = p->page_size; s->by_page = FastDiv(p->page_size); s->pages = p->pages;
  s->width = p->table_width;
  return GN_OK;
}

}  // namespace
}  // namespace gn

using namespace gn;

extern "C" {

int gn_attention_sink_workspace(const gn_sink_params* p, int backward, int64_t* bytes) {
  GN_REQUIRE(bytes, "attention_sink_workspace: null bytes");
  StreamRows s;
  GN_TRY(sink_rows(p, &s));
  *bytes = s.rows && s.seq ? sink_bytes(s, backward) : 0;
  return GN_OK;
}

int gn_attention_sink_forward(const gn_sink_params* p, const gn_view* out, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  StreamRows s;
  GN_TRY(sink_rows(p, &s));
  if (!s.rows || !s.seq) return GN_OK;
  GN_TRY(sink_pointers(p));
  GN_REQUIRE(out && out->data && lse, "attention_sink_forward: null output");
  GN_REQUIRE(strides_ok(*out) && apart(*out, s.rows, s.Hq, s.seq, s.D), "attention_sink_forward: elements of out share memory");
  GN_TRY(on_this_device(out->data, "attention_sink_forward: out")); GN_TRY(on_this_device(lse, "attention_sink_forward: lse"));
  GN_TRY(workspace_ok(workspace, workspace_bytes, sink_bytes(s, 0), "attention_sink_forward"));
  return stream_tc_forward(s, *out, lse, workspace, (cudaStream_t)stream);
}

int gn_attention_sink_backward(const gn_sink_params* p, const gn_view* out, const gn_view* out_grad, const float* lse, const gn_view* dq, const gn_view* dk,
                               const gn_view* dv, int accumulate, void* workspace, int64_t workspace_bytes, void* stream) {
  StreamRows s;
  GN_TRY(sink_rows(p, &s));
  if (!s.rows || !s.seq) return GN_OK;
  GN_REQUIRE(out && out->data && out_grad && out_grad->data && lse && dq && dq->data && dk && dk->data && dv && dv->data, "attention_sink_backward: null tensor");
  GN_REQUIRE(strides_ok(*out) && strides_ok(*out_grad) && strides_ok(*dq) && strides_ok(*dk) && strides_ok(*dv), "attention_sink_backward: negative stride");
  GN_REQUIRE(apart(*dq, s.rows, s.Hq, s.seq, s.D) && apart(*dk, s.rows, s.Hkv, s.seq, s.D) && apart(*dv, s.rows, s.Hkv, s.seq, s.D),
             "attention_sink_backward: elements of a gradient share memory");
  GN_REQUIRE(dq->data != dk->data && dq->data != dv->data && dk->data != dv->data, "attention_sink_backward: two gradients share memory");
  GN_TRY(sink_pointers(p));
  const void* ptrs[] = {out->data, out_grad->data, lse, dq->data, dk->data, dv->data};
  for (const void* x : ptrs) GN_TRY(on_this_device(x, "attention_sink_backward"));
  GN_TRY(workspace_ok(workspace, workspace_bytes, sink_bytes(s, 1), "attention_sink_backward"));
  return stream_tc_backward(s, *out, *out_grad, lse, *dq, *dk, *dv, accumulate, workspace, (cudaStream_t)stream);
}

int gn_attention_paged_workspace(const gn_paged_params* p, int64_t* bytes) {
  GN_REQUIRE(bytes, "attention_paged_workspace: null bytes");
  StreamRows s;
  GN_TRY(paged_rows(p, &s));
  *bytes = s.rows && s.tokens && s.max_query ? paged_bytes(s, p->mass_out != nullptr) : 0;
  return GN_OK;
}

int gn_attention_paged(const gn_paged_params* p, const gn_view* out, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  StreamRows s;
  GN_TRY(paged_rows(p, &s));
  // in one buffer a key's weight is read and written by one thread; in two that share a piece, another key's
  const int64_t mass_bytes = (int64_t)p->rows * p->n_kv_head * p->table_width * p->page_size * 4;
  GN_REQUIRE(p->mass == p->mass_out || !overlap(p->mass, mass_bytes, p->mass_out, mass_bytes), "attention_paged: mass and mass_out share a part of their memory");
  if (s.rows && !(s.tokens && s.max_query) && p->mass_out && p->mass_out != p->mass && s.max_context) {
    GN_REQUIRE(p->context_lens, "attention_paged: null context_lens");
    for (const void* x : {(const void*)p->context_lens, (const void*)p->mass, (const void*)p->mass_out}) if (x) GN_TRY(on_this_device(x, "attention_paged"));
    stream_keep_mass_kernel<<<dim3(ceil_div(s.max_context, 256), s.Hkv, s.rows), 256, 0, (cudaStream_t)stream>>>(s, p->mass, p->mass_out);
    GN_LAUNCH_CHECK();
  }
  if (!s.rows || !s.tokens || !s.max_query) return GN_OK;
  GN_REQUIRE(p->query.data && p->query_starts && p->context_lens && out && out->data && lse, "attention_paged: null argument");
  GN_REQUIRE(p->max_context == 0 || (p->key_pages && p->value_pages && p->page_table), "attention_paged: null pages");
  GN_REQUIRE((p->new_key.data == nullptr) == (p->new_value.data == nullptr), "attention_paged: new_key and new_value come together");
  GN_REQUIRE(!p->mass || p->mass_out, "attention_paged: mass without mass_out");
  GN_REQUIRE(strides_ok(*out) && apart(*out, 1, s.Hq, s.tokens, s.D), "attention_paged: elements of out share memory");
  // the queries are read a second time for the weights, new tokens by the blocks of other heads
  GN_REQUIRE((out->data != p->query.data || !p->mass_out) && out->data != p->new_key.data && out->data != p->new_value.data, "attention_paged: out shares memory with an input");
  const void* ptrs[] = {p->query.data, p->query_starts, p->context_lens, out->data, lse, p->key_pages, p->value_pages, p->page_table, p->new_key.data,
                        p->new_value.data, p->mass, p->mass_out};
  for (const void* x : ptrs) if (x) GN_TRY(on_this_device(x, "attention_paged"));
  GN_TRY(workspace_ok(workspace, workspace_bytes, paged_bytes(s, p->mass_out != nullptr), "attention_paged"));
  cudaStream_t st = (cudaStream_t)stream;
  if (!paged_on_tensor_cores(s)) return stream_decode(s, p->new_key, p->new_value, *out, lse, p->mass, p->mass_out, workspace, st);
  if (p->new_key.data && s.max_context) {
    stream_append_kernel<<<dim3(ceil_div(s.max_query, 4), s.Hkv, s.rows), 128, 0, st>>>(s, p->new_key, p->new_value);
    GN_LAUNCH_CHECK();
  }
  PackedKeys packed;
  GN_TRY(stream_tc_forward(s, *out, lse, workspace, st, &packed));
  if (!p->mass_out || !s.max_context) return GN_OK;
  return stream_tc_mass(s, packed, lse, p->mass, p->mass_out, static_cast<uint8_t*>(workspace) + stream_tc_forward_bytes(s), st);
}

int gn_cache_evict(const gn_evict_params* p, int32_t* kept, int32_t* new_lens, float* mass_out, void* stream) {
  GN_REQUIRE(p, "cache_evict: null parameters");
  GN_REQUIRE(p->rows >= 0 && p->rows <= 32767 && p->n_kv_head > 0 && p->n_kv_head <= 65535 && p->head_dim > 0 && p->page_size > 0 && p->pages >= 0 && p->table_width >= 0 && p->new_width >= 0,
             "cache_evict: bad shape");
  GN_REQUIRE(p->budget >= 0 && p->sinks >= 0 && p->recent >= 0 && (int64_t)p->sinks + p->recent <= p->budget, "cache_evict: sinks %d + recent %d exceed the budget %d",
             p->sinks, p->recent, p->budget);
  GN_REQUIRE((int64_t)p->table_width * p->page_size <= kFar && p->budget <= kFar, "cache_evict: a table of %lld keys a row or a budget of %d exceeds 2^30",
             (long long)p->table_width * p->page_size, p->budget);   // indices that step over them stay in 32 bits
  GN_REQUIRE(p->max_context >= 0 && (int64_t)p->max_context <= (int64_t)p->table_width * p->page_size && p->max_context <= p->mass_stride,
             "cache_evict: max_context %d, but a row holds %lld keys and %d masses", p->max_context, (long long)p->table_width * p->page_size, p->mass_stride);
  GN_REQUIRE((int64_t)p->new_width * p->page_size >= std::min(p->budget, p->max_context), "cache_evict: new_table holds %lld keys a row, %d are kept",
             (long long)p->new_width * p->page_size, std::min(p->budget, p->max_context));
  if (!p->rows) return GN_OK;
  GN_REQUIRE(p->context_lens && new_lens && (p->budget == 0 || kept), "cache_evict: null argument");
  GN_REQUIRE(p->max_context == 0 || (p->key_pages && p->value_pages && p->mass && p->page_table && (p->new_table || p->budget == 0)), "cache_evict: null argument");
  // Blocks write the outputs while others still read the inputs.  (Lengths written over those that are read are left to the end.)
  const int64_t planes = (int64_t)p->rows * p->n_kv_head, store = (int64_t)p->pages * p->n_kv_head * p->page_size * p->head_dim * 4;
  const struct { const char* name; const void* at; int64_t bytes; } outs[] = {{"kept", kept, planes * p->budget * 4}, {"new_lens", new_lens, p->rows * 4ll},
                                                                              {"mass_out", mass_out, planes * p->budget * 4}},
      ins[] = {{"context_lens", p->context_lens, p->rows * 4ll}, {"mass", p->mass, planes * p->mass_stride * 4}, {"page_table", p->page_table, (int64_t)p->rows * p->table_width * 4},
               {"new_table", p->new_table, (int64_t)p->rows * p->new_width * 4}, {"key_pages", p->key_pages, store}, {"value_pages", p->value_pages, store}};
  for (int i = 0; i < 3; ++i) {
    for (const auto& in : ins) GN_REQUIRE((outs[i].at == new_lens && in.at == new_lens) || !overlap(outs[i].at, outs[i].bytes, in.at, in.bytes), "cache_evict: %s shares memory with %s", outs[i].name, in.name);
    for (int j = 0; j < i; ++j) GN_REQUIRE(!overlap(outs[i].at, outs[i].bytes, outs[j].at, outs[j].bytes), "cache_evict: %s shares memory with %s", outs[i].name, outs[j].name);
  }
  const void* ptrs[] = {p->context_lens, new_lens, kept, p->key_pages, p->value_pages, p->mass, p->page_table, p->new_table, mass_out};
  for (const void* x : ptrs) if (x) GN_TRY(on_this_device(x, "cache_evict"));
  return stream_evict(*p, kept, new_lens, mass_out, (cudaStream_t)stream);
}

}  // extern "C"
