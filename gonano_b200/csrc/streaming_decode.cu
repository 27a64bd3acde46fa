// Few new tokens a row (decode steps) over a paged cache, in float32.
//
// Bound: HBM, 8 D bytes a key and kv head, each read once for all query heads of the group.  A CTA takes a range of a (row, kv head)'s
// keys; its warps walk tiles of 16 of them, each on its own.  Scores: two lanes a key, half the channels each, the K tile in shared
// memory (asynchronous copies one tile ahead, 16-byte chunks swizzled so that 8 lanes meet no bank twice), the queries broadcast
// from shared memory: one shuffle a score, 4 multiplications per word read.  Output: lane = 4 channels, V rows straight from global memory
// (8 ahead), the weights broadcast.  Ranges and warps are joined by their maxima; a range of its own CTA through memory.
// New tokens' keys and values are read from where they are and written to their pages by the warp that meets them.
#include <algorithm>

#include "streaming.cuh"

namespace gn {

namespace {

constexpr int kWarps = 4;   // 3 CTAs of 4 warps (16 KB of K tiles each) an SM; 2 of 3 with tiles of 32 keys: half as fast, a CTA's start and end show
constexpr int kTile = 16;   // keys of a warp's tile
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Decode {
  StreamRows s;
  gn_view nk, nv, out;   // nk.data null: nothing to append
  float* lse;
  int splits, vec;
  float* part_o; float* part_l;    // splits > 1: [plane][split][R] rows of DP channels, log2-sum-exps
  float* scores;                   // null, or [plane][max_context][R] scores in log2 units, by virtual key
  const float* mass; float* mass_out;
};

// The keys that a row's new tokens see: [0, sinks) and [begin, ctx), the second at virtual keys sinks ...
struct Range { int sinks, begin, total; };
__device__ __forceinline__ Range seen_range(const StreamRows& s, const RowSpan& sp) {
  Range g;
  const int first = sp.ctx - sp.q_len;
  g.begin = s.window < 0 ? 0 : (int)max((int64_t)0, (int64_t)first - s.window);
  g.sinks = min(s.sinks, g.begin);
  g.total = g.sinks + max(0, sp.ctx - g.begin);
  return g;
}
__device__ __forceinline__ int key_of(const Range& g, int c) { return c < g.sinks ? c : g.begin + c - g.sinks; }

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <int R, int DP, bool MULTI>
__global__ void __launch_bounds__(32 * kWarps) stream_decode_kernel(const __grid_constant__ Decode p) {
  constexpr int ROWB = DP * 4, CH = DP / 4, LANES = DP / 4;   // LANES lanes hold a row's channels
  constexpr int STEP = 32 / LANES;                            // V rows of a load
  extern __shared__ __align__(16) float smem[];
  float* q_s = smem;                                           // [R][DP]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* p_s = smem + R * DP + warp * kTile * R;               // [kTile][R]
  float* k_s = smem + R * DP + kWarps * kTile * R + warp * 2 * kTile * DP;
  const StreamRows& s = p.s;
  const int split = blockIdx.x, hk = blockIdx.y, r = blockIdx.z;
  const RowSpan sp = row_span<true>(s, r);
  if (sp.q_len == 0) return;
  const int nq = sp.q_len * s.G, first = sp.ctx - sp.q_len;
  const Range rg = seen_range(s, sp);
  const int per = ((rg.total + p.splits - 1) / p.splits + kTile - 1) / kTile * kTile, c0 = split * per, c1 = min(rg.total, c0 + per);
  const int64_t plane = (int64_t)r * s.Hkv + hk;
  for (int i = threadIdx.x; i < R * DP; i += 32 * kWarps) {
    const int qi = i / DP, ch = i % DP;
    q_s[i] = qi < nq && ch < s.D ? s.q.data[token_offset<true>(s.q, r, hk * s.G + qi % s.G, sp.q_begin + qi / s.G) + ch] * (s.scale * kLog2e) : 0.0f;
  }
  __syncthreads();

  // where key c + lane is (16 lanes): its K and V rows (null: none, or no such page)
  auto locate = [&](int c, const float*& kp, const float*& vp) {
    kp = vp = nullptr;
    if (lane >= kTile || c + lane >= c1) return;
    const int key = key_of(rg, c + lane);
    const int64_t at = key_offset<true>(s, s.k, r, hk, key);
    if (at < 0) return;
    kp = s.pages_k + at; vp = s.pages_v + at;
    if (p.nk.data && key >= first) {
      kp = p.nk.data + token_offset<true>(p.nk, r, hk, sp.q_begin + key - first);
      vp = p.nv.data + token_offset<true>(p.nv, r, hk, sp.q_begin + key - first);
    }
  };
  auto fetch = [&](int buf, int c, const float* kp) {
    if (c < c1) {
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(k_s + buf * kTile * DP);
#pragma unroll 8
    for (int i = 0; i < kTile; i += STEP) {
      const int row = i + lane / LANES, ch = lane % LANES;
      const float* src = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(kp), row));
      const uint32_t at = dst + row * ROWB + ((ch ^ (row & 7)) << 4);
      if (p.vec) {
        copy16(at, src ? src + min(ch * 4, s.D - 4) : s.pages_k, src && ch * 4 < s.D ? 16 : 0);   // no bytes: zeros
      } else {
        float4 v = make_float4(0, 0, 0, 0);
        if (src) {
          if (ch * 4 < s.D) v.x = src[ch * 4];
          if (ch * 4 + 1 < s.D) v.y = src[ch * 4 + 1];
          if (ch * 4 + 2 < s.D) v.z = src[ch * 4 + 2];
          if (ch * 4 + 3 < s.D) v.w = src[ch * 4 + 3];
        }
        *reinterpret_cast<float4*>(reinterpret_cast<uint8_t*>(k_s) + buf * kTile * ROWB + row * ROWB + ((ch ^ (row & 7)) << 4)) = v;
      }
    }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float m[R], l[R], o[R][4];
#pragma unroll
  for (int q = 0; q < R; ++q) { m[q] = -INFINITY; l[q] = 0.0f; o[q][0] = o[q][1] = o[q][2] = o[q][3] = 0.0f; }
  // rows are located two tiles ahead (the table's latency), K tiles copied one ahead
  const float *kp, *vrow, *k_next, *v_next, *k_after, *v_after;
  constexpr int kStride = kTile * kWarps;
  int c = c0 + warp * kTile, buf = 0;
  locate(c, kp, vrow);
  locate(c + kStride, k_next, v_next);
  fetch(0, c, kp);
  for (; c < c1; c += kStride, buf ^= 1, kp = k_next, vrow = v_next, k_next = k_after, v_next = v_after) {
    fetch(buf ^ 1, c + kStride, k_next);
    locate(c + 2 * kStride, k_after, v_after);
    const bool valid = kp != nullptr;
    const int key = key_of(rg, c + lane);   // of the first 16 lanes, which locate
    if (p.nk.data) {   // the new tokens' own: to their slots
      for (uint32_t mine = __ballot_sync(0xffffffffu, valid && key >= first); mine; mine &= mine - 1) {
        const int i = __ffs(mine) - 1;
        const float* from_k = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(kp), i));
        const float* from_v = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(vrow), i));
        const int64_t at = key_offset<true>(s, s.k, r, hk, __shfl_sync(0xffffffffu, key, i));
        for (int e = lane; e < s.D; e += 32) { s.pages_k[at + e] = from_k[e]; s.pages_v[at + e] = from_v[e]; }
      }
    }
    // V rows of the first loads are on their way while the scores are computed
    constexpr int AHEAD = 8;
    auto load_v = [&](int i, float4& v) {
      const int row = i * STEP + lane / LANES, ch = (lane % LANES) * 4;
      const float* src = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(vrow), row));
      v = make_float4(0, 0, 0, 0);
      if (!src) return;
      if (p.vec) { if (ch < s.D) v = __ldg(reinterpret_cast<const float4*>(src + ch)); return; }
      if (ch < s.D) v.x = src[ch];
      if (ch + 1 < s.D) v.y = src[ch + 1];
      if (ch + 2 < s.D) v.z = src[ch + 2];
      if (ch + 3 < s.D) v.w = src[ch + 3];
    };
    float4 v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load_v(i, v[i]);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    float x[R];
#pragma unroll
    for (int q = 0; q < R; ++q) x[q] = 0.0f;
    const int mine = lane >> 1, half = lane & 1;   // this lane's key and half of its channels
    const float4* kt = reinterpret_cast<const float4*>(k_s + buf * kTile * DP + mine * DP);
#pragma unroll 4
    for (int i = 0; i < CH / 2; ++i) {
      const int ch = half ? CH / 2 + (i ^ 4) : i;   // the halves four chunks apart: other banks
      const float4 k = kt[ch ^ (mine & 7)];
#pragma unroll
      for (int q = 0; q < R; ++q) {
        const float4 y = *reinterpret_cast<const float4*>(q_s + q * DP + ch * 4);
        x[q] = fmaf(k.x, y.x, fmaf(k.y, y.y, fmaf(k.z, y.z, fmaf(k.w, y.w, x[q]))));
      }
    }
    const bool there = __shfl_sync(0xffffffffu, (int)valid, mine) != 0;
    const int my_key = MULTI ? __shfl_sync(0xffffffffu, key, mine) : 0;
    float alpha[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      x[q] += __shfl_xor_sync(0xffffffffu, x[q], 1);
      bool see = there;
      if (MULTI) see = see && q < nq && sees(s, first + q / s.G, my_key);
      if (!see) x[q] = -INFINITY;
      const float top = fmaxf(m[q], warp_max(x[q])), use = top == -INFINITY ? 0.0f : top;
      alpha[q] = ex2(m[q] - use);
      m[q] = top;
      const float w = ex2(x[q] - use);
      l[q] = fmaf(l[q], alpha[q], half ? 0.0f : w);
      if (!half) p_s[mine * R + q] = w;
    }
    if (p.scores && !half && c + mine < c1) {
      float* to = p.scores + (plane * s.max_context + c + mine) * R;
#pragma unroll
      for (int q = 0; q < R; q += 4) *reinterpret_cast<float4*>(to + q) = make_float4(x[q], x[q + 1], x[q + 2], x[q + 3]);
    }
    __syncwarp();
#pragma unroll
    for (int q = 0; q < R; ++q) { o[q][0] *= alpha[q]; o[q][1] *= alpha[q]; o[q][2] *= alpha[q]; o[q][3] *= alpha[q]; }
    constexpr int LOADS = kTile / STEP;
#pragma unroll 1
    for (int i0 = 0; i0 < LOADS; i0 += AHEAD) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const float4 y = v[i];
        if (i0 + AHEAD < LOADS) load_v(i0 + AHEAD + i, v[i]);
        const float* w = p_s + ((i0 + i) * STEP + lane / LANES) * R;
#pragma unroll
        for (int q = 0; q < R; q += 4) {
          const float4 w4 = *reinterpret_cast<const float4*>(w + q);
          const float ww[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (MULTI && ww[u] == 0.0f) continue;   // a query that does not see the key is not touched by what its value holds
            o[q + u][0] = fmaf(ww[u], y.x, o[q + u][0]); o[q + u][1] = fmaf(ww[u], y.y, o[q + u][1]);
            o[q + u][2] = fmaf(ww[u], y.z, o[q + u][2]); o[q + u][3] = fmaf(ww[u], y.w, o[q + u][3]);
          }
        }
      }
    }
    __syncwarp();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  // ------------------------------------------------------------- join the lanes, the warps
#pragma unroll
  for (int q = 0; q < R; ++q) {
    l[q] = warp_sum(l[q]);
#pragma unroll
    for (int d = LANES; d < 32; d <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[q][e] += __shfl_xor_sync(0xffffffffu, o[q][e], d);
  }
  __syncthreads();   // the tiles are no longer read
  float* o_s = smem + R * DP + kWarps * kTile * R;   // [warp][R][DP]
  float* ml = p_s;                                 // [R] maxima, [R] sums
#pragma unroll
  for (int q = 0; q < R; ++q) {
    if (lane < LANES) *reinterpret_cast<float4*>(o_s + (warp * R + q) * DP + lane * 4) = make_float4(o[q][0], o[q][1], o[q][2], o[q][3]);
    if (lane == 0) { ml[q] = m[q]; ml[R + q] = l[q]; }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * DP; i += 32 * kWarps) {
    const int q = i / DP, ch = i % DP;
    if (q >= nq) break;
    const float* all = smem + R * DP;
    float top = -INFINITY, sum = 0.0f, acc = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, all[w * kTile * R + q]);
    const float use = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float a = ex2(all[w * kTile * R + q] - use);
      sum = fmaf(all[w * kTile * R + R + q], a, sum);
      acc = fmaf(o_s[(w * R + q) * DP + ch], a, acc);
    }
    const float y = sum == 0.0f ? 0.0f : acc / sum, L = sum == 0.0f ? -INFINITY : top + log2f(sum);
    if (p.splits > 1) {
      const int64_t at = (plane * p.splits + split) * R + q;
      p.part_o[at * DP + ch] = y;
      if (ch == 0) p.part_l[at] = L;
    } else {
      const int h = hk * s.G + q % s.G, token = sp.q_begin + q / s.G;
      if (ch < s.D) p.out.data[token_offset<true>(p.out, r, h, token) + ch] = y;
      if (ch == 0) p.lse[stat_offset<true>(s, r, h, token)] = L * kLn2;
    }
  }
}

// A warp per query of a (row, kv head): joins the ranges.
template <int R, int DP>
__global__ void __launch_bounds__(128) stream_decode_join_kernel(const __grid_constant__ Decode p) {
  const StreamRows& s = p.s;
  const int q = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, hk = blockIdx.y, r = blockIdx.z;
  const RowSpan sp = row_span<true>(s, r);
  if (q >= sp.q_len * s.G) return;
  const int64_t plane = (int64_t)r * s.Hkv + hk, at = plane * p.splits * R + q;
  float top = -INFINITY;
  bool bad = false;
  for (int i = lane; i < p.splits; i += 32) { const float x = p.part_l[at + (int64_t)i * R]; bad |= isnan(x); top = fmaxf(top, x); }
  top = warp_max(top);
  bad = __any_sync(0xffffffffu, bad);
  float sum = 0.0f, o[DP / 32];
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) o[e] = 0.0f;
  if (top != -INFINITY)
#pragma unroll 4
    for (int i = 0; i < p.splits; ++i) {
      const float w = ex2(p.part_l[at + (int64_t)i * R] - top);
      sum += w;
#pragma unroll
      for (int e = 0; e < DP / 32; ++e) o[e] = fmaf(w, p.part_o[(at + (int64_t)i * R) * DP + lane + 32 * e], o[e]);
    }
  const int h = hk * s.G + q % s.G, token = sp.q_begin + q / s.G;
  float* dst = p.out.data + token_offset<true>(p.out, r, h, token);
  const float z = bad ? NAN : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) if (lane + 32 * e < s.D) dst[lane + 32 * e] = o[e] * z;
  if (lane == 0) p.lse[stat_offset<true>(s, r, h, token)] = bad ? NAN : sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// A thread per key: the weights that this call's queries gave it, from the kept scores and the final log-sum-exps.
template <int R>
__global__ void __launch_bounds__(256) stream_decode_mass_kernel(const __grid_constant__ Decode p) {
  const StreamRows& s = p.s;
  __shared__ float L[R];
  const int key = blockIdx.x * 256 + threadIdx.x, hk = blockIdx.y, r = blockIdx.z;
  const RowSpan sp = row_span<true>(s, r);
  if ((int)blockIdx.x * 256 >= sp.ctx) return;
  const int nq = sp.q_len * s.G, first = sp.ctx - sp.q_len;
  if (threadIdx.x < R) L[threadIdx.x] = threadIdx.x < nq ? p.lse[stat_offset<true>(s, r, hk * s.G + threadIdx.x % s.G, sp.q_begin + threadIdx.x / s.G)] * kLog2e : 0.0f;
  __syncthreads();
  if (key >= sp.ctx) return;
  const Range rg = seen_range(s, sp);
  const int64_t plane = (int64_t)r * s.Hkv + hk, at = plane * s.width * s.page_size + key;
  float sum = 0.0f;
  if (nq > 0 && (key < rg.sinks || key >= rg.begin)) {
    const float* x = p.scores + (plane * s.max_context + (key < rg.sinks ? key : key - rg.begin + rg.sinks)) * R;
    float y[R];
#pragma unroll
    for (int q = 0; q < R; q += 4) *reinterpret_cast<float4*>(y + q) = *reinterpret_cast<const float4*>(x + q);
#pragma unroll
    for (int q = 0; q < R; ++q) if (q < nq && y[q] != -INFINITY) sum += ex2(y[q] - L[q]);
  }
  p.mass_out[at] = (p.mass && key < first ? p.mass[at] : 0.0f) + sum;
}

int queries_of(const StreamRows& s) { const int n = s.max_query * s.G; return n <= 4 ? 4 : n <= 8 ? 8 : 16; }
int splits_of(const StreamRows& s) {
  // about as many CTAs as the machine holds at once, and no range below two tiles a warp
  int64_t seen = s.max_context;
  if (s.window >= 0) seen = std::min<int64_t>(seen, (int64_t)s.window + s.sinks + s.max_query);
  const int64_t ctas = (int64_t)s.rows * s.Hkv;
  return (int)std::max<int64_t>(1, std::min<int64_t>({(3 * 148 + ctas / 2) / ctas, seen / (2 * kTile * kWarps), 128}));
}
int64_t carve(const StreamRows& s, bool mass, uint8_t* base, Decode* d) {
  const int R = queries_of(s), DP = s.D <= 64 ? 64 : 128;
  const int64_t planes = (int64_t)s.rows * s.Hkv;
  int64_t used = 0;
  auto take = [&](int64_t floats) {
    float* at = base ? reinterpret_cast<float*>(base + used) : nullptr;
    used += (floats * 4 + 127) / 128 * 128;
    return at;
  };
  d->splits = splits_of(s);
  if (d->splits > 1) { d->part_o = take(planes * d->splits * R * DP); d->part_l = take(planes * d->splits * R); }
  if (mass) d->scores = take(planes * s.max_context * R);
  return used;
}

template <int R, int DP, bool MULTI>
int go(const Decode& d, cudaStream_t st) {
  constexpr int kSmem = (R * DP + kWarps * kTile * R + kWarps * 2 * kTile * DP) * 4;
  const StreamRows& s = d.s;
  static PerDeviceOnce once;
  if (once.first()) GN_CUDA(cudaFuncSetAttribute(stream_decode_kernel<R, DP, MULTI>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  stream_decode_kernel<R, DP, MULTI><<<dim3(d.splits, s.Hkv, s.rows), 32 * kWarps, kSmem, st>>>(d);
  GN_LAUNCH_CHECK();
  if (d.splits > 1) {
    stream_decode_join_kernel<R, DP><<<dim3(ceil_div(s.max_query * s.G, 4), s.Hkv, s.rows), 128, 0, st>>>(d);
    GN_LAUNCH_CHECK();
  }
  if (d.mass_out && s.max_context) {
    stream_decode_mass_kernel<R><<<dim3(ceil_div(s.max_context, 256), s.Hkv, s.rows), 256, 0, st>>>(d);
    GN_LAUNCH_CHECK();
  }
  return GN_OK;
}
template <int R>
int go_rows(const Decode& d, cudaStream_t st) {
  const bool multi = d.s.max_query > 1;
  if (d.s.D <= 64) return multi ? go<R, 64, true>(d, st) : go<R, 64, false>(d, st);
  return multi ? go<R, 128, true>(d, st) : go<R, 128, false>(d, st);
}

}  // namespace

int64_t stream_decode_bytes(const StreamRows& s, bool mass) {
  Decode d{};
  return carve(s, mass, nullptr, &d);
}
int stream_decode(const StreamRows& s, const gn_view& nk, const gn_view& nv, const gn_view& out, float* lse, const float* mass, float* mass_out, void* workspace,
                  cudaStream_t st) {
  Decode d{};
  d.s = s; d.nk = nk; d.nv = nv; d.out = out; d.lse = lse; d.mass = mass; d.mass_out = mass_out;
  carve(s, mass_out != nullptr, static_cast<uint8_t*>(workspace), &d);
  auto wide = [&](const gn_view& v) { return (reinterpret_cast<uintptr_t>(v.data) & 15) == 0 && v.head_stride % 4 == 0 && v.token_stride % 4 == 0; };
  d.vec = s.D % 4 == 0 && ((reinterpret_cast<uintptr_t>(s.pages_k) | reinterpret_cast<uintptr_t>(s.pages_v)) & 15) == 0 && (!nk.data || (wide(nk) && wide(nv)));
  switch (queries_of(s)) {
    case 4: return go_rows<4>(d, st);
    case 8: return go_rows<8>(d, st);
    default: return go_rows<16>(d, st);
  }
}

}  // namespace gn
