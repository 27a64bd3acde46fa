// Few new tokens a row (decode steps) over a paged cache.
//
// Bound: HBM, 8 D bytes a key and kv head, each read once for all query heads of the group.  A CTA takes a range of a (row, kv head)'s
// keys; its warps walk tiles of 16 of them, each on its own, K and V going from memory to registers and nowhere else.  The products
// are m16n8k8 tf32 instructions with the keys (then the channels) as their 16 rows and the queries as their 8 columns, so that no
// row is padding: S^T = K Q^T, O^T += V^T P^T.  The order of a contraction and of the rows is free, and is chosen so that what a
// lane needs of a K or V row is contiguous.  Float32 through tf32: x = hi + lo, lo*hi + hi*lo + hi*hi; the instruction itself cuts x to hi.
// (In float32 instructions the same kernel took 126 of them a key, 106 us for 512 rows of 384 keys, issue and latency bound.)
// 512 rows of up to 384 keys, 6 heads on 2: 84 us, 304 MB read (3.6 TB/s): 12 warps an SM at 168 registers wait for memory.
// Ranges and warps are joined by their maxima; a range of its own CTA through memory.  New tokens' keys and values are read from
// where they are and written to their pages by the warp that meets them.
#include <algorithm>

#include "streaming.cuh"

namespace gn {

namespace {

constexpr int kWarps = 4;
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
__device__ __forceinline__ float cut(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }   // what tf32 keeps
__device__ __forceinline__ float nearest(float x) { return __uint_as_float((__float_as_uint(x) + 0x1000u) & 0xffffe000u); }
__device__ __forceinline__ void mma(float (&c)[4], float a0, float a1, float a2, float a3, float b0, float b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(a2)), "r"(__float_as_uint(a3)), "r"(__float_as_uint(b0)),
                 "r"(__float_as_uint(b1)));
}

// R = 8 NT query rows.  Lane = (g, t) = (lane / 4, lane % 4), as the instruction's fragments are laid out: rows g and g + 8, contraction
// indices t and t + 4, columns g of the second operand and 2 t, 2 t + 1 of the result.
template <int NT, int DP, bool MULTI>
__global__ void __launch_bounds__(32 * kWarps, NT == 1 ? 3 : 2) stream_decode_kernel(const __grid_constant__ Decode p) {
  constexpr int R = 8 * NT, PAIRS = DP / 16, EACH = DP / 8;   // float4s of a K row in a lane; channels of a V row in a lane
  __shared__ __align__(16) float room[kWarps * R * DP];
  pdl_trigger();
  float (&q_s)[NT][PAIRS][2][32][4] = *reinterpret_cast<float (*)[NT][PAIRS][2][32][4]>(room);   // queries as fragments, hi and lo
  float (&o_s)[kWarps][R][DP] = *reinterpret_cast<float (*)[kWarps][R][DP]>(room);               // at the end, the warps' results
  __shared__ __align__(16) float p_s[kWarps][kTile * R];
  __shared__ float m_s[kWarps][R], l_s[kWarps][R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const StreamRows& s = p.s;
  const int split = blockIdx.x, hk = blockIdx.y, r = blockIdx.z;
  const RowSpan sp = row_span<true>(s, r);
  if (sp.q_len == 0) return;
  const int nq = sp.q_len * s.G, first = sp.ctx - sp.q_len;
  const Range rg = seen_range(s, sp);
  const int per = ((rg.total + p.splits - 1) / p.splits + kTile - 1) / kTile * kTile, c0 = split * per, c1 = min(rg.total, c0 + per);
  const int64_t plane = (int64_t)r * s.Hkv + hk;
#pragma unroll
  for (int i = threadIdx.x; i < R * DP / 4; i += 32 * kWarps) {   // four channels a thread; rows behind the last query are zeros
    const int qi = i / (DP / 4), ch = i % (DP / 4) * 4, qt = s.by_G.of(qi);
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (qi < nq) {
      const float* src = s.q.data + token_offset<true>(s.q, r, hk * s.G + qi - qt * s.G, sp.q_begin + qt) + ch;
#pragma unroll
      for (int e = 0; e < 4; ++e) if (ch + e < s.D) x[e] = src[e] * (s.scale * kLog2e);
    }
    float* to = &q_s[qi >> 3][ch >> 4][0][(qi & 7) * 4 + ((ch & 15) >> 2)][0];
    const float4 hi = make_float4(nearest(x[0]), nearest(x[1]), nearest(x[2]), nearest(x[3]));
    *reinterpret_cast<float4*>(to) = hi;
    *reinterpret_cast<float4*>(to + 128) = make_float4(x[0] - hi.x, x[1] - hi.y, x[2] - hi.z, x[3] - hi.w);
  }
  __syncthreads();

  // where key c + lane is (lanes 0 .. 15): a slot of the pages, -1 none, -2 - i the row's new token i
  auto locate = [&](int c) {
    if (lane >= kTile || c + lane >= c1) return -1;
    const int key = key_of(rg, c + lane);
    const int at = s.by_page.of(key), page = s.table[(int64_t)r * s.width + at];
    if ((unsigned)page >= (unsigned)s.pages) return -1;
    if (p.nk.data && key >= first) return -2 - (key - first);
    return (page * s.Hkv + hk) * s.page_size + key - at * s.page_size;
  };
  auto row_of = [&](int slot, const float* pages, const gn_view& fresh) -> const float* {
    if (slot >= 0) return pages + (int64_t)slot * s.D;
    return slot == -1 ? nullptr : fresh.data + token_offset<true>(fresh, r, hk, sp.q_begin - 2 - slot);
  };
  // four channels from ch on.  With 16-byte accesses without a condition, so that all of a tile's loads are in flight at once: channels
  // behind the last read the last ones (the queries are 0 there, and such outputs are not stored), a key that is not there the first slot
  auto load4 = [&](const float* row, const float* any, int ch, float* x) {
    if (p.vec) {
      const float4 v = __ldg(reinterpret_cast<const float4*>((row ? row : any) + min(ch, s.D - 4)));
      x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = row && ch + e < s.D ? row[ch + e] : 0.0f;
    }
  };
  float kr[2][PAIRS * 4];   // rows g and g + 8 of the tile, channels 16 i + 4 t ..
  auto load_k = [&](int slots) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float* row = row_of(__shfl_sync(0xffffffffu, slots, g + 8 * u), s.pages_k, p.nk);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) load4(row, s.pages_k, 16 * i + 4 * t, &kr[u][4 * i]);
    }
  };
  float m[2 * NT], l[2 * NT], o[NT][PAIRS][4];
#pragma unroll
  for (int q = 0; q < 2 * NT; ++q) { m[q] = -INFINITY; l[q] = 0.0f; }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.0f;

  constexpr int kStride = kTile * kWarps;
  int c = c0 + warp * kTile;
  int slots = locate(c), next = locate(c + kStride);   // the table is read two tiles ahead
  for (; c < c1; c += kStride) {
    const int after = locate(c + 2 * kStride);
    load_k(slots);
    // the instruction cuts its sums off: the small terms have sums of their own, and the large ones four that are then added rounded
    float x[NT][4], big[NT][4][4], small[NT][2][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        big[nt][0][e] = big[nt][1][e] = big[nt][2][e] = big[nt][3][e] = 0.0f;
        small[nt][0][e] = small[nt][1][e] = 0.0f;
      }
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
#pragma unroll
      for (int h = 0; h < 4; h += 2) {
        const float a0 = kr[0][4 * i + h], a1 = kr[1][4 * i + h], a2 = kr[0][4 * i + h + 1], a3 = kr[1][4 * i + h + 1];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 hi = *reinterpret_cast<const float2*>(&q_s[nt][i][0][lane][h]), lo = *reinterpret_cast<const float2*>(&q_s[nt][i][1][lane][h]);
          mma(small[nt][0], a0 - cut(a0), a1 - cut(a1), a2 - cut(a2), a3 - cut(a3), hi.x, hi.y);
          mma(small[nt][1], a0, a1, a2, a3, lo.x, lo.y);
          mma(big[nt][(2 * i + h / 2) & 3], a0, a1, a2, a3, hi.x, hi.y);
        }
      }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[nt][e] = ((big[nt][0][e] + big[nt][1][e]) + (big[nt][2][e] + big[nt][3][e])) + (small[nt][0][e] + small[nt][1][e]);
    float vr[4][EACH];   // V rows t, t + 4, t + 8, t + 12, channels EACH g ..
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float* row = row_of(__shfl_sync(0xffffffffu, slots, t + 4 * u), s.pages_v, p.nv);
#pragma unroll
      for (int e = 0; e < EACH; e += 4) load4(row, s.pages_v, EACH * g + e, &vr[u][e]);
    }
    if (__any_sync(0xffffffffu, lane < kTile && slots == -1)) {   // keys of weight 0, whatever was read for them
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (__shfl_sync(0xffffffffu, slots, t + 4 * u) == -1) {
#pragma unroll
          for (int e = 0; e < EACH; ++e) vr[u][e] = 0.0f;
        }
    }
    bool odd[2] = {false, false};
    if (MULTI) {   // a value that is not finite must reach only the queries that see it
      uint32_t bad = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < EACH; ++e) if ((__float_as_uint(vr[u][e]) & 0x7f800000u) == 0x7f800000u) { any = true; vr[u][e] = 0.0f; }
        const uint32_t lanes = __ballot_sync(0xffffffffu, any);
#pragma unroll
        for (int k = 0; k < 4; ++k) if (lanes & (0x11111111u << k)) bad |= 1u << (4 * u + k);
      }
      odd[0] = (bad >> g) & 1u; odd[1] = (bad >> (g + 8)) & 1u;
    }
    float shrink[NT][2];
    const int slot_a = __shfl_sync(0xffffffffu, slots, g), slot_b = __shfl_sync(0xffffffffu, slots, g + 8);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int q = nt * 8 + 2 * t + h;
        float a = x[nt][h], b = x[nt][2 + h];
        bool see_a = slot_a != -1, see_b = slot_b != -1;
        if (MULTI) {
          const int pos = first + s.by_G.of(q);
          see_a = see_a && q < nq && sees(s, pos, key_of(rg, c + g)); see_b = see_b && q < nq && sees(s, pos, key_of(rg, c + g + 8));
        }
        if (!see_a) a = -INFINITY;
        if (!see_b) b = -INFINITY;
        x[nt][h] = a; x[nt][2 + h] = b;
        float top = fmaxf(a, b);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4)); top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(m[2 * nt + h], fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)));
        const float use = top == -INFINITY ? 0.0f : top, alpha = ex2(m[2 * nt + h] - use);
        m[2 * nt + h] = top;
        a = ex2(a - use); b = ex2(b - use);
        l[2 * nt + h] = fmaf(l[2 * nt + h], alpha, a + b);
        if (MULTI && ((odd[0] && see_a) || (odd[1] && see_b))) l[2 * nt + h] = NAN;
        p_s[warp][g * R + q] = a; p_s[warp][(g + 8) * R + q] = b;
        shrink[nt][h] = alpha;
      }
      if (p.scores) {
        float* to = p.scores + (plane * s.max_context + c + g) * R + nt * 8 + 2 * t;
        if (c + g < c1) *reinterpret_cast<float2*>(to) = make_float2(x[nt][0], x[nt][1]);
        if (c + g + 8 < c1) *reinterpret_cast<float2*>(to + 8 * R) = make_float2(x[nt][2], x[nt][3]);
      }
    }
    __syncwarp();
    float hi[2][NT][2], lo[2][NT][2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float w = p_s[warp][(8 * k + 4 * h + t) * R + nt * 8 + g];
          hi[k][nt][h] = nearest(w); lo[k][nt][h] = w - hi[k][nt][h];
        }
    // a tile's products start from zero and are added to the rescaled output rounded
#pragma unroll
    for (int j = 0; j < PAIRS; ++j)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float a0 = vr[2 * k][2 * j], a1 = vr[2 * k][2 * j + 1], a2 = vr[2 * k + 1][2 * j], a3 = vr[2 * k + 1][2 * j + 1];
          mma(y, a0 - cut(a0), a1 - cut(a1), a2 - cut(a2), a3 - cut(a3), hi[k][nt][0], hi[k][nt][1]);
          mma(y, a0, a1, a2, a3, lo[k][nt][0], lo[k][nt][1]);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) mma(y, vr[2 * k][2 * j], vr[2 * k][2 * j + 1], vr[2 * k + 1][2 * j], vr[2 * k + 1][2 * j + 1], hi[k][nt][0], hi[k][nt][1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][j][e] = fmaf(o[nt][j][e], shrink[nt][e & 1], y[e]);
      }
    __syncwarp();
    if (p.nk.data) {   // the new tokens' own: to their slots
      for (uint32_t mine = __ballot_sync(0xffffffffu, slots <= -2); mine; mine &= mine - 1) {
        const int i = __ffs(mine) - 1, slot = __shfl_sync(0xffffffffu, slots, i);
        const int64_t at = key_offset<true>(s, s.k, r, hk, key_of(rg, c + i));
        const float* from_k = row_of(slot, nullptr, p.nk);
        const float* from_v = row_of(slot, nullptr, p.nv);
        for (int e = lane; e < s.D; e += 32) { s.pages_k[at + e] = from_k[e]; s.pages_v[at + e] = from_v[e]; }
      }
    }
    slots = next; next = after;
  }
  // ------------------------------------------------------------- join the lanes, the warps
  __syncthreads();
#pragma unroll
  for (int q = 0; q < 2 * NT; ++q) {
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) l[q] += __shfl_xor_sync(0xffffffffu, l[q], d);
    const int qi = (q >> 1) * 8 + 2 * t + (q & 1);
    if (g == 0) { m_s[warp][qi] = m[q]; l_s[warp][qi] = l[q]; }
#pragma unroll
    for (int j = 0; j < PAIRS; j += 2)
      *reinterpret_cast<float4*>(&o_s[warp][qi][EACH * g + 2 * j]) =
          make_float4(o[q >> 1][j][q & 1], o[q >> 1][j][2 + (q & 1)], o[q >> 1][j + 1][q & 1], o[q >> 1][j + 1][2 + (q & 1)]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * DP; i += 32 * kWarps) {
    const int q = i / DP, ch = i % DP;
    if (q >= nq) break;
    float top = -INFINITY, sum = 0.0f, acc = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, m_s[w][q]);
    const float use = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float a = ex2(m_s[w][q] - use);
      sum = fmaf(l_s[w][q], a, sum);
      acc = fmaf(o_s[w][q][ch], a, acc);
    }
    const float y = sum == 0.0f ? 0.0f : acc / sum, L = sum == 0.0f ? -INFINITY : top + log2f(sum);
    if (p.splits > 1) {
      const int64_t at = (plane * p.splits + split) * R + q;
      p.part_o[at * DP + ch] = y;
      if (ch == 0) p.part_l[at] = L;
    } else {
      const int qt = s.by_G.of(q), h = hk * s.G + q - qt * s.G, token = sp.q_begin + qt;
      if (ch < s.D) p.out.data[token_offset<true>(p.out, r, h, token) + ch] = y;
      if (ch == 0) p.lse[stat_offset<true>(s, r, h, token)] = L * kLn2;
    }
  }
}

// A warp per query of a (row, kv head): joins the ranges.
template <int R, int DP>
__global__ void __launch_bounds__(128) stream_decode_join_kernel(const __grid_constant__ Decode p) {
  pdl_trigger();
  pdl_wait();
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
  const int qt = s.by_G.of(q), h = hk * s.G + q - qt * s.G, token = sp.q_begin + qt;
  float* dst = p.out.data + token_offset<true>(p.out, r, h, token);
  const float z = bad ? NAN : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) if (lane + 32 * e < s.D) dst[lane + 32 * e] = o[e] * z;
  if (lane == 0) p.lse[stat_offset<true>(s, r, h, token)] = bad ? NAN : sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// A thread per key: the weights that this call's queries gave it, from the kept scores and the final log-sum-exps.
template <int R>
__global__ void __launch_bounds__(256) stream_decode_mass_kernel(const __grid_constant__ Decode p) {
  pdl_wait();
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

int queries_of(const StreamRows& s) { return s.max_query * s.G <= 8 ? 8 : 16; }
int splits_of(const StreamRows& s) {
  // about two CTAs an SM, and no range below two tiles a warp.  (Eight queries leave room for three an SM: 32 rows of 8704 keys would take 76 us
  // instead of 86, 100 of 1000 41 instead of 53, 512 of 384 the same 90.)
  int64_t seen = s.max_context;
  if (s.window >= 0) seen = std::min<int64_t>(seen, (int64_t)s.window + s.sinks + s.max_query);
  const int64_t ctas = (int64_t)s.rows * s.Hkv;
  return (int)std::max<int64_t>(1, std::min<int64_t>({(2 * 148 + ctas / 2) / ctas, seen / (2 * kTile * kWarps), 128}));
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

template <int NT, int DP, bool MULTI>
int go(const Decode& d, cudaStream_t st) {
  constexpr int R = 8 * NT;
  const StreamRows& s = d.s;
  stream_decode_kernel<NT, DP, MULTI><<<dim3(d.splits, s.Hkv, s.rows), 32 * kWarps, 0, st>>>(d);
  GN_LAUNCH_CHECK();
  if (d.splits > 1) GN_CUDA(launch_pdl(stream_decode_join_kernel<R, DP>, dim3(ceil_div(s.max_query * s.G, 4), s.Hkv, s.rows), dim3(128), 0, st, d));
  if (d.mass_out && s.max_context) GN_CUDA(launch_pdl(stream_decode_mass_kernel<R>, dim3(ceil_div(s.max_context, 256), s.Hkv, s.rows), dim3(256), 0, st, d));
  return GN_OK;
}
template <int NT>
int go_rows(const Decode& d, cudaStream_t st) {
  const bool multi = d.s.max_query > 1;
  if (d.s.D <= 64) return multi ? go<NT, 64, true>(d, st) : go<NT, 64, false>(d, st);
  return multi ? go<NT, 128, true>(d, st) : go<NT, 128, false>(d, st);
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
  return queries_of(s) == 8 ? go_rows<1>(d, st) : go_rows<2>(d, st);
}

}  // namespace gn
