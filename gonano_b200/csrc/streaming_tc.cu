// Streaming attention forward on the 5th-generation tensor cores: padded batches, and chunks of new tokens over paged caches.
//
// Keys and values are packed once per call (streaming_tc.cuh); then one CTA takes 128 query rows of a (row, kv head) - the heads of
// a group side by side, row f = token * group + head, so that a key tile serves all of them - and walks the keys that any of
// them sees, 128 at a time.  The sinks and the window are two runs of keys that meet inside a tile, so the gap costs nothing.
#include <algorithm>

#include "streaming_tc.cuh"

namespace gn {

namespace {

// ------------------------------------------------------------------ packing
// Which keys of a row its new tokens can see at all: [0, sinks) and [begin, ctx), both widened to the eights that are copied.
template <bool PAGED>
__device__ __forceinline__ int first_needed(const StreamRows& s, const RowSpan& sp) {
  if (!PAGED || s.window < 0) return 0;
  return (int)max((int64_t)0, (int64_t)sp.ctx - sp.q_len - s.window) & ~7;
}
template <bool PAGED>
__device__ __forceinline__ bool is_needed(const StreamRows& s, const RowSpan& sp, int begin, int j) { return j < sp.ctx && (j >= begin || (j & ~7) < s.sinks); }

// Half a warp per key: lane i holds channels 4 i .. 4 i + 3 and, for 128 channels, 64 + 4 i ...
template <int CB, bool PAGED>
__device__ __forceinline__ bool load_key(const StreamRows& s, bool value, bool vec, int r, int hk, int j, float (&x)[4 * CB]) {
  const int l16 = threadIdx.x & 15;
  const int64_t off = key_offset<PAGED>(s, value ? s.v : s.k, r, hk, j);
#pragma unroll
  for (int e = 0; e < 4 * CB; ++e) x[e] = 0.0f;
  if (PAGED && off < 0) return false;
  const float* p = (PAGED ? (value ? s.pages_v : s.pages_k) : (value ? s.v.data : s.k.data)) + off;
#pragma unroll
  for (int b = 0; b < CB; ++b) {
    const int c = b * 64 + l16 * 4;
    if (vec) {
      if (c < s.D) {
        const float4 v = *reinterpret_cast<const float4*>(p + c);
        x[4 * b] = v.x; x[4 * b + 1] = v.y; x[4 * b + 2] = v.z; x[4 * b + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) if (c + e < s.D) x[4 * b + e] = p[c + e];
    }
  }
  return true;
}

constexpr int kPackRows = 128;   // keys of a CTA (256 threads, 16 half warps, 8 keys each)

template <int CB, bool PAGED>
__global__ void __launch_bounds__(256) stream_amax_kernel(const __grid_constant__ StreamRows s, PackedKeys pk, int vec) {
  const int hk = blockIdx.y, r = blockIdx.z >> 1, value = blockIdx.z & 1, half = threadIdx.x >> 4;
  const RowSpan sp = row_span<PAGED>(s, r);
  const int begin = first_needed<PAGED>(s, sp), j0 = blockIdx.x * kPackRows;
  if (j0 >= sp.ctx) return;
  uint32_t top = 0;
#pragma unroll 4
  for (int u = 0; u < kPackRows / 16; ++u) {
    const int j = j0 + u * 16 + half;
    if (!is_needed<PAGED>(s, sp, begin, j)) continue;
    float x[4 * CB];
    load_key<CB, PAGED>(s, value, vec, r, hk, j, x);
#pragma unroll
    for (int e = 0; e < 4 * CB; ++e) if (finite_bits(x[e])) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0 && top) atomicMax(pk.amax + ((int64_t)r * s.Hkv + hk) * 2 + value, top);   // a maximum does not depend on the order
}

template <int CB, bool PAGED>
__global__ void __launch_bounds__(256) stream_pack_kernel(const __grid_constant__ StreamRows s, PackedKeys pk, uint32_t* norms, int vec) {
  const int hk = blockIdx.y, r = blockIdx.z >> 1, value = blockIdx.z & 1, half = threadIdx.x >> 4, l16 = threadIdx.x & 15;
  const RowSpan sp = row_span<PAGED>(s, r);
  const int begin = first_needed<PAGED>(s, sp), j0 = blockIdx.x * kPackRows;
  const Packed& dst = value ? pk.v : pk.k;
  const int last = min(dst.rows, (sp.ctx + 15) / 16 * 16 + 16);   // zero rows behind the sequence: a tile is copied in 16s
  if (j0 >= last) return;
  const int64_t plane = (int64_t)r * s.Hkv + hk;
  uint8_t* base = dst.data + plane * dst.plane_bytes(CB);
  uint8_t* flags = (value ? pk.flags_v : pk.flags_k) + plane * dst.rows;
  float sc, inv;
  plane_scale(pk.amax[plane * 2 + value], sc, inv);
  float top = 0.0f;
#pragma unroll 2
  for (int u = 0; u < kPackRows / 16; ++u) {
    const int j = j0 + u * 16 + half;
    float x[4 * CB];
#pragma unroll
    for (int e = 0; e < 4 * CB; ++e) x[e] = 0.0f;
    uint8_t flag = 0;
    const bool needed = is_needed<PAGED>(s, sp, begin, j);
    if (needed && !load_key<CB, PAGED>(s, value, vec, r, hk, j, x)) flag = kAbsent;
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 4 * CB; ++e) if (!finite_bits(x[e])) { odd = true; x[e] = 0.0f; }
    const uint32_t odds = __ballot_sync(0xffffffffu, odd);
    if ((odds >> (threadIdx.x & 16)) & 0xffffu) flag |= kOdd;
    if (norms && value) {
      float sq = 0.0f;
#pragma unroll
      for (int e = 0; e < 4 * CB; ++e) sq = fmaf(x[e] * sc, x[e] * sc, sq);
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, d);
      top = fmaxf(top, sq);
    }
    if (j >= last || (!needed && j < sp.ctx)) continue;
#pragma unroll
    for (int b = 0; b < CB; ++b) {
      uint2 hi, lo;
      split_f16(x[4 * b] * sc, x[4 * b + 1] * sc, hi.x, lo.x);
      split_f16(x[4 * b + 2] * sc, x[4 * b + 3] * sc, hi.y, lo.y);
      uint8_t* at = base + ((int64_t)b * 2 * dst.rows + j) * 128 + ((((l16 >> 1) ^ (j & 7)) << 4) | ((l16 & 1) << 3));
      *reinterpret_cast<uint2*>(at) = hi;
      *reinterpret_cast<uint2*>(at + (int64_t)dst.rows * 128) = lo;
    }
    if (l16 == 0) {
      flags[j] = flag;
      if (flag) pk.odd[plane] = 1;
    }
  }
  if (norms && value) {
    top = warp_max(top);
    if ((threadIdx.x & 31) == 0 && top > 0.0f) atomicMax(norms + plane * 2, __float_as_uint(top));
  }
}

// ------------------------------------------------------------------ forward
struct ForwardTc {
  StreamRows s;
  PackedKeys pk;
  gn_view out;
  float* lse;
  int vec_q, vec_out, tiles, splits;
  float* part_o; float* part_l;   // splits > 1: [plane][tile][split][128] rows of DP channels, and their log2-sum-exps
};

constexpr int kRowsT = 128;      // query rows of a CTA = keys of a tile = UMMA M and N
constexpr int kThreads = 320;    // 8 softmax warps, the issuing warp, the copying warp

// One CTA per (128 query rows, kv head, row, key split), 320 threads:
//   warps 0-7  two threads per query row, 64 keys of a tile and half the channels each.  They convert Q once (raw float32 rows to
//              the swizzled hi / lo tile), then per tile read S from tensor memory, take the running maximum, and write
//              2^15 p as f16 pairs over the scores they came from: P is the A operand of O = P V straight from tensor memory.
//              Each tile's O starts from zero in one of two buffers and is added to float32 registers one tile later, where the
//              rescaling by the grown maximum costs nothing extra: sums over many keys are rounded, not cut off.
//   warp 8     issues S_{j+1} = Q K^T (24 instructions of 128 x 128 x 16), then O_j = P_j V, so that the tensor pipe works on the
//              next scores while the softmax threads work on these;
//   warp 9     copies K and V tiles (bulk copies of packed rows) as their buffers fall free.
// Tensor memory: two score / weight buffers of 128 columns, two O buffers of 128.  Shared memory: Q, K, V tiles, hi and lo.
// Bound: 48 instructions of 64 cycles a tile = 3072 cycles of tensor pipe.  Every wait is bounded; a kernel whose wait ran out
// writes NaN.
template <int DP, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1) stream_tc_forward_kernel(const __grid_constant__ ForwardTc p) {
  constexpr int CB = DP / 64, HC = DP / 2, STAGES = DP == 64 ? 2 : 1;
  constexpr uint32_t TILE = CB * 32768u, OFF_K = TILE, OFF_V = TILE + STAGES * TILE, BARS = OFF_V + STAGES * TILE, XCH = BARS + 256;
  extern __shared__ uint8_t smem_raw[];
  const StreamRows& s = p.s;
  const int hk = blockIdx.y, r = blockIdx.z, sp_i = blockIdx.x % p.splits, tile = p.tiles - 1 - (int)blockIdx.x / p.splits;   // the long tiles first
  const RowSpan sp = row_span<PAGED>(s, r);
  const int f0 = tile * kRowsT, nf = sp.q_len * s.G;
  if (f0 >= (PAGED ? nf : s.seq * s.G)) return;
  const int first = sp.ctx - sp.q_len;   // position of the row's first new token
  KeyRuns runs{0, 0, 0};
  if (f0 < nf) runs = key_runs(s, first + f0 / s.G, first + min(f0 + kRowsT - 1, nf - 1) / s.G);
  const int all = (runs.total + kRowsT - 1) / kRowsT, per = (all + p.splits - 1) / p.splits;
  const int j0 = sp_i * per, n = max(0, min(all, j0 + per) - j0);
  const int64_t plane = (int64_t)r * s.Hkv + hk;

  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + BARS;
  const uint32_t q_full = bars;
  auto k_full = [&](int i) { return bars + 8u + 8u * i; };
  auto k_empty = [&](int i) { return bars + 24u + 8u * i; };
  auto v_full = [&](int i) { return bars + 40u + 8u * i; };
  auto v_empty = [&](int i) { return bars + 56u + 8u * i; };
  auto s_full = [&](int i) { return bars + 72u + 8u * i; };
  auto p_full = [&](int i) { return bars + 88u + 8u * i; };
  auto o_full = [&](int i) { return bars + 104u + 8u * i; };
  auto o_empty = [&](int i) { return bars + 120u + 8u * i; };
  const uint32_t tmem_slot = bars + 136;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 256);
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full(i), 1); mbar_init(k_empty(i), 1); mbar_init(v_full(i), 1); mbar_init(v_empty(i), 1);
      mbar_init(s_full(i), 1); mbar_init(p_full(i), 256); mbar_init(o_full(i), 1); mbar_init(o_empty(i), 256);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gen + BARS + 136);
  auto rows16 = [&](int j) { return min(kRowsT, (runs.total - (j0 + j) * kRowsT + 15) & ~15); };   // keys of tile j, in 16s

  if (warp == 9) {
    // ------------------------------------------------------------- copies
    if (lane == 0) {
      bool ok = true;
      auto copy_tile = [&](const Packed& src, uint32_t dst, uint32_t bar, int j) {
        const int c0 = (j0 + j) * kRowsT, rows = rows16(j), na = min(max(runs.a_len - c0, 0), rows), nb = rows - na;
        const uint8_t* from = src.data + plane * src.plane_bytes(CB);
        mbar_expect_tx(bar, (uint32_t)CB * 2u * rows * 128u);
#pragma unroll
        for (int b = 0; b < CB * 2; ++b) {
          if (na) bulk_load(dst + b * 16384, from + ((int64_t)b * src.rows + c0) * 128, na * 128, bar);
          if (nb) bulk_load(dst + b * 16384 + na * 128, from + ((int64_t)b * src.rows + c0 + na + runs.shift) * 128, nb * 128, bar);
        }
      };
      int jk = 0, jv = 0;
      for (uint32_t idle = 0; jv < n && ok;) {   // whichever buffer is free next
        bool did = false;
        if (jk < n && (jk < STAGES || mbar_test(k_empty(jk % STAGES), (jk / STAGES - 1) & 1))) {
          copy_tile(p.pk.k, base + OFF_K + (jk % STAGES) * TILE, k_full(jk % STAGES), jk);
          ++jk; did = true;
        }
        if (jv < jk && (jv < STAGES || mbar_test(v_empty(jv % STAGES), (jv / STAGES - 1) & 1))) {
          copy_tile(p.pk.v, base + OFF_V + (jv % STAGES) * TILE, v_full(jv % STAGES), jv);
          ++jv; did = true;
        }
        if (did) idle = 0;
        else if (++idle > kSpinLimit) ok = false;
        else if (idle > 4096) __nanosleep(64);
      }
      if (!ok)   // copies in flight land before the CTA goes
        for (int st = 0; st < STAGES; ++st)
          for (int ph = 0; ph < 2; ++ph) { mbar_wait(k_full(st), ph); mbar_wait(v_full(st), ph); }
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------- instructions
    if (lane == 0 && n > 0) {
      bool ok = mbar_wait(q_full, 0);
      auto scores = [&](int j) {
        const int st = j % STAGES;
        ok = ok && mbar_wait(k_full(st), (j / STAGES) & 1);
        if (!ok) return;
        tc_fence_after();
        const uint32_t d = tmem + (j & 1) * 128, id = instr_desc_f16(128, rows16(j), 0);
        const uint32_t q = base, k = base + OFF_K + st * TILE;
        auto one = [&](int ks, int ql, int kl, uint32_t acc) {
          const uint32_t in = (ks >> 2) * 32768u;
          umma_f16(d, smem_desc_sw128(q + in + ql * 16384) + 2u * (ks & 3), smem_desc_sw128(k + in + kl * 16384) + 2u * (ks & 3), id, acc);
        };
#pragma unroll
        for (int ks = 0; ks < CB * 4; ++ks) { one(ks, 1, 0, ks > 0); one(ks, 0, 1, 1); }
#pragma unroll
        for (int ks = 0; ks < CB * 4; ++ks) one(ks, 0, 0, 1);
        umma_commit(k_empty(st));
        umma_commit(s_full(j & 1));
      };
      scores(0);
      for (int j = 0; j < n && ok; ++j) {
        if (j + 1 < n) scores(j + 1);
        const int st = j % STAGES, b = j & 1;
        ok = ok && mbar_wait(p_full(b), (j >> 1) & 1) && mbar_wait(v_full(st), (j / STAGES) & 1) && (j < 2 || mbar_wait(o_empty(b), ((j >> 1) - 1) & 1));
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + 256 + b * 128, w = tmem + b * 128, id = instr_desc_f16(128, DP, 1), v = base + OFF_V + st * TILE;
        const int slices = rows16(j) >> 4;
        auto one = [&](int ks, int wl, int vl, uint32_t acc) {
          umma_f16_ts(d, w + (ks >> 2) * 64 + wl * 32 + (ks & 3) * 8, smem_desc_mn(v + vl * 16384 + ks * 2048, 32768), id, acc);
        };
        for (int ks = 0; ks < slices; ++ks) { one(ks, 1, 0, ks > 0); one(ks, 0, 1, 1); }
        for (int ks = 0; ks < slices; ++ks) one(ks, 0, 0, 1);
        umma_commit(v_empty(st));
        umma_commit(o_full(b));
      }
    }
  } else {
    // ------------------------------------------------------------- softmax threads
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    float* xch = reinterpret_cast<float*>(gen + XCH);
    auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); };   // the two warps of these 32 rows
    const int f = f0 + row;
    const bool live = f < nf;
    const int t = f / s.G, g = f - t * s.G, token = sp.q_begin + t, pos = first + t;
    float c = 0.0f;   // from products of scaled operands to log2 units
    if (n > 0) {
      float x[HC];
      const float* src = s.q.data + token_offset<PAGED>(s.q, r, hk * s.G + g, token);
#pragma unroll
      for (int e = 0; e < HC; e += 4) {
        const int ch = half * HC + e;
        if (p.vec_q) {
          float4 v = make_float4(0, 0, 0, 0);
          if (live && ch < s.D) v = *reinterpret_cast<const float4*>(src + ch);
          x[e] = v.x; x[e + 1] = v.y; x[e + 2] = v.z; x[e + 3] = v.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[e + i] = (live && ch + i < s.D) ? src[ch + i] : 0.0f;
        }
      }
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < HC; ++e) if (finite_bits(x[e])) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
      reinterpret_cast<uint32_t*>(xch)[half * 128 + row] = top;
      meet();
      top = max(top, reinterpret_cast<uint32_t*>(xch)[(half ^ 1) * 128 + row]);
      float sq, iq, sk, ik;
      plane_scale(top, sq, iq);
      plane_scale(p.pk.amax[plane * 2], sk, ik);
      // a negative scale goes into Q, so that larger products are larger scores; a vanishing one stays a positive number
      c = fmaxf(fabsf(s.scale) * kLog2e * iq * ik, 1e-30f);
      if (s.scale < 0.0f) sq = -sq;
#pragma unroll
      for (int e = 0; e < HC; e += 8) {
        uint4 hi, lo;
        split_f16(x[e] * sq, x[e + 1] * sq, hi.x, lo.x); split_f16(x[e + 2] * sq, x[e + 3] * sq, hi.y, lo.y);
        split_f16(x[e + 4] * sq, x[e + 5] * sq, hi.z, lo.z); split_f16(x[e + 6] * sq, x[e + 7] * sq, hi.w, lo.w);
        const int ch = half * HC + e;
        uint8_t* at = gen + (ch >> 6) * 32768 + row * 128 + ((((ch & 63) >> 3) ^ (row & 7)) << 4);
        *reinterpret_cast<uint4*>(at) = hi;
        *reinterpret_cast<uint4*>(at + 16384) = lo;
      }
      fence_async_smem();
      mbar_arrive(q_full);
      meet();   // xch is read before it is used again
    }
    // what the row sees, in virtual keys: [0, s_end) and [lo, hi]
    const int s_end = live ? max(0, min(s.sinks, pos + 1)) : 0;
    const int lo_key = live ? (s.window < 0 ? 0 : max(0, pos - s.window)) - runs.shift : 0, hi_key = live ? pos - runs.shift : -1;
    const bool odd_plane = n > 0 && p.pk.odd[plane] != 0;
    float m = -INFINITY, l = 0.0f, alpha_prev = 0.0f;
    bool ok = true, poison = false;
    float o[HC];
#pragma unroll
    for (int e = 0; e < HC; ++e) o[e] = 0.0f;
    auto gather = [&](int j, float alpha) {   // O += tile j's, against the maximum that tile j used
      ok = ok && mbar_wait(o_full(j & 1), (j >> 1) & 1);
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < HC / 32; ++h) {
        uint32_t y[32];
        tmem_ld32(lane_addr + 256 + (j & 1) * 128 + half * HC + h * 32, y);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) o[h * 32 + e] = fmaf(o[h * 32 + e], alpha, __uint_as_float(y[e]));
      }
      tc_fence_before();
      mbar_arrive(o_empty(j & 1));
    };
    for (int j = 0; j < n; ++j) {
      ok = ok && mbar_wait(s_full(j & 1), (j >> 1) & 1);
      tc_fence_after();
      float x[64];
      {
        uint32_t y[32];
        tmem_ld32(lane_addr + (j & 1) * 128 + half * 64, y);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = __uint_as_float(y[e]);
        tmem_ld32(lane_addr + (j & 1) * 128 + half * 64 + 32, y);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) x[32 + e] = __uint_as_float(y[e]);
      }
      const int c0 = (j0 + j) * kRowsT + half * 64;
      uint64_t see = bits_below(s_end - c0) | (bits_below(hi_key + 1 - c0) & ~bits_below(lo_key - c0));
      if (odd_plane) {
        for (int e = 0; e < 64; ++e)
          if ((see >> e) & 1ull) {
            const int key = c0 + e < runs.a_len ? c0 + e : c0 + e + runs.shift;
            const uint8_t flag = p.pk.flags_k[plane * p.pk.k.rows + key] | p.pk.flags_v[plane * p.pk.v.rows + key];
            if (flag & kAbsent) see &= ~(1ull << e);
            else if (flag & kOdd) poison = true;
          }
      }
      if (__any_sync(0xffffffffu, see != ~0ull)) {
        const uint32_t s0 = (uint32_t)see, s1 = (uint32_t)(see >> 32);
#pragma unroll
        for (int e = 0; e < 32; ++e) { if (!((s0 >> e) & 1u)) x[e] = -INFINITY; if (!((s1 >> e) & 1u)) x[32 + e] = -INFINITY; }
      }
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 64; ++e) top = fmaxf(top, x[e]);
      xch[half * 128 + row] = top;
      meet();
      top = fmaxf(top, xch[(half ^ 1) * 128 + row]);
      const float m_new = fmaxf(m, top == -INFINITY ? -INFINITY : top * c), m_use = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = exp2_fast(m - m_use), off = kWeightShift - m_use;
      m = m_new;
      float sum = 0.0f;
      {
        uint32_t hi[32], lo[32];
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
          const float a = exp2_fast(fmaf(x[e], c, off)), b = exp2_fast(fmaf(x[e + 1], c, off));
          sum += a + b;
          split_f16(a, b, hi[e >> 1], lo[e >> 1]);
        }
        tmem_st32(lane_addr + (j & 1) * 128 + half * 64, hi);
        tmem_st32(lane_addr + (j & 1) * 128 + half * 64 + 32, lo);
        tmem_st_wait();
      }
      tc_fence_before();
      mbar_arrive(p_full(j & 1));
      l = fmaf(l, alpha, sum);
      if (j > 0) gather(j - 1, alpha_prev);
      alpha_prev = alpha;
      meet();   // both have read xch
    }
    if (n > 0) gather(n - 1, alpha_prev);
    // ------------------------------------------------------------- result
    xch[half * 128 + row] = l;
    xch[256 + half * 128 + row] = (poison || !ok) ? 1.0f : 0.0f;
    meet();
    const float sum = xch[row] + xch[128 + row];
    const bool bad = xch[256 + row] + xch[384 + row] > 0.0f;
    float sv, iv;
    plane_scale(n > 0 ? p.pk.amax[plane * 2 + 1] : 0u, sv, iv);
    const float z = bad ? NAN : sum == 0.0f ? 0.0f : iv / sum;
    const float L = bad ? NAN : sum == 0.0f ? -INFINITY : m - kWeightShift + log2f(sum);
    if (p.splits > 1) {
      const int64_t at = ((plane * p.tiles + tile) * p.splits + sp_i) * kRowsT + row;
#pragma unroll
      for (int e = 0; e < HC; e += 4) *reinterpret_cast<float4*>(p.part_o + at * DP + half * HC + e) = make_float4(o[e] * z, o[e + 1] * z, o[e + 2] * z, o[e + 3] * z);
      if (half == 0) p.part_l[at] = L;
    } else if (f < (PAGED ? nf : s.seq * s.G)) {
      float* dst = p.out.data + token_offset<PAGED>(p.out, r, hk * s.G + g, token);
#pragma unroll
      for (int e = 0; e < HC; e += 4) {
        const int ch = half * HC + e;
        if (p.vec_out) {
          if (ch < s.D) *reinterpret_cast<float4*>(dst + ch) = make_float4(o[e] * z, o[e + 1] * z, o[e + 2] * z, o[e + 3] * z);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) if (ch + i < s.D) dst[ch + i] = o[e + i] * z;
        }
      }
      if (half == 0) p.lse[stat_offset<PAGED>(s, r, hk * s.G + g, token)] = L * kLn2;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

// Joins the key splits of a row: a warp per query row.
template <int DP, bool PAGED>
__global__ void __launch_bounds__(256) stream_tc_combine_kernel(const __grid_constant__ ForwardTc p) {
  const StreamRows& s = p.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hk = blockIdx.y, r = blockIdx.z, f = blockIdx.x * 8 + warp;
  const RowSpan sp = row_span<PAGED>(s, r);
  if (f >= (PAGED ? sp.q_len : s.seq) * s.G) return;
  const int64_t plane = (int64_t)r * s.Hkv + hk, at = ((plane * p.tiles + f / kRowsT) * p.splits) * kRowsT + f % kRowsT;
  float top = -INFINITY;
  bool bad = false;
  for (int i = 0; i < p.splits; ++i) { const float x = p.part_l[at + (int64_t)i * kRowsT]; bad |= isnan(x); top = fmaxf(top, x); }
  float sum = 0.0f, o[DP / 32];
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) o[e] = 0.0f;
  if (top != -INFINITY)
    for (int i = 0; i < p.splits; ++i) {
      const float w = exp2f(p.part_l[at + (int64_t)i * kRowsT] - top);
      sum += w;
#pragma unroll
      for (int e = 0; e < DP / 32; ++e) o[e] = fmaf(w, p.part_o[(at + (int64_t)i * kRowsT) * DP + lane + 32 * e], o[e]);
    }
  const int t = f / s.G, h = hk * s.G + f % s.G, token = sp.q_begin + t;
  float* dst = p.out.data + token_offset<PAGED>(p.out, r, h, token);
  const float z = bad ? NAN : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) if (lane + 32 * e < s.D) dst[lane + 32 * e] = o[e] * z;
  if (lane == 0) p.lse[stat_offset<PAGED>(s, r, h, token)] = bad ? NAN : sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// ------------------------------------------------------------------ host
struct Plan { int DP, tiles, splits; int64_t planes, max_q, max_k; };
Plan plan_forward(const StreamRows& s) {
  Plan pl;
  pl.DP = s.D <= 64 ? 64 : 128;
  pl.planes = (int64_t)s.rows * s.Hkv;
  pl.max_q = s.paged() ? s.max_query : s.seq;
  pl.max_k = s.paged() ? s.max_context : s.seq;
  pl.tiles = ceil_div(pl.max_q * s.G, kRowsT);
  // Splitting the keys of a tile: only while there are fewer CTAs than SMs, and no finer than four key tiles a CTA (a split
  // repeats the conversion of Q and adds a pass over the partial results).
  int64_t seen = pl.max_k;
  if (s.window >= 0) seen = std::min<int64_t>(seen, (int64_t)s.window + s.sinks + kRowsT / s.G + 1);
  const int64_t ctas = pl.planes * pl.tiles;
  pl.splits = (int)std::max<int64_t>(1, std::min<int64_t>({148 / std::max<int64_t>(ctas, 1), ceil_div(seen, 4 * kRowsT), 64}));
  return pl;
}
int64_t carve_forward(const StreamRows& s, const Plan& pl, void* workspace, ForwardTc* f) {
  Carve c{static_cast<uint8_t*>(workspace)};
  const int rows = packed_rows(pl.max_k);
  PackedKeys& pk = f->pk;
  pk.amax = c.take<uint32_t>(pl.planes * 3);   // amax and odd in one piece: cleared together
  pk.odd = reinterpret_cast<int*>(pk.amax + pl.planes * 2);
  pk.k.rows = pk.v.rows = rows;
  pk.k.data = c.take<uint8_t>(pl.planes * pk.k.plane_bytes(pl.DP / 64));
  pk.v.data = c.take<uint8_t>(pl.planes * pk.v.plane_bytes(pl.DP / 64));
  pk.flags_k = c.take<uint8_t>(pl.planes * rows);
  pk.flags_v = c.take<uint8_t>(pl.planes * rows);
  if (pl.splits > 1) {
    f->part_o = c.take<float>(pl.planes * pl.tiles * pl.splits * kRowsT * pl.DP);
    f->part_l = c.take<float>(pl.planes * pl.tiles * pl.splits * kRowsT);
  }
  return c.used;
}
bool vec_keys(const StreamRows& s) {
  if (!s.paged()) return vec_view(s.k, s.D) && vec_view(s.v, s.D);
  return s.D % 4 == 0 && ((reinterpret_cast<uintptr_t>(s.pages_k) | reinterpret_cast<uintptr_t>(s.pages_v)) & 15) == 0;
}

template <int CB, bool PAGED>
int pack_go(const StreamRows& s, const PackedKeys& pk, uint32_t* norms, cudaStream_t st) {
  const int vec = vec_keys(s), keys = pk.k.rows;
  stream_amax_kernel<CB, PAGED><<<dim3(ceil_div(keys, kPackRows), s.Hkv, 2 * s.rows), 256, 0, st>>>(s, pk, vec);
  GN_LAUNCH_CHECK();
  stream_pack_kernel<CB, PAGED><<<dim3(ceil_div(keys, kPackRows), s.Hkv, 2 * s.rows), 256, 0, st>>>(s, pk, norms, vec);
  GN_LAUNCH_CHECK();
  return GN_OK;
}

template <int DP, bool PAGED>
int forward_go(const StreamRows& s, const Plan& pl, ForwardTc& f, cudaStream_t st) {
  constexpr int CB = DP / 64, STAGES = DP == 64 ? 2 : 1;
  constexpr int kSmem = CB * 32768 * (1 + 2 * STAGES) + 256 + 2048 + 1024;
  GN_CUDA(cudaMemsetAsync(f.pk.amax, 0, pl.planes * 3 * sizeof(uint32_t), st));
  GN_TRY(stream_pack_keys(s, f.pk, nullptr, st));
  static PerDeviceOnce once;
  if (once.first()) GN_CUDA(cudaFuncSetAttribute(stream_tc_forward_kernel<DP, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  stream_tc_forward_kernel<DP, PAGED><<<dim3(pl.tiles * pl.splits, s.Hkv, s.rows), kThreads, kSmem, st>>>(f);
  GN_LAUNCH_CHECK();
  if (pl.splits > 1) {
    stream_tc_combine_kernel<DP, PAGED><<<dim3(ceil_div(pl.max_q * s.G, 8), s.Hkv, s.rows), 256, 0, st>>>(f);
    GN_LAUNCH_CHECK();
  }
  return GN_OK;
}

}  // namespace

int stream_pack_keys(const StreamRows& s, const PackedKeys& pk, uint32_t* norms, cudaStream_t st) {
  if (s.D <= 64) return s.paged() ? pack_go<1, true>(s, pk, norms, st) : pack_go<1, false>(s, pk, norms, st);
  return s.paged() ? pack_go<2, true>(s, pk, norms, st) : pack_go<2, false>(s, pk, norms, st);
}

int64_t stream_tc_forward_bytes(const StreamRows& s) {
  ForwardTc f{};
  return carve_forward(s, plan_forward(s), nullptr, &f);
}
int stream_tc_forward(const StreamRows& s, const gn_view& out, float* lse, void* workspace, cudaStream_t st) {
  const Plan pl = plan_forward(s);
  ForwardTc f{};
  f.s = s; f.out = out; f.lse = lse; f.tiles = pl.tiles; f.splits = pl.splits;
  carve_forward(s, pl, workspace, &f);
  f.vec_q = vec_view(s.q, s.D); f.vec_out = vec_view(out, s.D);
  if (pl.DP == 64) return s.paged() ? forward_go<64, true>(s, pl, f, st) : forward_go<64, false>(s, pl, f, st);
  return s.paged() ? forward_go<128, true>(s, pl, f, st) : forward_go<128, false>(s, pl, f, st);
}

}  // namespace gn
