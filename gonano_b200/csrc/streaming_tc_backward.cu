// Streaming attention backward on the 5th-generation tensor cores, padded batches.
//
// With P = exp(s - lse), dS = P (dO.V - delta), delta = dO.O:  dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K.  Two kernels,
// one that keeps 128 keys and walks the query rows that see them (dK, dV), one that keeps 128 query rows and walks their keys (dQ);
// both recompute S and dO.V.  That is seven products instead of five, and no sum depends on an order: no atomics.
// As in the forward pass the heads of a group are rows side by side (f = token * group + head), so the sum over a group's heads
// that dK and dV want is part of the contraction, and the query rows that see key j are one run [j G, (j + window + 1) G).
//
// Operands are f16 pairs (streaming_tc.cuh).  dS has no bound known before the call; |dO.V - delta| <= 2 max|dO| max|V| (row norms,
// found while packing) gives the power of two that keeps it in f16's range.  A query row with a non-finite component gets
// NaN for its lse, which reaches exactly the gradients of what it sees.
#include <algorithm>

#include "streaming_tc.cuh"

namespace gn {

namespace {

struct BackwardTc {
  StreamRows s;
  PackedKeys pk;
  Packed q, g;                   // queries and dO, rows f
  uint32_t* qamax;               // [plane][2]: q, dO
  uint32_t* norms;               // [plane][2]: largest squared norm of a scaled row of V, dO
  float* off; float* delta;      // [plane][q.rows]: 15 - lse in log2 units; delta times the scales of dO and V
  gn_view out, dout, dq, dk, dv;
  const float* lse;
  int accumulate, vec_in, vec_dq, vec_dkv;
  int q_tiles, key_tiles, sink_tiles, parts_sink, parts, units;
  float* part;                   // [plane][unit][dV, dK][128][DP] of key tiles in several parts
};

constexpr int kWholePlaneQ = 256;   // planes up to here are one CTA's
constexpr int kPackRowsQ = 64;   // 256 threads, 16 half warps

// Half a warp per query row f: channels 4 i .. of the 64-channel blocks.
template <int CB>
__device__ __forceinline__ void load_query_row(const StreamRows& s, const gn_view& v, int vec, int r, int hk, int f, float (&x)[4 * CB]) {
  const int l16 = threadIdx.x & 15, t = f / s.G, h = hk * s.G + f - t * s.G;
  const float* p = v.data + token_offset<false>(v, r, h, t);
#pragma unroll
  for (int b = 0; b < CB; ++b) {
    const int c = b * 64 + l16 * 4;
    if (vec) {
      float4 y = make_float4(0, 0, 0, 0);
      if (c < s.D) y = *reinterpret_cast<const float4*>(p + c);
      x[4 * b] = y.x; x[4 * b + 1] = y.y; x[4 * b + 2] = y.z; x[4 * b + 3] = y.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * b + e] = c + e < s.D ? p[c + e] : 0.0f;
    }
  }
}

template <int CB>
__global__ void __launch_bounds__(256) stream_query_amax_kernel(const __grid_constant__ BackwardTc p) {
  const StreamRows& s = p.s;
  const int hk = blockIdx.y, r = blockIdx.z, half = threadIdx.x >> 4, f0 = blockIdx.x * kPackRowsQ;
  const int nf = row_span<false>(s, r).q_len * s.G;
  if (f0 >= nf) return;
  uint32_t top[2] = {0, 0};
#pragma unroll
  for (int u = 0; u < kPackRowsQ / 16; ++u) {
    const int f = f0 + u * 16 + half;
    if (f >= nf) continue;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float x[4 * CB];
      load_query_row<CB>(s, w ? p.dout : s.q, p.vec_in, r, hk, f, x);
#pragma unroll
      for (int e = 0; e < 4 * CB; ++e) if (finite_bits(x[e])) top[w] = max(top[w], __float_as_uint(x[e]) & 0x7fffffffu);
    }
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint32_t x = __reduce_max_sync(0xffffffffu, top[w]);
    if ((threadIdx.x & 31) == 0 && x) atomicMax(p.qamax + ((int64_t)r * s.Hkv + hk) * 2 + w, x);
  }
}

// Packs q and dO and leaves each row's lse and delta in the form that the kernels use.
template <int CB>
__global__ void __launch_bounds__(256) stream_query_pack_kernel(const __grid_constant__ BackwardTc p, int whole) {
  const StreamRows& s = p.s;
  const int hk = blockIdx.y, r = blockIdx.z, half = threadIdx.x >> 4, l16 = threadIdx.x & 15, f0 = blockIdx.x * kPackRowsQ;
  const int nf = row_span<false>(s, r).q_len * s.G, last = min(p.q.rows, (nf + 15) / 16 * 16 + 16);
  if (f0 >= last) return;
  const int64_t plane = (int64_t)r * s.Hkv + hk;
  __shared__ uint32_t most[2], norm;
  if (whole) {   // the plane is this CTA's: its largest magnitudes first
    if (threadIdx.x == 0) most[0] = most[1] = norm = 0;
    __syncthreads();
    uint32_t top[2] = {0, 0};
    for (int f = half; f < nf; f += 16)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        float x[4 * CB];
        load_query_row<CB>(s, w ? p.dout : s.q, p.vec_in, r, hk, f, x);
#pragma unroll
        for (int e = 0; e < 4 * CB; ++e) if (finite_bits(x[e])) top[w] = max(top[w], __float_as_uint(x[e]) & 0x7fffffffu);
      }
#pragma unroll
    for (int w = 0; w < 2; ++w) if (top[w]) atomicMax(&most[w], top[w]);
    __syncthreads();
    if (threadIdx.x < 2) p.qamax[plane * 2 + threadIdx.x] = most[threadIdx.x];
  }
  float sc[2], inv, sv;
  plane_scale(whole ? most[0] : p.qamax[plane * 2], sc[0], inv);
  plane_scale(whole ? most[1] : p.qamax[plane * 2 + 1], sc[1], inv);
  plane_scale(p.pk.amax[plane * 2 + 1], sv, inv);
  float top = 0.0f;
  const int steps = whole ? (last + 15) / 16 : kPackRowsQ / 16;
#pragma unroll 1
  for (int u = 0; u < steps; ++u) {
    const int f = f0 + u * 16 + half;
    float x[2][4 * CB], delta = 0.0f, sq = 0.0f;
    bool odd = false;
#pragma unroll
    for (int e = 0; e < 4 * CB; ++e) x[0][e] = x[1][e] = 0.0f;
    if (f < nf) {
      load_query_row<CB>(s, s.q, p.vec_in, r, hk, f, x[0]);
      load_query_row<CB>(s, p.dout, p.vec_in, r, hk, f, x[1]);
      float o[4 * CB];
      load_query_row<CB>(s, p.out, p.vec_in, r, hk, f, o);
#pragma unroll
      for (int e = 0; e < 4 * CB; ++e) delta = fmaf(x[1][e], o[e], delta);
    }
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int e = 0; e < 4 * CB; ++e) {
        if (!finite_bits(x[w][e])) { odd = true; x[w][e] = 0.0f; }
        x[w][e] *= sc[w];
        if (w == 1) sq = fmaf(x[w][e], x[w][e], sq);
      }
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) { delta += __shfl_xor_sync(0xffffffffu, delta, d); sq += __shfl_xor_sync(0xffffffffu, sq, d); }
    top = fmaxf(top, sq);
    odd = ((__ballot_sync(0xffffffffu, odd) >> (threadIdx.x & 16)) & 0xffffu) != 0;
    if (f >= last) continue;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const Packed& dst = w ? p.g : p.q;
#pragma unroll
      for (int b = 0; b < CB; ++b) {
        uint2 hi, lo;
        split_f16(x[w][4 * b], x[w][4 * b + 1], hi.x, lo.x);
        split_f16(x[w][4 * b + 2], x[w][4 * b + 3], hi.y, lo.y);
        uint8_t* at = dst.data + plane * dst.plane_bytes(CB) + ((int64_t)b * 2 * dst.rows + f) * 128 + ((((l16 >> 1) ^ (f & 7)) << 4) | ((l16 & 1) << 3));
        *reinterpret_cast<uint2*>(at) = hi;
        *reinterpret_cast<uint2*>(at + (int64_t)dst.rows * 128) = lo;
      }
    }
    if (l16 == 0) {
      float off = 0.0f;
      if (f < nf) { const int t = f / s.G; off = odd ? NAN : kWeightShift - p.lse[stat_offset<false>(s, r, hk * s.G + f - t * s.G, t)] * kLog2e; }
      p.off[plane * p.q.rows + f] = off;
      p.delta[plane * p.q.rows + f] = delta * sc[1] * sv;
    }
  }
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0 && top > 0.0f) atomicMax(whole ? &norm : p.norms + plane * 2 + 1, __float_as_uint(top));
  if (whole) {
    __syncthreads();
    if (threadIdx.x == 0) p.norms[plane * 2 + 1] = norm;
  }
}

// Factors of a plane: scores to log2 units, dO.V - delta (scaled) into f16's range with the weights' 2^15 taken out, and the
// results back.
struct PlaneFactors { float score, grad, dq, dk, dv; };
__device__ __forceinline__ PlaneFactors plane_factors(const BackwardTc& p, int64_t plane) {
  float sq, iq, sg, ig, sk, ik, sv, iv;
  plane_scale(p.qamax[plane * 2], sq, iq);
  plane_scale(p.qamax[plane * 2 + 1], sg, ig);
  plane_scale(p.pk.amax[plane * 2], sk, ik);
  plane_scale(p.pk.amax[plane * 2 + 1], sv, iv);
  // |dO.V| and |delta| of scaled rows are at most their norms' product, below 2^37; dS then stays below 2^15: reach < 2^e, twice that times 2^(14 - e)
  const float reach = sqrtf(__uint_as_float(p.norms[plane * 2])) * sqrtf(__uint_as_float(p.norms[plane * 2 + 1]));
  const int e = reach > 0.0f ? (int)(__float_as_uint(reach) >> 23) - 127 + 1 : 0;   // reach < 2^e
  PlaneFactors f;
  f.score = p.s.scale * kLog2e * iq * ik;
  f.grad = exp2f((float)(14 - e) - kWeightShift);
  const float back = exp2f((float)(e - 14)) * ig * iv * p.s.scale;
  f.dq = back * ik; f.dk = back * iq; f.dv = exp2f(-kWeightShift) * ig;
  return f;
}

constexpr int kThreadsB = 384;        // two warpgroups of softmax threads, one for the issuing and the copying warp
constexpr int kRegsSoftmax = 224, kRegsOther = 56;
constexpr int kFlush = 2;             // steps whose sums are left to the tensor core before they are rounded into registers
// Adds 32 * N columns of an accumulator to registers.
template <int N>
__device__ __forceinline__ void add_columns(uint32_t taddr, float* acc) {
#pragma unroll
  for (int h = 0; h < N; ++h) {
    uint32_t y[32];
    tmem_ld32(taddr + h * 32, y);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 32; ++e) acc[h * 32 + e] += __uint_as_float(y[e]);
  }
}
// 32 values of a row to f16 pairs in tensor memory: 16 columns of hi, 16 of lo.
__device__ __forceinline__ void store_pairs(uint32_t taddr, const float (&x)[32]) {
  uint32_t y[32];
#pragma unroll
  for (int e = 0; e < 32; e += 2) split_f16(x[e], x[e + 1], y[e >> 1], y[16 + (e >> 1)]);
  tmem_st32(taddr, y);
  tmem_st_wait();
}
// Row `row` of a packed plane's hi half (channels 64 * block ..), unswizzled, to 32 columns of tensor memory.
__device__ __forceinline__ void row_to_tmem(uint32_t taddr, const uint8_t* src, int row, bool live) {
  uint32_t y[32];
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (live) v = *reinterpret_cast<const uint4*>(src + (int64_t)row * 128 + ((c ^ (row & 7)) << 4));
    y[4 * c] = v.x; y[4 * c + 1] = v.y; y[4 * c + 2] = v.z; y[4 * c + 3] = v.w;
  }
  tmem_st32(taddr, y);
}

// dK and dV.  One CTA per (128 keys or a part of their query rows, kv head, sequence): S^T = K Q^T and dP^T = V dO^T of 64 query rows a
// step, a softmax thread per (key, 32 query rows) turns them into P^T and dS^T in place, and dV += P^T dO, dK += dS^T Q take them
// from tensor memory.  The hi half of K lives in tensor memory too, which leaves room for two stages of Q and dO.
// Tensor memory: S^T 2 x 64 columns, dP^T 64, K hi 64, dV 128, dK 128.  Shared memory: V 64 KB, K lo 32 KB, 2 x (Q 32 KB + dO 32 KB).
// Every kFlush steps dV and dK are added to float32 registers (64 + 64 a thread).  Bound: tensor pipe.
template <int DP>
__global__ void __launch_bounds__(kThreadsB, 1) stream_tc_dkv_kernel(const __grid_constant__ BackwardTc p) {
  constexpr int CB = DP / 64, HC = DP / 2;
  constexpr uint32_t SLOT = CB * 16384u, OFF_KL = CB * 32768u, OFF_Q = OFF_KL + CB * 16384u, OFF_G = OFF_Q + 2 * SLOT, STATS = OFF_G + 2 * SLOT, BARS = STATS + 1024;
  constexpr uint32_t COL_S = 0, COL_DP = 128, COL_KH = 192, COL_DV = 256, COL_DK = 384;
  extern __shared__ uint8_t smem_raw[];
  const StreamRows& s = p.s;
  const int hk = blockIdx.y, r = blockIdx.z, x0 = blockIdx.x;
  const bool sink = x0 < p.sink_tiles * p.parts_sink;
  const int parts = sink ? p.parts_sink : p.parts, y0 = sink ? x0 : x0 - p.sink_tiles * p.parts_sink;
  const int kt = (sink ? 0 : p.sink_tiles) + y0 / parts, part = y0 % parts, k0 = kt * 128;
  const int len = row_span<false>(s, r).ctx;
  if (k0 >= len && parts > 1) return;   // the summing kernel does not look at padding
  const int nf = len * s.G;
  const int64_t t_end = (s.window < 0 || k0 < s.sinks) ? len : min((int64_t)len, (int64_t)k0 + 128 + s.window);
  const int f_begin = (k0 * s.G) & ~7, f_end = (int)t_end * s.G;
  const int steps = k0 < len ? (f_end - f_begin + 63) / 64 : 0, per = (steps + parts - 1) / parts;
  const int i0 = part * per, n = max(0, min(steps, i0 + per) - i0);
  const int64_t plane = (int64_t)r * s.Hkv + hk;

  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + BARS;
  const uint32_t v_full = bars, kh_ready = bars + 8, dp_full = bars + 16, ds_full = bars + 24, acc_full = bars + 32, acc_empty = bars + 40, tmem_slot = bars + 128;
  auto q_full = [&](int i) { return bars + 48u + 8u * i; };
  auto g_full = [&](int i) { return bars + 64u + 8u * i; };
  auto q_empty = [&](int i) { return bars + 80u + 8u * i; };
  auto g_empty = [&](int i) { return bars + 96u + 8u * i; };
  auto s_full = [&](int i) { return bars + 112u + 8u * i; };
  auto p_full = [&](int i) { return bars + 136u + 8u * i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(v_full, 1); mbar_init(kh_ready, 256); mbar_init(dp_full, 1); mbar_init(ds_full, 256); mbar_init(acc_full, 1); mbar_init(acc_empty, 256);
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full(i), 1); mbar_init(g_full(i), 1); mbar_init(q_empty(i), 1); mbar_init(g_empty(i), 1); mbar_init(s_full(i), 1); mbar_init(p_full(i), 256);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gen + BARS + 128);
  auto row0 = [&](int i) { return f_begin + (i0 + i) * 64; };
  auto rows16 = [&](int i) { return min(64, (f_end - row0(i) + 15) & ~15); };

  if (warp >= 8) {
    regs_dec<kRegsOther>();
    if (warp == 9 && lane == 0 && n > 0) {
      // ----------------------------------------------------------- copies
      const int keys = min(128, (len - k0 + 15) & ~15);
      mbar_expect_tx(v_full, (uint32_t)CB * 3u * keys * 128u);
      const uint8_t* vp = p.pk.v.data + plane * p.pk.v.plane_bytes(CB); const uint8_t* kp = p.pk.k.data + plane * p.pk.k.plane_bytes(CB);
      for (int b = 0; b < CB * 2; ++b) bulk_load(base + b * 16384, vp + ((int64_t)b * p.pk.v.rows + k0) * 128, keys * 128, v_full);
      for (int b = 0; b < CB; ++b) bulk_load(base + OFF_KL + b * 16384, kp + ((int64_t)(2 * b + 1) * p.pk.k.rows + k0) * 128, keys * 128, v_full);
      const uint8_t* qp = p.q.data + plane * p.q.plane_bytes(CB); const uint8_t* gp = p.g.data + plane * p.g.plane_bytes(CB);
      bool ok = true;
      int jq = 0, jg = 0;
      for (uint32_t idle = 0; jg < n && ok;) {
        bool did = false;
        if (jq < n && (jq < 2 || mbar_test(q_empty(jq & 1), ((jq >> 1) - 1) & 1))) {
          const int rows = rows16(jq);
          const uint32_t bar = q_full(jq & 1), dst = base + OFF_Q + (jq & 1) * SLOT, st = base + STATS + (jq & 1) * 512;
          mbar_expect_tx(bar, (uint32_t)CB * 2u * rows * 128u + 2u * rows * 4u);
          for (int b = 0; b < CB * 2; ++b) bulk_load(dst + b * 8192, qp + ((int64_t)b * p.q.rows + row0(jq)) * 128, rows * 128, bar);
          bulk_load(st, p.off + plane * p.q.rows + row0(jq), rows * 4, bar);
          bulk_load(st + 256, p.delta + plane * p.q.rows + row0(jq), rows * 4, bar);
          ++jq; did = true;
        }
        if (jg < jq && (jg < 2 || mbar_test(g_empty(jg & 1), ((jg >> 1) - 1) & 1))) {
          const int rows = rows16(jg);
          const uint32_t bar = g_full(jg & 1), dst = base + OFF_G + (jg & 1) * SLOT;
          mbar_expect_tx(bar, (uint32_t)CB * 2u * rows * 128u);
          for (int b = 0; b < CB * 2; ++b) bulk_load(dst + b * 8192, gp + ((int64_t)b * p.g.rows + row0(jg)) * 128, rows * 128, bar);
          ++jg; did = true;
        }
        if (did) idle = 0;
        else if (++idle > kSpinLimit) ok = false;
        else if (idle > 4096) __nanosleep(64);
      }
      if (!ok)   // copies in flight land before the CTA goes
        for (int i = 0; i < 2; ++i)
          for (int ph = 0; ph < 2; ++ph) { mbar_wait(q_full(i), ph); mbar_wait(g_full(i), ph); }
      mbar_wait(v_full, 0);
    }
    if (warp == 8 && n > 0) {
      const uint32_t el = elect_lane();
      // ----------------------------------------------------------- instructions: whichever product has its operands
      int is = 0, ip = 0, iv = 0, ik = 0, chunk = 0;   // next S, dP, dV, dK; the accumulation chunk that may be written
      bool ok = mbar_wait(v_full, 0) && mbar_wait(kh_ready, 0);
      tc_fence_after();
      const uint32_t kl = base + OFF_KL;
      auto in_chunk = [&](int i) {
        if (i / kFlush > chunk && mbar_test(acc_empty, chunk & 1)) ++chunk;
        return i / kFlush <= chunk;
      };
      // rows of a query tile as the MN-major operand of dV, dK
      auto accumulate = [&](uint32_t d, uint32_t a, uint32_t slot, int i) {
        const uint32_t id = instr_desc_f16(128, DP, 1);
        const int slices = rows16(i) >> 4;
        const uint32_t fresh = i % kFlush == 0 ? 0u : 1u;
        auto one = [&](int ks, int al, int bl, uint32_t acc) {
          umma_f16_ts(el, d, a + (ks >> 1) * 32 + al * 16 + (ks & 1) * 8, smem_desc_mn(slot + bl * 8192 + ks * 2048, 16384), id, acc);
        };
        for (int ks = 0; ks < slices; ++ks) { one(ks, 1, 0, ks > 0 ? 1u : fresh); one(ks, 0, 1, 1); }
        for (int ks = 0; ks < slices; ++ks) one(ks, 0, 0, 1);
      };
      auto end_chunk = [&]() { if (iv == ik && (iv % kFlush == 0 || iv == n)) commit_by(el, acc_full); };
      for (uint32_t idle = 0; (ik < n || iv < n) && ok;) {
        bool did = false;
        if (ik < ip && in_chunk(ik) && mbar_test(ds_full, ik & 1)) {
          tc_fence_after();
          accumulate(tmem + COL_DK, tmem + COL_DP, base + OFF_Q + (ik & 1) * SLOT, ik);
          commit_by(el, q_empty(ik & 1));
          ++ik; did = true;
          end_chunk();
        }
        if (ip < n && ip <= ik && mbar_test(g_full(ip & 1), (ip >> 1) & 1)) {
          tc_fence_after();
          const uint32_t id = instr_desc_f16(128, rows16(ip), 0), g = base + OFF_G + (ip & 1) * SLOT;
          auto one = [&](int ks, int vl, int gl, uint32_t acc) {
            umma_f16(el, tmem + COL_DP, smem_desc_sw128(base + (ks >> 2) * 32768 + vl * 16384) + 2u * (ks & 3),
                     smem_desc_sw128(g + (ks >> 2) * 16384 + gl * 8192) + 2u * (ks & 3), id, acc);
          };
#pragma unroll
          for (int ks = 0; ks < CB * 4; ++ks) { one(ks, 1, 0, ks > 0); one(ks, 0, 1, 1); }
#pragma unroll
          for (int ks = 0; ks < CB * 4; ++ks) one(ks, 0, 0, 1);
          commit_by(el, dp_full);
          ++ip; did = true;
        }
        if (iv < is && iv < ip && in_chunk(iv) && mbar_test(p_full(iv & 1), (iv >> 1) & 1)) {
          tc_fence_after();
          accumulate(tmem + COL_DV, tmem + COL_S + (iv & 1) * 64, base + OFF_G + (iv & 1) * SLOT, iv);
          commit_by(el, g_empty(iv & 1));
          ++iv; did = true;
          end_chunk();
        }
        if (is < n && is < iv + 2 && mbar_test(q_full(is & 1), (is >> 1) & 1)) {
          tc_fence_after();
          const uint32_t d = tmem + COL_S + (is & 1) * 64, id = instr_desc_f16(128, rows16(is), 0), q = base + OFF_Q + (is & 1) * SLOT;
          auto b_of = [&](int ks, int ql) { return smem_desc_sw128(q + (ks >> 2) * 16384 + ql * 8192) + 2u * (ks & 3); };
#pragma unroll
          for (int ks = 0; ks < CB * 4; ++ks) {
            umma_f16(el, d, smem_desc_sw128(kl + (ks >> 2) * 16384) + 2u * (ks & 3), b_of(ks, 0), id, ks > 0);
            umma_f16_ts(el, d, tmem + COL_KH + ks * 8, b_of(ks, 1), id, 1);
          }
#pragma unroll
          for (int ks = 0; ks < CB * 4; ++ks) umma_f16_ts(el, d, tmem + COL_KH + ks * 8, b_of(ks, 0), id, 1);
          commit_by(el, s_full(is & 1));
          ++is; did = true;
        }
        if (did) idle = 0;
        else if (++idle > kSpinLimit) ok = false;
        else if (idle > 4096) __nanosleep(64);
      }
    }
  } else {
    regs_inc<kRegsSoftmax>();
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane, key = k0 + row;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    const PlaneFactors fc = plane_factors(p, plane);
    if (n > 0) {
      if (half < CB) row_to_tmem(lane_addr + COL_KH + half * 32, p.pk.k.data + plane * p.pk.k.plane_bytes(CB) + (int64_t)half * 2 * p.pk.k.rows * 128, key, key < len);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(kh_ready);
    }
    // the query rows that see the key
    const int f_lo = key < len ? key * s.G : 0;
    const int f_hi = key >= len ? 0 : (s.window < 0 || key < s.sinks) ? nf : (int)min((int64_t)nf, ((int64_t)key + s.window + 1) * s.G);
    float dv[HC], dk[HC];
#pragma unroll
    for (int e = 0; e < HC; ++e) dv[e] = dk[e] = 0.0f;
    bool ok = true;
    // a chunk's sums are fetched one step later, between that step's weights and its dS: the products that end the chunk run meanwhile
    auto flush = [&](int chunk) {
      ok = ok && mbar_wait(acc_full, chunk & 1);
      tc_fence_after();
      add_columns<HC / 32>(lane_addr + COL_DV + half * HC, dv);
      add_columns<HC / 32>(lane_addr + COL_DK + half * HC, dk);
      tc_fence_before();
      mbar_arrive(acc_empty);
    };
    for (int i = 0; i < n; ++i) {
      const int f0 = row0(i) + half * 32;
      const uint32_t see = (uint32_t)(bits_below(f_hi - f0) & ~bits_below(f_lo - f0));
      const float* off = reinterpret_cast<const float*>(gen + STATS + (i & 1) * 512) + half * 32;
      float w[32];
      ok = ok && mbar_wait(q_full(i & 1), (i >> 1) & 1) && mbar_wait(s_full(i & 1), (i >> 1) & 1);
      tc_fence_after();
      {
        uint32_t y[32];
        tmem_ld32(lane_addr + COL_S + (i & 1) * 64 + half * 32, y);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) w[e] = ((see >> e) & 1u) ? exp2_fast(fmaf(__uint_as_float(y[e]), fc.score, off[e])) : 0.0f;
      }
      store_pairs(lane_addr + COL_S + (i & 1) * 64 + half * 32, w);
      tc_fence_before();
      mbar_arrive(p_full(i & 1));
      if (i > 0 && i % kFlush == 0) flush(i / kFlush - 1);
      ok = ok && mbar_wait(dp_full, i & 1);
      tc_fence_after();
      {
        uint32_t y[32];
        tmem_ld32(lane_addr + COL_DP + half * 32, y);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) w[e] = ((see >> e) & 1u) ? w[e] * ((__uint_as_float(y[e]) - off[64 + e]) * fc.grad) : 0.0f;
      }
      store_pairs(lane_addr + COL_DP + half * 32, w);
      tc_fence_before();
      mbar_arrive(ds_full);
    }
    if (n > 0) flush((n - 1) / kFlush);
    const float zk = ok ? fc.dk : NAN, zv = ok ? fc.dv : NAN;
    if (parts > 1) {
      float* at = p.part + (((plane * p.units + x0) * 2) * 128 + row) * DP + half * HC;
#pragma unroll
      for (int e = 0; e < HC; e += 4) {
        *reinterpret_cast<float4*>(at + e) = make_float4(dv[e] * zv, dv[e + 1] * zv, dv[e + 2] * zv, dv[e + 3] * zv);
        *reinterpret_cast<float4*>(at + 128 * DP + e) = make_float4(dk[e] * zk, dk[e + 1] * zk, dk[e + 2] * zk, dk[e + 3] * zk);
      }
    } else if (key < s.seq) {
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const gn_view& view = which ? p.dk : p.dv;
        const float* acc = which ? dk : dv;
        const float z = which ? zk : zv;
        float* dst = view.data + token_offset<false>(view, r, hk, key);
#pragma unroll
        for (int e = 0; e < HC; e += 4) {
          const int ch = half * HC + e;
          if (p.vec_dkv) {
            if (ch < s.D) {
              float4 v = make_float4(acc[e] * z, acc[e + 1] * z, acc[e + 2] * z, acc[e + 3] * z);
              if (p.accumulate) { const float4 o = *reinterpret_cast<const float4*>(dst + ch); v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w; }
              *reinterpret_cast<float4*>(dst + ch) = v;
            }
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) if (ch + u < s.D) dst[ch + u] = __fadd_rn(p.accumulate ? dst[ch + u] : 0.0f, acc[e + u] * z);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

// Sums the parts of key tiles that were divided, in their order: a warp per key row and tensor.
template <int DP>
__global__ void __launch_bounds__(256) stream_tc_dkv_sum_kernel(const __grid_constant__ BackwardTc p) {
  const StreamRows& s = p.s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hk = blockIdx.y, r = blockIdx.z >> 1, which = blockIdx.z & 1, key = blockIdx.x * 8 + warp;
  if (key >= s.seq) return;
  const int kt = key / 128;
  const bool sink = kt < p.sink_tiles;
  const int parts = sink ? p.parts_sink : p.parts, unit = sink ? kt * parts : p.sink_tiles * p.parts_sink + (kt - p.sink_tiles) * parts;
  if (parts == 1) return;
  const int64_t plane = (int64_t)r * s.Hkv + hk;
  float x[DP / 32];
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) x[e] = 0.0f;
  if (key < row_span<false>(s, r).ctx)
    for (int i = 0; i < parts; ++i) {
      const float* at = p.part + (((plane * p.units + unit + i) * 2 + which) * 128 + key % 128) * DP;
#pragma unroll
      for (int e = 0; e < DP / 32; ++e) x[e] += at[lane + 32 * e];
    }
  const gn_view& view = which ? p.dk : p.dv;
  float* dst = view.data + token_offset<false>(view, r, hk, key);
#pragma unroll
  for (int e = 0; e < DP / 32; ++e)
    if (lane + 32 * e < s.D) dst[lane + 32 * e] = p.accumulate ? dst[lane + 32 * e] + x[e] : x[e];
}

// dQ.  One CTA per (128 query rows, kv head, sequence): S = Q K^T and dP = dO V^T of 64 keys a step, dS in place of dP, dQ += dS K with
// dS from tensor memory and the same K tile read the other way.
// Tensor memory: Q hi 64 columns, dO hi 64, S 2 x 64, dP 2 x 64, dQ 128.  Shared memory: Q lo, dO lo 32 KB each, 3 K and 2 V tiles of 32 KB.
template <int DP>
__global__ void __launch_bounds__(kThreadsB, 1) stream_tc_dq_kernel(const __grid_constant__ BackwardTc p) {
  constexpr int CB = DP / 64, HC = DP / 2;
  constexpr uint32_t SLOT = CB * 16384u, OFF_GL = CB * 16384u, OFF_K = 2 * CB * 16384u, OFF_V = OFF_K + 3 * SLOT, BARS = OFF_V + 2 * SLOT;
  constexpr uint32_t COL_Q = 0, COL_G = 64, COL_S = 128, COL_DP = 256, COL_DQ = 384;
  extern __shared__ uint8_t smem_raw[];
  const StreamRows& s = p.s;
  const int hk = blockIdx.y, r = blockIdx.z, tile = p.q_tiles - 1 - (int)blockIdx.x, f0 = tile * 128;
  const int len = row_span<false>(s, r).ctx, nf = len * s.G;
  KeyRuns runs{0, 0, 0};
  if (f0 < nf) runs = key_runs(s, f0 / s.G, min(f0 + 127, nf - 1) / s.G);
  const int n = (runs.total + 63) / 64;
  const int64_t plane = (int64_t)r * s.Hkv + hk;

  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + BARS;
  const uint32_t lo_full = bars, hi_ready = bars + 8, acc_full = bars + 16, acc_empty = bars + 24, tmem_slot = bars + 136;
  auto k_full = [&](int i) { return bars + 32u + 8u * i; };
  auto k_empty = [&](int i) { return bars + 56u + 8u * i; };
  auto v_full = [&](int i) { return bars + 80u + 8u * i; };
  auto v_empty = [&](int i) { return bars + 96u + 8u * i; };
  auto sp_full = [&](int i) { return bars + 112u + 8u * i; };
  auto ds_full = [&](int i) { return bars + 144u + 8u * i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(lo_full, 1); mbar_init(hi_ready, 256); mbar_init(acc_full, 1); mbar_init(acc_empty, 256);
    for (int i = 0; i < 3; ++i) { mbar_init(k_full(i), 1); mbar_init(k_empty(i), 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(v_full(i), 1); mbar_init(v_empty(i), 1); mbar_init(sp_full(i), 1); mbar_init(ds_full(i), 256); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gen + BARS + 136);
  auto rows16 = [&](int j) { return min(64, (runs.total - j * 64 + 15) & ~15); };

  if (warp >= 8) {
    regs_dec<kRegsOther>();
    if (warp == 9 && lane == 0 && n > 0) {
      const int rows = min(128, (nf - f0 + 15) & ~15);
      mbar_expect_tx(lo_full, (uint32_t)CB * 2u * rows * 128u);
      for (int w = 0; w < 2; ++w) {
        const Packed& src = w ? p.g : p.q;
        for (int b = 0; b < CB; ++b)
          bulk_load(base + w * OFF_GL + b * 16384, src.data + plane * src.plane_bytes(CB) + ((int64_t)(2 * b + 1) * src.rows + f0) * 128, rows * 128, lo_full);
      }
      auto copy_tile = [&](const Packed& src, uint32_t dst, uint32_t bar, int j) {
        const int c0 = j * 64, m = rows16(j), na = min(max(runs.a_len - c0, 0), m), nb = m - na;
        const uint8_t* from = src.data + plane * src.plane_bytes(CB);
        mbar_expect_tx(bar, (uint32_t)CB * 2u * m * 128u);
        for (int b = 0; b < CB * 2; ++b) {
          if (na) bulk_load(dst + b * 8192, from + ((int64_t)b * src.rows + c0) * 128, na * 128, bar);
          if (nb) bulk_load(dst + b * 8192 + na * 128, from + ((int64_t)b * src.rows + c0 + na + runs.shift) * 128, nb * 128, bar);
        }
      };
      bool ok = true;
      int jk = 0, jv = 0;
      for (uint32_t idle = 0; (jv < n || jk < n) && ok;) {
        bool did = false;
        if (jk < n && (jk < 3 || mbar_test(k_empty(jk % 3), (jk / 3 - 1) & 1))) { copy_tile(p.pk.k, base + OFF_K + (jk % 3) * SLOT, k_full(jk % 3), jk); ++jk; did = true; }
        if (jv < jk && (jv < 2 || mbar_test(v_empty(jv & 1), ((jv >> 1) - 1) & 1))) { copy_tile(p.pk.v, base + OFF_V + (jv & 1) * SLOT, v_full(jv & 1), jv); ++jv; did = true; }
        if (did) idle = 0;
        else if (++idle > kSpinLimit) ok = false;
        else if (idle > 4096) __nanosleep(64);
      }
      if (!ok)
        for (int ph = 0; ph < 2; ++ph) {
          for (int i = 0; i < 3; ++i) mbar_wait(k_full(i), ph);
          for (int i = 0; i < 2; ++i) mbar_wait(v_full(i), ph);
        }
      mbar_wait(lo_full, 0);
    }
    if (warp == 8 && n > 0) {
      const uint32_t el = elect_lane();
      bool ok = mbar_wait(lo_full, 0) && mbar_wait(hi_ready, 0);
      tc_fence_after();
      auto scores = [&](int j) {
        const uint32_t id = instr_desc_f16(128, rows16(j), 0);
        for (int w = 0; w < 2 && ok; ++w) {
          ok = ok && (w ? mbar_wait(v_full(j & 1), (j >> 1) & 1) : mbar_wait(k_full(j % 3), (j / 3) & 1));
          if (!ok) break;
          tc_fence_after();
          const uint32_t d = tmem + (w ? COL_DP : COL_S) + (j & 1) * 64, hi = tmem + (w ? COL_G : COL_Q), lo = base + w * OFF_GL;
          const uint32_t slot = w ? base + OFF_V + (j & 1) * SLOT : base + OFF_K + (j % 3) * SLOT;
          auto b_of = [&](int ks, int l) { return smem_desc_sw128(slot + (ks >> 2) * 16384 + l * 8192) + 2u * (ks & 3); };
#pragma unroll
          for (int ks = 0; ks < CB * 4; ++ks) {
            umma_f16(el, d, smem_desc_sw128(lo + (ks >> 2) * 16384) + 2u * (ks & 3), b_of(ks, 0), id, ks > 0);
            umma_f16_ts(el, d, hi + ks * 8, b_of(ks, 1), id, 1);
          }
#pragma unroll
          for (int ks = 0; ks < CB * 4; ++ks) umma_f16_ts(el, d, hi + ks * 8, b_of(ks, 0), id, 1);
        }
        if (!ok) return;
        commit_by(el, v_empty(j & 1));
        commit_by(el, sp_full(j & 1));
      };
      if (ok) scores(0);
      for (int j = 0; j < n && ok; ++j) {
        if (j + 1 < n) scores(j + 1);
        ok = ok && mbar_wait(ds_full(j & 1), (j >> 1) & 1) && (j < kFlush || j % kFlush || mbar_wait(acc_empty, (j / kFlush - 1) & 1));
        if (!ok) break;
        tc_fence_after();
        const uint32_t id = instr_desc_f16(128, DP, 1), a = tmem + COL_DP + (j & 1) * 64, slot = base + OFF_K + (j % 3) * SLOT;
        const int slices = rows16(j) >> 4;
        const uint32_t fresh = j % kFlush == 0 ? 0u : 1u;
        auto one = [&](int ks, int al, int bl, uint32_t acc) {
          umma_f16_ts(el, tmem + COL_DQ, a + (ks >> 1) * 32 + al * 16 + (ks & 1) * 8, smem_desc_mn(slot + bl * 8192 + ks * 2048, 16384), id, acc);
        };
        for (int ks = 0; ks < slices; ++ks) { one(ks, 1, 0, ks > 0 ? 1u : fresh); one(ks, 0, 1, 1); }
        for (int ks = 0; ks < slices; ++ks) one(ks, 0, 0, 1);
        commit_by(el, k_empty(j % 3));
        if ((j + 1) % kFlush == 0 || j + 1 == n) commit_by(el, acc_full);
      }
    }
  } else {
    regs_inc<kRegsSoftmax>();
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane, f = f0 + row;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    const bool live = f < nf;
    const int t = f / s.G, h = hk * s.G + f - t * s.G;
    const PlaneFactors fc = plane_factors(p, plane);
    float off = 0.0f, delta = 0.0f;
    if (n > 0) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const Packed& src = w ? p.g : p.q;
        if (half < CB) row_to_tmem(lane_addr + (w ? COL_G : COL_Q) + half * 32, src.data + plane * src.plane_bytes(CB) + (int64_t)half * 2 * src.rows * 128, f, live);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(hi_ready);
      if (live) { off = p.off[plane * p.q.rows + f]; delta = p.delta[plane * p.q.rows + f]; }
    }
    const int s_end = live ? min(s.sinks, t + 1) : 0;
    const int lo_key = live ? (s.window < 0 ? 0 : max(0, t - s.window)) - runs.shift : 0, hi_key = live ? t - runs.shift : -1;
    float acc[HC];
#pragma unroll
    for (int e = 0; e < HC; ++e) acc[e] = 0.0f;
    bool ok = true;
    auto flush = [&](int chunk) {   // one step later, as above
      ok = ok && mbar_wait(acc_full, chunk & 1);
      tc_fence_after();
      add_columns<HC / 32>(lane_addr + COL_DQ + half * HC, acc);
      tc_fence_before();
      mbar_arrive(acc_empty);
    };
    for (int j = 0; j < n; ++j) {
      const int c0 = j * 64 + half * 32;
      const uint32_t see = (uint32_t)(bits_below(s_end - c0) | (bits_below(hi_key + 1 - c0) & ~bits_below(lo_key - c0)));
      ok = ok && mbar_wait(sp_full(j & 1), (j >> 1) & 1);
      tc_fence_after();
      float w[32];
      {
        uint32_t y[32];
        tmem_ld32(lane_addr + COL_S + (j & 1) * 64 + half * 32, y);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) w[e] = exp2_fast(fmaf(__uint_as_float(y[e]), fc.score, off));
        tmem_ld32(lane_addr + COL_DP + (j & 1) * 64 + half * 32, y);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) w[e] = ((see >> e) & 1u) ? w[e] * ((__uint_as_float(y[e]) - delta) * fc.grad) : 0.0f;
      }
      store_pairs(lane_addr + COL_DP + (j & 1) * 64 + half * 32, w);
      tc_fence_before();
      mbar_arrive(ds_full(j & 1));
      if (j > 0 && j % kFlush == 0) flush(j / kFlush - 1);
    }
    if (n > 0) flush((n - 1) / kFlush);
    if (f < s.seq * s.G) {
      const float z = ok ? fc.dq : NAN;
      float* dst = p.dq.data + token_offset<false>(p.dq, r, h, t);
#pragma unroll
      for (int e = 0; e < HC; e += 4) {
        const int ch = half * HC + e;
        if (p.vec_dq) {
          if (ch < s.D) {
            float4 v = make_float4(acc[e] * z, acc[e + 1] * z, acc[e + 2] * z, acc[e + 3] * z);
            if (p.accumulate) { const float4 o = *reinterpret_cast<const float4*>(dst + ch); v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w; }
            *reinterpret_cast<float4*>(dst + ch) = v;
          }
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u) if (ch + u < s.D) dst[ch + u] = __fadd_rn(p.accumulate ? dst[ch + u] : 0.0f, acc[e + u] * z);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------ host
int64_t carve_backward(const StreamRows& s, void* workspace, BackwardTc* b) {
  const int DP = s.D <= 64 ? 64 : 128, CB = DP / 64;
  const int64_t planes = (int64_t)s.rows * s.Hkv;
  b->q_tiles = ceil_div((int64_t)s.seq * s.G, 128);
  b->key_tiles = ceil_div(s.seq, 128);
  // Key tiles whose steps (64 query rows each) would make a long tail are divided.  A tile of sinks is seen by every later
  // query and gets as many parts as make them about as long as the others'; and when there are fewer than four waves
  // of CTAs all tiles are divided, while a part keeps 16 steps (writing and summing a part costs about one step).
  const bool windowed = s.window >= 0 && s.sinks > 0 && (int64_t)s.window + 128 < s.seq;
  b->sink_tiles = windowed ? std::min(b->key_tiles, ceil_div(s.sinks, 128)) : 0;
  const int64_t reach = s.window >= 0 ? std::min<int64_t>(s.seq, (int64_t)s.window + 128) : s.seq;
  const int64_t steps = ceil_div(reach * s.G, 64), steps_sink = ceil_div((int64_t)s.seq * s.G, 64);
  const int64_t ctas = planes * b->key_tiles;
  b->parts = (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(4 * 148, ctas), steps / 16));
  b->parts_sink = b->sink_tiles ? (int)std::max<int64_t>(1, ceil_div(steps_sink * b->parts, steps)) : 1;
  b->units = b->sink_tiles * b->parts_sink + (b->key_tiles - b->sink_tiles) * b->parts;
  Carve c{static_cast<uint8_t*>(workspace)};
  PackedKeys& pk = b->pk;
  pk.amax = c.take<uint32_t>(planes * 4);
  pk.odd = reinterpret_cast<int*>(pk.amax + planes * 2);
  b->qamax = c.take<uint32_t>(planes * 2);
  b->norms = c.take<uint32_t>(planes * 2);
  pk.k.rows = pk.v.rows = packed_rows(s.seq);
  b->q.rows = b->g.rows = packed_rows((int64_t)s.seq * s.G);
  pk.k.data = c.take<uint8_t>(planes * pk.k.plane_bytes(CB));
  pk.v.data = c.take<uint8_t>(planes * pk.v.plane_bytes(CB));
  pk.flags_k = c.take<uint8_t>(planes * pk.k.rows);
  pk.flags_v = c.take<uint8_t>(planes * pk.v.rows);
  b->q.data = c.take<uint8_t>(planes * b->q.plane_bytes(CB));
  b->g.data = c.take<uint8_t>(planes * b->g.plane_bytes(CB));
  b->off = c.take<float>(planes * b->q.rows);
  b->delta = c.take<float>(planes * b->q.rows);
  if (b->parts > 1 || b->parts_sink > 1) b->part = c.take<float>(planes * b->units * 2 * 128 * DP);
  return c.used;
}

template <int DP>
int backward_go(const StreamRows& s, BackwardTc& b, cudaStream_t st) {
  constexpr int CB = DP / 64;
  constexpr int kSmemKv = CB * (32768 + 16384 + 4 * 16384) + 1024 + 256 + 1024, kSmemQ = CB * (2 * 16384 + 5 * 16384) + 256 + 1024;
  static PerDeviceOnce once;
  if (once.first()) {
    GN_TRY(check_registers(reinterpret_cast<const void*>(stream_tc_dkv_kernel<DP>), kThreadsB, 256 * kRegsSoftmax + 128 * kRegsOther));
    GN_TRY(check_registers(reinterpret_cast<const void*>(stream_tc_dq_kernel<DP>), kThreadsB, 256 * kRegsSoftmax + 128 * kRegsOther));
    GN_CUDA(cudaFuncSetAttribute(stream_tc_dkv_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemKv));
    GN_CUDA(cudaFuncSetAttribute(stream_tc_dq_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemQ));
  }
  const int64_t planes = (int64_t)s.rows * s.Hkv;
  GN_TRY(stream_pack_keys(s, b.pk, b.norms, st));
  const int whole = b.q.rows <= kWholePlaneQ;
  if (!whole) {
    const dim3 rows(ceil_div(b.q.rows, kPackRowsQ), s.Hkv, s.rows);
    GN_CUDA(cudaMemsetAsync(b.qamax, 0, planes * 2 * sizeof(uint32_t), st));
    GN_CUDA(cudaMemset2DAsync(b.norms + 1, 2 * sizeof(uint32_t), 0, sizeof(uint32_t), planes, st));
    stream_query_amax_kernel<CB><<<rows, 256, 0, st>>>(b);
    GN_LAUNCH_CHECK();
  }
  stream_query_pack_kernel<CB><<<dim3(whole ? 1 : ceil_div(b.q.rows, kPackRowsQ), s.Hkv, s.rows), 256, 0, st>>>(b, whole);
  GN_LAUNCH_CHECK();
  stream_tc_dkv_kernel<DP><<<dim3(b.units, s.Hkv, s.rows), kThreadsB, kSmemKv, st>>>(b);
  GN_LAUNCH_CHECK();
  if (b.parts > 1 || b.parts_sink > 1) {
    stream_tc_dkv_sum_kernel<DP><<<dim3(ceil_div(s.seq, 8), s.Hkv, 2 * s.rows), 256, 0, st>>>(b);
    GN_LAUNCH_CHECK();
  }
  stream_tc_dq_kernel<DP><<<dim3(b.q_tiles, s.Hkv, s.rows), kThreadsB, kSmemQ, st>>>(b);
  GN_LAUNCH_CHECK();
  return GN_OK;
}

}  // namespace

int64_t stream_tc_backward_bytes(const StreamRows& s) {
  BackwardTc b{};
  return carve_backward(s, nullptr, &b);
}
int stream_tc_backward(const StreamRows& s, const gn_view& out, const gn_view& dout, const float* lse, const gn_view& dq, const gn_view& dk, const gn_view& dv,
                       int accumulate, void* workspace, cudaStream_t st) {
  BackwardTc b{};
  b.s = s; b.out = out; b.dout = dout; b.lse = lse; b.dq = dq; b.dk = dk; b.dv = dv; b.accumulate = accumulate;
  carve_backward(s, workspace, &b);
  b.vec_in = vec_view(s.q, s.D) && vec_view(dout, s.D) && vec_view(out, s.D);
  b.vec_dq = vec_view(dq, s.D);
  b.vec_dkv = vec_view(dk, s.D) && vec_view(dv, s.D);
  return s.D <= 64 ? backward_go<64>(s, b, st) : backward_go<128>(s, b, st);
}

}  // namespace gn
