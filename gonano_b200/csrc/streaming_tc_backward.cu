// Streaming attention backward on the 5th-generation tensor cores, padded batches.
//
// With P = exp(s - lse), dS = P (dO.V - delta), delta = dO.O:  dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K.  Two kernels,
// one that keeps 128 keys and walks the query rows that see them (dK, dV), one that keeps 128 query rows and walks their keys (dQ);
// both recompute S and dO.V.  That is seven products instead of five, and no sum depends on an order: no atomics.
// As in the forward pass the heads of a group are rows side by side (f = token * group + head), so the sum over a group's heads
// that dK and dV want is part of the contraction, and the query rows that see key j are one run [j G, (j + window + 1) G).
//
// Operands are f16 pairs (streaming_tc.cuh), and a pair's smallest step is absolute.  dO differs between tokens by orders of magnitude (and dS
// by p more), so scales are as local as the sums allow.  Keys and values have one per plane.  Queries and dO have one per tile of 128 query rows: dK and dV
// leave tensor memory after each such tile, and its factors go in where they are added.  Inside a tile a row whose dO is small moves what it has to
// spare from one factor of a sum to the other, for i the row, 2^u_i <= 2^16 its distance from the tile's largest dO in norm, 2^h_i <= 2^6 in components:
//   q_i 2^-u_i   against  dS_i 2^u_i    in dK (scores take 2^u_i back),         dO_i 2^h_i  against  P_i 2^-h_i  in dV.
// dQ's rows are their own: dS_i has the scale that |dO.V - delta| <= 2 |dO_i| max|V| allows.  (With one scale per plane, dQ of rows whose dO was 1e-5
// of the sequence's largest had a relative error of 5e-4.)  A query row with a non-finite component gets NaN for its lse, which reaches exactly the
// gradients of what it sees.
#include <algorithm>

#include "streaming_tc.cuh"

namespace gn {

namespace {

struct BackwardTc {
  StreamRows s;
  PackedKeys pk;
  Packed q, g;                   // queries and dO, rows f
  uint32_t* norms;               // [plane]: largest squared norm of a scaled row of V
  float* off; float* delta; float* score;   // [plane][q.rows]: 15 - h_i - lse in log2 units; delta times the scales of dO, V and dS; from products to log2 units
  float4* own;                   // [plane][q.rows], for dQ: score, dS's scale, delta times that of dO, V and dS, from sums to dQ
  float4* tile;                  // [plane][q_tiles], for dK and dV: (bits of) dS's scale over score's, from sums to dK, to dV
  gn_view out, dout, dq, dk, dv;
  const float* lse;
  int accumulate, vec_in, vec_dq, vec_dkv;
  int q_tiles, key_tiles, sink_tiles, parts_sink, parts, units;
  float* part;                   // [plane][unit][dV, dK][128][DP] of key tiles in several parts
};

// Half a warp per query row f: channels 4 i .. of the 64-channel blocks.
template <int CB>
__device__ __forceinline__ void load_query_row(const StreamRows& s, const gn_view& v, int vec, int r, int hk, int f, float (&x)[4 * CB]) {
  const int l16 = threadIdx.x & 15, t = s.by_G.of(f), h = hk * s.G + f - t * s.G;
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

// x 2^n, cut to what is finite.
__device__ __forceinline__ float times_pow2(float x, int n) { return fminf(fmaxf(ldexpf(x, n), -3.4028234e38f), 3.4028234e38f); }
__device__ __forceinline__ int exponent(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }   // of x >= 0: below 2^(exponent + 1)

constexpr int kThreadsQ = 256, kTileQ = 128, kHalves = kThreadsQ / 16, kRowsEach = kTileQ / kHalves;   // half a warp per row, eight rows one after the other

// Packs q and dO of a tile of query rows and leaves each row's lse, delta and scales in the form that the kernels use: one reading for magnitudes,
// norms and delta = dO.O (four shuffles), a second, from the cache, for the halves.  Bound: HBM, 12 D bytes a row in and 8 D out; 77 us for 2 x 69632 rows of 128 channels (215 MB in, 143 out:
// 4.6 TB/s).  Rows kept in registers between the two, one block of 512 threads an SM, took 99 us: nothing else reads while it waits and stores.
template <int CB>
__global__ void __launch_bounds__(kThreadsQ, 4) stream_query_pack_kernel(const __grid_constant__ BackwardTc p) {
  pdl_trigger();
  const StreamRows& s = p.s;
  const int hk = blockIdx.y, r = blockIdx.z, half = threadIdx.x >> 4, l16 = threadIdx.x & 15, f0 = blockIdx.x * kTileQ + half;
  const int nf = row_span<false>(s, r).q_len * s.G, last = min(p.q.rows, (nf + 15) / 16 * 16);   // a tile is copied in 16s
  if ((int)blockIdx.x * kTileQ >= last) { pdl_wait(); return; }
  const int64_t plane = (int64_t)r * s.Hkv + hk;
  __shared__ uint32_t found[3];   // largest magnitudes of q and dO, largest squared norm of a row of dO times its scale
  if (threadIdx.x < 3) found[threadIdx.x] = 0;
  __syncthreads();
  // lane u of the half warp keeps what row u has: the bits of dO's largest magnitude, its squared norm over that's power of two, delta (not finite: the row is odd)
  uint32_t top_q = 0, my_top = 0;
  float my_sq = 0.0f, my_delta = 0.0f;
#pragma unroll 2
  for (int u = 0; u < kRowsEach; ++u) {
    const int f = f0 + u * kHalves, at = min(f, nf - 1);   // loads without a condition: a row behind the last reads the last, and counts for nothing
    float x[2][4 * CB], o[4 * CB], delta = 0.0f, sq = 0.0f;
    load_query_row<CB>(s, s.q, p.vec_in, r, hk, at, x[0]);
    load_query_row<CB>(s, p.dout, p.vec_in, r, hk, at, x[1]);
    load_query_row<CB>(s, p.out, p.vec_in, r, hk, at, o);
    uint32_t top = 0;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4 * CB; ++e) {
#pragma unroll
      for (int w = 0; w < 2; ++w) if (!finite_bits(x[w][e])) { bad = true; x[w][e] = 0.0f; }
      if (f < nf) top_q = max(top_q, __float_as_uint(x[0][e]) & 0x7fffffffu);
      top = max(top, __float_as_uint(x[1][e]) & 0x7fffffffu);
      delta = fmaf(x[1][e], o[e], delta);
    }
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float by = ldexpf(1.0f, scale_exponent(top));
#pragma unroll
    for (int e = 0; e < 4 * CB; ++e) sq = fmaf(x[1][e] * by, x[1][e] * by, sq);
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) { delta += __shfl_xor_sync(0xffffffffu, delta, d); sq += __shfl_xor_sync(0xffffffffu, sq, d); }
    if ((__ballot_sync(0xffffffffu, bad) >> (threadIdx.x & 16)) & 0xffffu) delta = NAN;
    if (l16 == u && f < nf) { my_top = top; my_sq = sq; my_delta = delta; }
  }
  const uint32_t top_g = __reduce_max_sync(0xffffffffu, my_top);
  top_q = __reduce_max_sync(0xffffffffu, top_q);
  if ((threadIdx.x & 31) == 0) { atomicMax(&found[0], top_q); atomicMax(&found[1], top_g); }
  __syncthreads();
  const int nq = scale_exponent(found[0]), ng = scale_exponent(found[1]);
  my_sq = my_top == 0 ? 0.0f : ldexpf(my_sq, 2 * (ng - scale_exponent(my_top)));   // with the tile's scale
  const uint32_t most_bits = __reduce_max_sync(0xffffffffu, __float_as_uint(my_sq));
  if ((threadIdx.x & 31) == 0) atomicMax(&found[2], most_bits);
  __syncthreads();
  const float most = __uint_as_float(found[2]);
  pdl_wait();   // for what the packing of keys and values found
  const int nk = scale_exponent(p.pk.amax[plane * 2]), nv = scale_exponent(p.pk.amax[plane * 2 + 1]);
  const float norm_v = sqrtf(__uint_as_float(p.norms[plane]));
  // scores below 2^-100 of the products are zeros, whatever their factor
  const float unit = times_pow2(s.scale * kLog2e, -nq - nk), score = copysignf(fminf(fmaxf(fabsf(unit), 0x1p-100f), 0x1p100f), unit);
  // |dO.V| and |delta| of scaled rows are at most their norms' product, below 2^37: with reach < 2^e twice that times 2^(14 - e) is below 2^15.
  // The weights' 2^15 goes out at the same time.
  auto above = [](float reach) { return reach > 0.0f ? exponent(reach) + 1 : 0; };
  const int e_tile = above(sqrtf(most) * norm_v);
  const float grad = ldexpf(1.0f, -1 - e_tile);
  if (threadIdx.x == 0)
    p.tile[plane * p.q_tiles + blockIdx.x] = make_float4(__uint_as_float(__float_as_uint(grad) - __float_as_uint(score)), times_pow2(s.scale, e_tile - 14 - ng - nv - nq),
                                                         ldexpf(1.0f, -15 - ng), 0.0f);
  const int my_up = min(max((exponent(most) - exponent(my_sq) - 1) >> 1, 0), 16);                                                  // the row's norm 2^up is at most the largest
  const int my_lift = min(max(exponent(__uint_as_float(found[1])) - exponent(__uint_as_float(my_top)), 0), 6);   // and its components 2^lift
  const int mine = f0 + l16 * kHalves;
  if (l16 < kRowsEach && mine < last) {
    const int64_t at = plane * p.q.rows + mine;
    const int e = above(sqrtf(my_sq) * norm_v) + my_lift;
    const bool odd = !isfinite(my_delta);
    const float gain = ldexpf(1.0f, my_lift - 1 - e), scaled = odd ? 0.0f : times_pow2(my_delta, ng + my_lift + nv), t = ldexpf(score, my_up);
    float off = 0.0f;
    if (mine < nf) {
      const int token = s.by_G.of(mine);
      off = odd ? NAN : kWeightShift - (float)my_lift - p.lse[stat_offset<false>(s, r, hk * s.G + mine - token * s.G, token)] * kLog2e;
    }
    p.off[at] = off;
    p.delta[at] = scaled * ldexpf(grad, my_up);
    p.score[at] = t;
    p.own[at] = make_float4(t, gain, scaled * gain, times_pow2(s.scale, e - 14 - ng - my_lift - nv - nk));
  }
#pragma unroll 2
  for (int u = kRowsEach - 1; u >= 0; --u) {   // backwards: what was read last is in the cache
    const int f = f0 + u * kHalves, from = (threadIdx.x & 16) + u;
    const float by[2] = {ldexpf(1.0f, nq - __shfl_sync(0xffffffffu, my_up, from)), ldexpf(1.0f, ng + __shfl_sync(0xffffffffu, my_lift, from))};
    float x[2][4 * CB];
    load_query_row<CB>(s, s.q, p.vec_in, r, hk, min(f, nf - 1), x[0]);
    load_query_row<CB>(s, p.dout, p.vec_in, r, hk, min(f, nf - 1), x[1]);
    if (f >= last) continue;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const Packed& dst = w ? p.g : p.q;
#pragma unroll
      for (int e = 0; e < 4 * CB; ++e) x[w][e] = f < nf && finite_bits(x[w][e]) ? x[w][e] * by[w] : 0.0f;
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
  }
}

constexpr int kThreadsB = 640;        // four warpgroups of softmax threads, one for the issuing and the copying warps
constexpr int kRegsSoftmax = 104, kRegsOther = 64;   // shares of the launch's 5 x 96
constexpr int kFlush = 2;             // steps whose sums are left to the tensor core before they are rounded into registers: the error of
                                      // dk and dv grows with it (1: 6.9e-7 of the largest norm, 2: 8.4e-7, 4: 1.2e-6, 8: 2.0e-6)

// Adds N (32 or 16) columns of an accumulator, times z, to registers.
template <int N>
__device__ __forceinline__ void add_columns(uint32_t taddr, float (&acc)[N], float z) {
  uint32_t y[N];
  if constexpr (N == 32) tmem_ld32(taddr, y);
  else tmem_ld16(taddr, y);
  tmem_ld_wait();
#pragma unroll
  for (int e = 0; e < N; ++e) acc[e] = fmaf(__uint_as_float(y[e]), z, acc[e]);
}
// 16 values of a row to f16 pairs in tensor memory: 8 columns of hi, 8 of lo.
__device__ __forceinline__ void store_pairs(uint32_t taddr, const float (&x)[16]) {
  uint32_t y[16];
#pragma unroll
  for (int e = 0; e < 16; e += 2) split_f16(x[e], x[e + 1], y[e >> 1], y[8 + (e >> 1)]);
  __syncwarp();
  tmem_st16(taddr, y);
  tmem_st_wait();
}
// A quarter of a packed hi row that a bulk copy left in shared memory (half a 64-channel block, unswizzled) to 16 columns of tensor memory.
__device__ __forceinline__ void row_to_tmem(uint32_t taddr, const uint8_t* block, int row, int half) {
  uint32_t y[16];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint4 v = *reinterpret_cast<const uint4*>(block + row * 128 + (((half * 4 + c) ^ (row & 7)) << 4));
    y[4 * c] = v.x; y[4 * c + 1] = v.y; y[4 * c + 2] = v.z; y[4 * c + 3] = v.w;
  }
  __syncwarp();
  tmem_st16(taddr, y);
}
// A thread's QC channels, from ch on, of a gradient row (dst null: no row); a warp's 32 threads hold as many rows.
template <int QC>
__device__ __forceinline__ void write_row(float* dst, int ch, int D, float (&acc)[QC], float z, bool accumulate, bool vec) {
#pragma unroll
  for (int e = 0; e < QC; ++e) acc[e] *= z;
  if (vec) {
    constexpr int N = QC / 4;
    const int lane = threadIdx.x & 31, c = ch + (lane & (N - 1)) * 4;
    transpose_blocks<N>(acc);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float* at = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), (lane & ~(N - 1)) + k));
      if (!at || c >= D) continue;
      float4 v = make_float4(acc[4 * k], acc[4 * k + 1], acc[4 * k + 2], acc[4 * k + 3]);
      if (accumulate) { const float4 o = *reinterpret_cast<const float4*>(at + c); v.x = __fadd_rn(o.x, v.x); v.y = __fadd_rn(o.y, v.y); v.z = __fadd_rn(o.z, v.z); v.w = __fadd_rn(o.w, v.w); }
      *reinterpret_cast<float4*>(at + c) = v;
    }
  } else if (dst) {
#pragma unroll
    for (int e = 0; e < QC; ++e) if (ch + e < D) dst[ch + e] = accumulate ? __fadd_rn(dst[ch + e], acc[e]) : acc[e];
  }
}

// dK and dV.  One CTA per (128 keys or a part of their query rows, kv head, sequence): S^T = K Q^T and dP^T = V dO^T of 64 query rows a
// step, a softmax thread per (key, 16 query rows) writes P^T over the scores and, once dV += P^T dO has read it, dS^T over P^T, from where
// dK += dS^T Q takes it: dP^T is free for the next step as soon as it is read (with dS^T in its place the chain dP, dS, dK, next dP
// took 4500 cycles a step).  The hi half of K lives in tensor memory too, which leaves room for two stages of Q and dO.  Two warps issue,
// one the scores and one the sums, so that neither's waits hold up the other's instructions.
// Tensor memory: S^T / P^T / dS^T 2 x 64 columns, dP^T 64, K hi 64, dV 128, dK 128.  Shared memory: V 64 KB, K lo 32 KB, 2 x (Q 32 KB + dO 32 KB).
// Every kFlush steps dV and dK are added to float32 registers (32 + 32 a thread), one step later, between that step's weights and
// its dS, while the products that end the chunk run.  Bound: tensor pipe, 48 instructions of 46 cycles and 24 of 64 a step.
// 2 x 8704 tokens, 8 heads on one, window 512: 337 us, tensor pipe busy 47 %, 4500 to 5700 cycles a step.
template <int DP>
__global__ void __launch_bounds__(kThreadsB, 1) stream_tc_dkv_kernel(const __grid_constant__ BackwardTc p) {
  constexpr int CB = DP / 64, QC = DP / 4;
  constexpr uint32_t SLOT = CB * 16384u, OFF_KL = CB * 32768u, OFF_Q = OFF_KL + CB * 16384u, OFF_G = OFF_Q + 2 * SLOT, STATS = OFF_G + 2 * SLOT, BARS = STATS + 1536, FACTORS = BARS + 208;
  constexpr uint32_t COL_S = 0, COL_DP = 128, COL_KH = 192, COL_DV = 256, COL_DK = 384;
  extern __shared__ uint8_t smem_raw[];
  const StreamRows& s = p.s;
  const int hk = blockIdx.y, r = blockIdx.z, x0 = blockIdx.x;
  const bool sink = x0 < p.sink_tiles * p.parts_sink;
  const int parts = sink ? p.parts_sink : p.parts, y0 = sink ? x0 : x0 - p.sink_tiles * p.parts_sink;
  const int kt = (sink ? 0 : p.sink_tiles) + y0 / parts, part_i = y0 % parts, k0 = kt * 128;
  const int len = row_span<false>(s, r).ctx;
  if (k0 >= len && parts > 1) { pdl_wait(); return; }   // the summing kernel does not look at padding
  const int nf = len * s.G;
  const int64_t t_end = (s.window < 0 || k0 < s.sinks) ? len : min((int64_t)len, (int64_t)k0 + 128 + s.window);
  const int f_begin = k0 * s.G, f_end = (int)t_end * s.G;
  const int steps = k0 < len ? (f_end - f_begin + 63) / 64 : 0, per = (steps + parts * kFlush - 1) / (parts * kFlush) * kFlush;   // whole tiles of query rows
  const int i0 = part_i * per, n = max(0, min(steps, i0 + per) - i0);
  const int64_t plane = (int64_t)r * s.Hkv + hk;

  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + BARS;
  const uint32_t v_full = bars, kh_ready = bars + 8, dp_full = bars + 16, ds_full = bars + 24, acc_full = bars + 32, acc_empty = bars + 40, dp_free = bars + 152, kh_full = bars + 144, tmem_slot = bars + 176;
  auto q_full = [&](int i) { return bars + 48u + 8u * i; };
  auto g_full = [&](int i) { return bars + 64u + 8u * i; };
  auto q_empty = [&](int i) { return bars + 80u + 8u * i; };
  auto g_empty = [&](int i) { return bars + 96u + 8u * i; };
  auto s_full = [&](int i) { return bars + 112u + 8u * i; };
  auto p_full = [&](int i) { return bars + 128u + 8u * i; };
  auto s_free = [&](int i) { return bars + 160u + 8u * i; };
  auto v_done = [&](int i) { return bars + 184u + 8u * i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    static_assert(kFlush * 64 == kTileQ && FACTORS + 32 <= BARS + 256);   // a tile's sums have its factors
    mbar_init(v_full, 1); mbar_init(kh_full, 1); mbar_init(kh_ready, 512); mbar_init(dp_full, 1); mbar_init(ds_full, 512); mbar_init(acc_full, 1); mbar_init(acc_empty, 512); mbar_init(dp_free, 512);
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full(i), 1); mbar_init(g_full(i), 1); mbar_init(q_empty(i), 1); mbar_init(g_empty(i), 2); mbar_init(s_full(i), 1); mbar_init(p_full(i), 512);
      mbar_init(s_free(i), 1); mbar_init(v_done(i), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 16) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gen + BARS + 176);
  pdl_wait();
  pdl_trigger();   // not before: the dQ kernel starts without a wait
  auto row0 = [&](int i) { return f_begin + (i0 + i) * 64; };
  auto rows16 = [&](int i) { return min(64, (f_end - row0(i) + 15) & ~15); };

  if (warp >= 16) {
    regs_dec<kRegsOther>();
    if (warp == 17 && lane == 0 && n > 0) {
      // ----------------------------------------------------------- copies
      const int keys = min(128, (len - k0 + 15) & ~15);
      mbar_expect_tx(v_full, (uint32_t)CB * 3u * keys * 128u);
      const uint8_t* vp = p.pk.v.data + plane * p.pk.v.plane_bytes(CB); const uint8_t* kp = p.pk.k.data + plane * p.pk.k.plane_bytes(CB);
#pragma unroll 1
      for (int b = 0; b < CB * 2; ++b) bulk_load(base + b * 16384, vp + ((int64_t)b * p.pk.v.rows + k0) * 128, keys * 128, v_full);
#pragma unroll 1
      for (int b = 0; b < CB; ++b) bulk_load(base + OFF_KL + b * 16384, kp + ((int64_t)(2 * b + 1) * p.pk.k.rows + k0) * 128, keys * 128, v_full);
      // K hi passes through the second dO stage on its way to tensor memory
      mbar_expect_tx(kh_full, (uint32_t)CB * keys * 128u);
#pragma unroll 1
      for (int b = 0; b < CB; ++b) bulk_load(base + OFF_G + SLOT + b * 16384, kp + ((int64_t)(2 * b) * p.pk.k.rows + k0) * 128, keys * 128, kh_full);
      const uint8_t* qp = p.q.data + plane * p.q.plane_bytes(CB); const uint8_t* gp = p.g.data + plane * p.g.plane_bytes(CB);
      bool ok = true;
      for (int i = 0; i < n && ok; ++i) {
        const int rows = rows16(i), f = row0(i), b2 = i & 1;
        if (i >= 2) ok = hold(q_empty(b2), ((i >> 1) - 1) & 1);
        if (!ok) break;
        mbar_expect_tx(q_full(b2), (uint32_t)CB * 2u * rows * 128u + 3u * rows * 4u + 16u);
#pragma unroll 1
        for (int b = 0; b < CB * 2; ++b) bulk_load(base + OFF_Q + b2 * SLOT + b * 8192, qp + ((int64_t)b * p.q.rows + f) * 128, rows * 128, q_full(b2));
        bulk_load(base + STATS + b2 * 768, p.off + plane * p.q.rows + f, rows * 4, q_full(b2));
        bulk_load(base + STATS + b2 * 768 + 256, p.delta + plane * p.q.rows + f, rows * 4, q_full(b2));
        bulk_load(base + STATS + b2 * 768 + 512, p.score + plane * p.q.rows + f, rows * 4, q_full(b2));
        bulk_load(base + FACTORS + b2 * 16, p.tile + plane * p.q_tiles + (f >> 7), 16, q_full(b2));
        if (i == 1) ok = hold(kh_ready, 0);
        if (i >= 2) ok = hold(g_empty(b2), ((i >> 1) - 1) & 1);
        if (!ok) break;
        mbar_expect_tx(g_full(b2), (uint32_t)CB * 2u * rows * 128u);
#pragma unroll 1
        for (int b = 0; b < CB * 2; ++b) bulk_load(base + OFF_G + b2 * SLOT + b * 8192, gp + ((int64_t)b * p.g.rows + f) * 128, rows * 128, g_full(b2));
      }
      if (!ok)   // copies in flight land before the CTA goes
        for (int i = 0; i < 2; ++i)
          for (int ph = 0; ph < 2; ++ph) { hold(q_full(i), ph); hold(g_full(i), ph); }
      hold(v_full, 0);
      hold(kh_full, 0);
    }
    if (warp == 16 && n > 0) {
      // ----------------------------------------------------------- scores: S^T(0), dP^T(0), S^T(1), dP^T(1), ...
      const uint32_t el = elect_lane();
      bool ok = hold_warp(v_full, 0) && hold_warp(kh_ready, 0);
      tc_fence_after();
      const uint64_t kl = smem_desc_sw128(base + OFF_KL), vd = smem_desc_sw128(base);
      for (int i = 0; i < n && ok; ++i) {
        const int b2 = i & 1;
        const uint32_t id = instr_desc_f16(128, rows16(i), 0);
        ok = hold_warp(q_full(b2), (i >> 1) & 1) && (i < 2 || hold_warp(s_free(b2), ((i >> 1) - 1) & 1));
        if (!ok) break;
        tc_fence_after();
        {
          const uint32_t d = tmem + COL_S + b2 * 64;
          const uint64_t q = smem_desc_sw128(base + OFF_Q + b2 * SLOT);
#pragma unroll 2
          for (int ks = 0; ks < CB * 4; ++ks) {   // a 64-channel block is 16 KB of 128 rows, 2 x 8 KB of 64
            const uint32_t in = (ks & 3) * 2;
            umma_f16(el, d, kl + (ks >> 2) * 1024 + in, q + (ks >> 2) * 1024 + in, id, ks > 0);
            umma_f16_ts(el, d, tmem + COL_KH + ks * 8, q + (ks >> 2) * 1024 + 512 + in, id, 1);
          }
#pragma unroll 2
          for (int ks = 0; ks < CB * 4; ++ks) umma_f16_ts(el, d, tmem + COL_KH + ks * 8, q + (ks >> 2) * 1024 + (ks & 3) * 2, id, 1);
          commit_by(el, s_full(b2));
        }
        ok = hold_warp(g_full(b2), (i >> 1) & 1) && (i < 1 || hold_warp(dp_free, (i - 1) & 1));
        if (!ok) break;
        tc_fence_after();
        {
          const uint32_t d = tmem + COL_DP;
          const uint64_t g = smem_desc_sw128(base + OFF_G + b2 * SLOT);
#pragma unroll 2
          for (int ks = 0; ks < CB * 4; ++ks) {
            const uint64_t a = vd + (ks >> 2) * 2048 + (ks & 3) * 2, bb = g + (ks >> 2) * 1024 + (ks & 3) * 2;
            umma_f16(el, d, a + 1024, bb, id, ks > 0);
            umma_f16(el, d, a, bb + 512, id, 1);
          }
#pragma unroll 2
          for (int ks = 0; ks < CB * 4; ++ks) umma_f16(el, d, vd + (ks >> 2) * 2048 + (ks & 3) * 2, g + (ks >> 2) * 1024 + (ks & 3) * 2, id, 1);
          commit_by(el, dp_full);
          commit_by(el, g_empty(b2));
        }
      }
    }
    if (warp == 18 && n > 0) {
      // ----------------------------------------------------------- sums: dV(0), dK(0), dV(1), ...
      const uint32_t el = elect_lane(), id = instr_desc_f16(128, DP, 1);
      bool ok = true;
      auto accumulate = [&](uint32_t d, uint32_t a, uint32_t slot, int slices, uint32_t fresh) {
        const uint64_t b = smem_desc_mn(slot, 16384);
#pragma unroll 1
        for (int ks = 0; ks < slices; ++ks) {
          umma_f16_ts(el, d, a + ks * 16 + 8, b + ks * 128, id, ks > 0 ? 1u : fresh);
          umma_f16_ts(el, d, a + ks * 16, b + ks * 128 + 512, id, 1);
        }
#pragma unroll 1
        for (int ks = 0; ks < slices; ++ks) umma_f16_ts(el, d, a + ks * 16, b + ks * 128, id, 1);
      };
      for (int i = 0; i < n && ok; ++i) {
        const int b2 = i & 1, slices = rows16(i) >> 4;
        const uint32_t fresh = i % kFlush == 0 ? 0u : 1u;
        ok = hold_warp(p_full(b2), (i >> 1) & 1) && hold_warp(g_full(b2), (i >> 1) & 1) && (fresh || i == 0 || hold_warp(acc_empty, (i / kFlush - 1) & 1));
        if (!ok) break;
        tc_fence_after();
        accumulate(tmem + COL_DV, tmem + COL_S + b2 * 64, base + OFF_G + b2 * SLOT, slices, fresh);
        commit_by(el, v_done(b2));
        commit_by(el, g_empty(b2));
        ok = hold_warp(ds_full, i & 1);
        if (!ok) break;
        tc_fence_after();
        accumulate(tmem + COL_DK, tmem + COL_S + b2 * 64, base + OFF_Q + b2 * SLOT, slices, fresh);
        commit_by(el, q_empty(b2));
        commit_by(el, s_free(b2));
        if ((i + 1) % kFlush == 0 || i + 1 == n) commit_by(el, acc_full);
      }
      // what the instructions still signal, nobody else waits for: it has arrived before this CTA's shared memory goes to another
      for (int i = max(0, n - 2); i < n && ok; ++i)
        ok = hold_warp(q_empty(i & 1), (i >> 1) & 1) && hold_warp(g_empty(i & 1), (i >> 1) & 1) && hold_warp(s_free(i & 1), (i >> 1) & 1);
    }
  } else {
    regs_inc<kRegsSoftmax>();
    const int quarter = warp & 3, part = warp >> 2, row = quarter * 32 + lane, key = k0 + row;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    bool ok = true;
    if (n > 0) {
      ok = hold_warp(kh_full, 0);
      if (part < 2 * CB) row_to_tmem(lane_addr + COL_KH + part * 16, gen + OFF_G + SLOT + (part >> 1) * 16384, row, part & 1);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(kh_ready);
    }
    // the query rows that see the key
    const int f_lo = key < len ? key * s.G : 0;
    const int f_hi = key >= len ? 0 : (s.window < 0 || key < s.sinks) ? nf : (int)min((int64_t)nf, ((int64_t)key + s.window + 1) * s.G);
    float dv[QC], dk[QC];
#pragma unroll
    for (int e = 0; e < QC; ++e) dv[e] = dk[e] = 0.0f;
    float zk = 0.0f, zv = 0.0f;   // from sums to gradients, of the query rows whose sums stand in tensor memory
    auto flush = [&](int chunk) {
      ok = ok && hold_warp(acc_full, chunk & 1);
      tc_fence_after();
      add_columns<QC>(lane_addr + COL_DV + part * QC, dv, zv);
      add_columns<QC>(lane_addr + COL_DK + part * QC, dk, zk);
      tc_fence_before();
      mbar_arrive(acc_empty);
    };
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int f0 = row0(i) + part * 16;
      const uint32_t see = (uint32_t)(bits_below(f_hi - f0) & ~bits_below(f_lo - f0));
      const float4* off = reinterpret_cast<const float4*>(gen + STATS + (i & 1) * 768 + part * 64);   // and delta 16 on, score 32 on
      float w[16];
      ok = ok && hold_warp(q_full(i & 1), (i >> 1) & 1) && hold_warp(s_full(i & 1), (i >> 1) & 1);
      tc_fence_after();
      {
        uint32_t y[16];
        tmem_ld16(lane_addr + COL_S + (i & 1) * 64 + part * 16, y);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 c = off[e >> 2], t = off[32 + (e >> 2)];
          w[e] = exp2_fast(fmaf(__uint_as_float(y[e]), t.x, c.x)); w[e + 1] = exp2_fast(fmaf(__uint_as_float(y[e + 1]), t.y, c.y));
          w[e + 2] = exp2_fast(fmaf(__uint_as_float(y[e + 2]), t.z, c.z)); w[e + 3] = exp2_fast(fmaf(__uint_as_float(y[e + 3]), t.w, c.w));
        }
      }
      const bool whole = __all_sync(0xffffffffu, (see & 0xffffu) == 0xffffu);
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 16; ++e) if (!((see >> e) & 1u)) w[e] = 0.0f;
      }
      store_pairs(lane_addr + COL_S + (i & 1) * 64 + part * 16, w);
      tc_fence_before();
      mbar_arrive(p_full(i & 1));
      if (i > 0 && i % kFlush == 0) flush(i / kFlush - 1);
      const float4 fc = *reinterpret_cast<const float4*>(gen + FACTORS + (i & 1) * 16);
      if (i % kFlush == 0) { zk = fc.y; zv = fc.z; }
      ok = ok && hold_warp(dp_full, i & 1);
      tc_fence_after();
      {
        uint32_t y[16];
        tmem_ld16(lane_addr + COL_DP + part * 16, y);
        tmem_ld_wait();
        tc_fence_before();
        mbar_arrive(dp_free);
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 c = off[16 + (e >> 2)], t = off[32 + (e >> 2)];
          auto gain = [&](float score) { return __uint_as_float(__float_as_uint(score) + __float_as_uint(fc.x)); };   // dS's scale goes with the score's
          w[e] *= fmaf(__uint_as_float(y[e]), gain(t.x), -c.x); w[e + 1] *= fmaf(__uint_as_float(y[e + 1]), gain(t.y), -c.y);
          w[e + 2] *= fmaf(__uint_as_float(y[e + 2]), gain(t.z), -c.z); w[e + 3] *= fmaf(__uint_as_float(y[e + 3]), gain(t.w), -c.w);
        }
      }
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 16; ++e) if (!((see >> e) & 1u)) w[e] = 0.0f;   // what stands in a masked place may not be a number
      }
      ok = ok && hold_warp(v_done(i & 1), (i >> 1) & 1);
      tc_fence_after();
      store_pairs(lane_addr + COL_S + (i & 1) * 64 + part * 16, w);
      tc_fence_before();
      mbar_arrive(ds_full);
    }
    if (n > 0) flush((n - 1) / kFlush);
    const float z = ok ? 1.0f : NAN;
    if (parts > 1) {
      float* at = p.part + (((plane * p.units + x0) * 2) * 128 + row) * DP;
      write_row<QC>(at, part * QC, DP, dv, z, false, true);
      write_row<QC>(at + 128 * DP, part * QC, DP, dk, z, false, true);
    } else {
      write_row<QC>(key < s.seq ? p.dv.data + token_offset<false>(p.dv, r, hk, key) : nullptr, part * QC, s.D, dv, z, p.accumulate, p.vec_dkv);
      write_row<QC>(key < s.seq ? p.dk.data + token_offset<false>(p.dk, r, hk, key) : nullptr, part * QC, s.D, dk, z, p.accumulate, p.vec_dkv);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 16) tmem_dealloc(tmem, 512);
}

// Sums the parts of key tiles that were divided, in their order: DP / 4 threads per key row and tensor.  Bound: reading them; 23 us for 63 MB.
template <int DP>
__global__ void __launch_bounds__(256) stream_tc_dkv_sum_kernel(const __grid_constant__ BackwardTc p) {
  pdl_wait();
  constexpr int LANES = DP / 4;
  const StreamRows& s = p.s;
  const int hk = blockIdx.y, r = blockIdx.z >> 1, which = blockIdx.z & 1, key = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, ch = threadIdx.x % LANES * 4;
  if (key >= s.seq) return;
  const int kt = key / 128;
  const bool sink = kt < p.sink_tiles;
  const int parts = sink ? p.parts_sink : p.parts, unit = sink ? kt * parts : p.sink_tiles * p.parts_sink + (kt - p.sink_tiles) * parts;
  if (parts == 1) return;
  const int64_t plane = (int64_t)r * s.Hkv + hk;
  float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (key < row_span<false>(s, r).ctx) {
    const float* at = p.part + (((plane * p.units + unit) * 2 + which) * 128 + key % 128) * DP + ch;
#pragma unroll 8
    for (int i = 0; i < parts; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(at + (int64_t)i * 2 * 128 * DP);
      x[0] += v.x; x[1] += v.y; x[2] += v.z; x[3] += v.w;
    }
  }
  const gn_view& view = which ? p.dk : p.dv;
  float* dst = view.data + token_offset<false>(view, r, hk, key) + ch;
  if (p.vec_dkv) {
    if (ch >= s.D) return;
    float4 v = make_float4(x[0], x[1], x[2], x[3]);
    if (p.accumulate) { const float4 o = *reinterpret_cast<const float4*>(dst); v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w; }
    *reinterpret_cast<float4*>(dst) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) if (ch + e < s.D) dst[e] = p.accumulate ? dst[e] + x[e] : x[e];
  }
}

// dQ.  One CTA per (128 query rows, kv head, sequence): S = Q K^T and dP = dO V^T of 64 keys a step, dS in place of dP, dQ += dS K with
// dS from tensor memory and the same K tile read the other way.  Threads, issuing warps and the rounding of sums as above.
// It needs nothing from the dK and dV kernel, which stands before it on the stream: its CTAs fill the SMs that that one's last CTAs leave
// free.  (They start once every CTA there has seen the packing kernels complete, and end after it has ended.)
// Tensor memory: Q hi 64 columns, dO hi 64, S 2 x 64, dP 2 x 64, dQ 128.  Shared memory: Q lo, dO lo 32 KB each, 3 K and 2 V tiles of 32 KB.
// Bound: tensor pipe; the call above 205 us, busy 41 %: 4050 cycles a step, and 5000 and 3500 for a CTA's start and end.
template <int DP>
__global__ void __launch_bounds__(kThreadsB, 1) stream_tc_dq_kernel(const __grid_constant__ BackwardTc p) {
  constexpr int CB = DP / 64, QC = DP / 4;
  constexpr uint32_t SLOT = CB * 16384u, OFF_GL = CB * 16384u, OFF_K = 2 * CB * 16384u, OFF_V = OFF_K + 3 * SLOT, BARS = OFF_V + 2 * SLOT;
  constexpr uint32_t COL_Q = 0, COL_G = 64, COL_S = 128, COL_DP = 256, COL_DQ = 384;
  extern __shared__ uint8_t smem_raw[];
  const StreamRows& s = p.s;
  const int hk = blockIdx.y, r = blockIdx.z, tile = p.q_tiles - 1 - (int)blockIdx.x, f0 = tile * 128;
  const int len = row_span<false>(s, r).ctx, nf = len * s.G;
  KeyRuns runs{0, 0, 0};
  if (f0 < nf) runs = key_runs(s, s.by_G.of(f0), s.by_G.of(min(f0 + 127, nf - 1)));
  const int n = (runs.total + 63) / 64;
  const int64_t plane = (int64_t)r * s.Hkv + hk;

  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + BARS;
  const uint32_t lo_full = bars, hi_ready = bars + 8, acc_full = bars + 16, acc_empty = bars + 24, hi_full = bars + 160, tmem_slot = bars + 176;
  auto k_full = [&](int i) { return bars + 32u + 8u * i; };
  auto k_empty = [&](int i) { return bars + 56u + 8u * i; };
  auto v_full = [&](int i) { return bars + 80u + 8u * i; };
  auto v_empty = [&](int i) { return bars + 96u + 8u * i; };
  auto sp_full = [&](int i) { return bars + 112u + 8u * i; };
  auto ds_full = [&](int i) { return bars + 128u + 8u * i; };
  auto ds_free = [&](int i) { return bars + 144u + 8u * i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(lo_full, 1); mbar_init(hi_full, 1); mbar_init(hi_ready, 512); mbar_init(acc_full, 1); mbar_init(acc_empty, 512);
    for (int i = 0; i < 3; ++i) { mbar_init(k_full(i), 1); mbar_init(k_empty(i), 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(v_full(i), 1); mbar_init(v_empty(i), 1); mbar_init(sp_full(i), 1); mbar_init(ds_full(i), 512); mbar_init(ds_free(i), 1); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_trigger();
  if (warp == 16) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gen + BARS + 176);
  auto rows16 = [&](int j) { return min(64, (runs.total - j * 64 + 15) & ~15); };

  if (warp >= 16) {
    regs_dec<kRegsOther>();
    if (warp == 17 && lane == 0 && n > 0) {
      const int rows = min(128, (nf - f0 + 15) & ~15);
      mbar_expect_tx(lo_full, (uint32_t)CB * 2u * rows * 128u);
      for (int w = 0; w < 2; ++w) {
        const Packed& src = w ? p.g : p.q;
        for (int b = 0; b < CB; ++b)
          bulk_load(base + w * OFF_GL + b * 16384, src.data + plane * src.plane_bytes(CB) + ((int64_t)(2 * b + 1) * src.rows + f0) * 128, rows * 128, lo_full);
      }
      // the hi halves pass through the last K and V tiles' places on their way to tensor memory
      mbar_expect_tx(hi_full, (uint32_t)CB * 2u * rows * 128u);
      for (int w = 0; w < 2; ++w) {
        const Packed& src = w ? p.g : p.q;
        for (int b = 0; b < CB; ++b)
          bulk_load(base + (w ? OFF_V + SLOT : OFF_K + 2 * SLOT) + b * 16384, src.data + plane * src.plane_bytes(CB) + ((int64_t)(2 * b) * src.rows + f0) * 128, rows * 128, hi_full);
      }
      auto copy_tile = [&](const Packed& src, uint32_t dst, uint32_t bar, int j) {
        const int c0 = j * 64, m = rows16(j), na = min(max(runs.a_len - c0, 0), m), nb = m - na;
        const uint8_t* from = src.data + plane * src.plane_bytes(CB) + (int64_t)c0 * 128;
        mbar_expect_tx(bar, (uint32_t)CB * 2u * m * 128u);
#pragma unroll 1
        for (int b = 0; b < CB * 2; ++b) {
          if (na) bulk_load(dst, from, na * 128, bar);
          if (nb) bulk_load(dst + na * 128, from + (int64_t)(na + runs.shift) * 128, nb * 128, bar);
          dst += 8192; from += (int64_t)src.rows * 128;
        }
      };
      bool ok = true;
      for (int j = 0; j < n && ok; ++j) {
        if (j == 2) ok = hold(hi_ready, 0);
        if (j >= 3) ok = hold(k_empty(j % 3), (j / 3 - 1) & 1);
        if (!ok) break;
        copy_tile(p.pk.k, base + OFF_K + (j % 3) * SLOT, k_full(j % 3), j);
        if (j == 1) ok = hold(hi_ready, 0);
        if (j >= 2) ok = hold(v_empty(j & 1), ((j >> 1) - 1) & 1);
        if (!ok) break;
        copy_tile(p.pk.v, base + OFF_V + (j & 1) * SLOT, v_full(j & 1), j);
      }
      if (!ok)
        for (int ph = 0; ph < 2; ++ph) {
          for (int i = 0; i < 3; ++i) hold(k_full(i), ph);
          for (int i = 0; i < 2; ++i) hold(v_full(i), ph);
        }
      hold(lo_full, 0);
      hold(hi_full, 0);
    }
    if (warp == 16 && n > 0) {
      // ----------------------------------------------------------- scores
      const uint32_t el = elect_lane();
      bool ok = hold_warp(lo_full, 0) && hold_warp(hi_ready, 0);
      tc_fence_after();
      for (int j = 0; j < n && ok; ++j) {
        const uint32_t id = instr_desc_f16(128, rows16(j), 0);
        for (int w = 0; w < 2 && ok; ++w) {
          ok = w ? hold_warp(v_full(j & 1), (j >> 1) & 1) : hold_warp(k_full(j % 3), (j / 3) & 1) && (j < 2 || hold_warp(ds_free(j & 1), ((j >> 1) - 1) & 1));
          if (!ok) break;
          tc_fence_after();
          const uint32_t d = tmem + (w ? COL_DP : COL_S) + (j & 1) * 64, hi = tmem + (w ? COL_G : COL_Q);
          const uint64_t lo = smem_desc_sw128(base + w * OFF_GL), slot = smem_desc_sw128(w ? base + OFF_V + (j & 1) * SLOT : base + OFF_K + (j % 3) * SLOT);
#pragma unroll 2
          for (int ks = 0; ks < CB * 4; ++ks) {
            const uint32_t in = (ks >> 2) * 1024 + (ks & 3) * 2;
            umma_f16(el, d, lo + in, slot + in, id, ks > 0);
            umma_f16_ts(el, d, hi + ks * 8, slot + in + 512, id, 1);
          }
#pragma unroll 2
          for (int ks = 0; ks < CB * 4; ++ks) umma_f16_ts(el, d, hi + ks * 8, slot + (ks >> 2) * 1024 + (ks & 3) * 2, id, 1);
        }
        if (!ok) break;
        commit_by(el, v_empty(j & 1));
        commit_by(el, sp_full(j & 1));
      }
      for (int j = max(0, n - 2); j < n && ok; ++j) ok = hold_warp(v_empty(j & 1), (j >> 1) & 1);   // the last signals, as above
    }
    if (warp == 18 && n > 0) {
      // ----------------------------------------------------------- sums
      const uint32_t el = elect_lane(), id = instr_desc_f16(128, DP, 1);
      bool ok = true;
      for (int j = 0; j < n && ok; ++j) {
        const uint32_t fresh = j % kFlush == 0 ? 0u : 1u;
        ok = hold_warp(ds_full(j & 1), (j >> 1) & 1) && hold_warp(k_full(j % 3), (j / 3) & 1) && (fresh || j == 0 || hold_warp(acc_empty, (j / kFlush - 1) & 1));
        if (!ok) break;
        tc_fence_after();
        const uint32_t a = tmem + COL_DP + (j & 1) * 64;
        const uint64_t b = smem_desc_mn(base + OFF_K + (j % 3) * SLOT, 16384);
        const int slices = rows16(j) >> 4;
#pragma unroll 1
        for (int ks = 0; ks < slices; ++ks) {
          umma_f16_ts(el, tmem + COL_DQ, a + ks * 16 + 8, b + ks * 128, id, ks > 0 ? 1u : fresh);
          umma_f16_ts(el, tmem + COL_DQ, a + ks * 16, b + ks * 128 + 512, id, 1);
        }
#pragma unroll 1
        for (int ks = 0; ks < slices; ++ks) umma_f16_ts(el, tmem + COL_DQ, a + ks * 16, b + ks * 128, id, 1);
        commit_by(el, k_empty(j % 3));
        commit_by(el, ds_free(j & 1));
        if ((j + 1) % kFlush == 0 || j + 1 == n) commit_by(el, acc_full);
      }
      for (int j = max(0, n - 3); j < n && ok; ++j)
        ok = hold_warp(k_empty(j % 3), (j / 3) & 1) && (j + 2 < n || hold_warp(ds_free(j & 1), (j >> 1) & 1));
    }
  } else {
    regs_inc<kRegsSoftmax>();
    const int quarter = warp & 3, part = warp >> 2, row = quarter * 32 + lane, f = f0 + row;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    const bool live = f < nf;
    const int t = s.by_G.of(f), h = hk * s.G + f - t * s.G;
    float off = 0.0f;
    float4 fc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    bool ok = true;
    if (n > 0) {
      ok = hold_warp(hi_full, 0);
#pragma unroll
      for (int w = 0; w < 2; ++w)
        if (part < 2 * CB)
          row_to_tmem(lane_addr + (w ? COL_G : COL_Q) + part * 16, gen + (w ? OFF_V + SLOT : OFF_K + 2 * SLOT) + (part >> 1) * 16384, row, part & 1);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(hi_ready);
      if (live) { off = p.off[plane * p.q.rows + f]; fc = p.own[plane * p.q.rows + f]; }
    }
    const int s_end = live ? min(s.sinks, t + 1) : 0;
    const int lo_key = live ? (s.window < 0 ? 0 : max(0, t - s.window)) - runs.shift : 0, hi_key = live ? t - runs.shift : -1;
    float acc[QC];
#pragma unroll
    for (int e = 0; e < QC; ++e) acc[e] = 0.0f;
    auto flush = [&](int chunk) {   // one step later, as above
      ok = ok && hold_warp(acc_full, chunk & 1);
      tc_fence_after();
      add_columns<QC>(lane_addr + COL_DQ + part * QC, acc, 1.0f);
      tc_fence_before();
      mbar_arrive(acc_empty);
    };
#pragma unroll 1
    for (int j = 0; j < n; ++j) {
      const int c0 = j * 64 + part * 16;
      const uint32_t see = (uint32_t)(bits_below(s_end - c0) | (bits_below(hi_key + 1 - c0) & ~bits_below(lo_key - c0)));
      ok = ok && hold_warp(sp_full(j & 1), (j >> 1) & 1);
      tc_fence_after();
      float w[16];
      {
        uint32_t y[16], z[16];
        tmem_ld16(lane_addr + COL_S + (j & 1) * 64 + part * 16, y);
        tmem_ld16(lane_addr + COL_DP + (j & 1) * 64 + part * 16, z);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = exp2_fast(fmaf(__uint_as_float(y[e]), fc.x, off)) * fmaf(__uint_as_float(z[e]), fc.y, -fc.z);
      }
      if (!__all_sync(0xffffffffu, (see & 0xffffu) == 0xffffu)) {
#pragma unroll
        for (int e = 0; e < 16; ++e) if (!((see >> e) & 1u)) w[e] = 0.0f;
      }
      store_pairs(lane_addr + COL_DP + (j & 1) * 64 + part * 16, w);
      tc_fence_before();
      mbar_arrive(ds_full(j & 1));
      if (j > 0 && j % kFlush == 0) flush(j / kFlush - 1);
    }
    if (n > 0) flush((n - 1) / kFlush);
    write_row<QC>(f < s.seq * s.G ? p.dq.data + token_offset<false>(p.dq, r, h, t) : nullptr, part * QC, s.D, acc, ok ? fc.w : NAN, p.accumulate, p.vec_dq);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 16) tmem_dealloc(tmem, 512);
  pdl_wait();
}

// ------------------------------------------------------------------ host
int64_t carve_backward(const StreamRows& s, void* workspace, BackwardTc* b) {
  const int DP = s.D <= 64 ? 64 : 128, CB = DP / 64;
  const int64_t planes = (int64_t)s.rows * s.Hkv;
  b->q_tiles = ceil_div((int64_t)s.seq * s.G, 128);
  b->key_tiles = ceil_div(s.seq, 128);
  // Key tiles whose steps (64 query rows each) would make a long tail are divided.  A tile of sinks is seen by every later
  // query and gets as many parts as make them about as long as the others'.
  const bool windowed = s.window >= 0 && s.sinks > 0 && (int64_t)s.window + 128 < s.seq;
  b->sink_tiles = windowed ? std::min(b->key_tiles, ceil_div(s.sinks, 128)) : 0;
  const int64_t reach = s.window >= 0 ? std::min<int64_t>(s.seq, (int64_t)s.window + 128) : s.seq;
  const int64_t steps = ceil_div(reach * s.G, 64), steps_sink = ceil_div((int64_t)s.seq * s.G, 64);
  // Parts: the fewest rounds of 148 CTAs, counted in steps with 5 for a CTA's start and end, and the partial results' way to memory
  // and back (0.02 of a step a CTA).
  double best = 0.0;
  for (int parts = 1; parts <= 16 && (parts == 1 || steps / parts >= 8); ++parts) {
    const int64_t sink_parts = b->sink_tiles ? std::max<int64_t>(1, ceil_div(steps_sink * parts, steps)) : 1;
    const int64_t units = planes * (b->sink_tiles * sink_parts + (int64_t)(b->key_tiles - b->sink_tiles) * parts);
    const double cost = (double)ceil_div(units, 148) * (ceil_div(steps, parts) + 5) + (parts > 1 ? 0.02 * (double)units : 0.0);
    if (parts == 1 || cost < best) { best = cost; b->parts = parts; b->parts_sink = (int)sink_parts; }
  }
  b->units = b->sink_tiles * b->parts_sink + (b->key_tiles - b->sink_tiles) * b->parts;
  Carve c{static_cast<uint8_t*>(workspace)};
  PackedKeys& pk = b->pk;
  pk.amax = c.take<uint32_t>(planes * 4);
  pk.odd = reinterpret_cast<int*>(pk.amax + planes * 2);
  b->norms = c.take<uint32_t>(planes);
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
  b->score = c.take<float>(planes * b->q.rows);
  b->own = c.take<float4>(planes * b->q.rows);
  b->tile = c.take<float4>(planes * b->q_tiles);
  if (b->parts > 1 || b->parts_sink > 1) b->part = c.take<float>(planes * b->units * 2 * 128 * DP);
  return c.used;
}

template <int DP>
int backward_go(const StreamRows& s, BackwardTc& b, cudaStream_t st) {
  constexpr int CB = DP / 64;
  constexpr int kSmemKv = CB * (32768 + 16384 + 4 * 16384) + 1536 + 256 + 1024, kSmemQ = CB * (2 * 16384 + 5 * 16384) + 256 + 1024;
  static std::atomic<uint64_t> ready_kv{0}, ready_q{0};
  constexpr int kShared = 512 * kRegsSoftmax + 128 * kRegsOther;
  GN_TRY(prepare_kernel(ready_kv, reinterpret_cast<const void*>(stream_tc_dkv_kernel<DP>), kSmemKv, kThreadsB, kShared));
  GN_TRY(prepare_kernel(ready_q, reinterpret_cast<const void*>(stream_tc_dq_kernel<DP>), kSmemQ, kThreadsB, kShared));
  GN_TRY(stream_pack_keys(s, b.pk, b.norms, st));
  GN_CUDA(launch_pdl(stream_query_pack_kernel<CB>, dim3(b.q_tiles, s.Hkv, s.rows), dim3(kThreadsQ), 0, st, b));
  GN_CUDA(launch_pdl(stream_tc_dkv_kernel<DP>, dim3(b.units, s.Hkv, s.rows), dim3(kThreadsB), kSmemKv, st, b));
  GN_CUDA(launch_pdl(stream_tc_dq_kernel<DP>, dim3(b.q_tiles, s.Hkv, s.rows), dim3(kThreadsB), kSmemQ, st, b));
  if (b.parts > 1 || b.parts_sink > 1)
    GN_CUDA(launch_pdl(stream_tc_dkv_sum_kernel<DP>, dim3(ceil_div(s.seq, 1024 / DP), s.Hkv, 2 * s.rows), dim3(256), 0, st, b));
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
