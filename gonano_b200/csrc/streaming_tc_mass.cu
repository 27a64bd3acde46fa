// The attention weight that a chunk's queries give every cached key (gn_attention_paged with mass_out), on the tensor cores.
//
// mass_j = sum over queries i and heads of the group of exp(s_ij - lse_i): the scores once more, now that the log-sum-exps are known,
// with the keys as the rows of the product: S^T = K Q^T, so that a thread sums along a row and no sum crosses lanes.  Queries are
// packed with a scale of their own each (one pass over them); keys as the forward pass packed them.
// Bound: 24 instructions of 128 x 128 x 16 (1536 cycles) a tile of 128 keys x 128 query rows.  24 chunks of up to 64 tokens, 6 heads on 2, over up
// to 2000 keys: 8 us for the queries and 20 us for the sums, launch and start-up of one or two tiles a CTA.
#include "streaming_tc.cuh"

namespace gn {

namespace {

struct MassTc {
  StreamRows s;
  PackedKeys pk;
  Packed q;
  float* factor; float* off;   // [plane][q.rows]: from products to log2 units, minus the log-sum-exp
  const float* lse;
  const float* mass; float* mass_out;
  int vec_q;
};

// Half a warp per query row f = token * group + head.
template <int CB>
__global__ void __launch_bounds__(256) stream_mass_pack_kernel(const __grid_constant__ MassTc p) {
  pdl_trigger();
  pdl_wait();
  const StreamRows& s = p.s;
  const int hk = blockIdx.y, r = blockIdx.z, half = threadIdx.x >> 4, l16 = threadIdx.x & 15;
  const RowSpan sp = row_span<true>(s, r);
  const int nf = sp.q_len * s.G, last = nf == 0 ? 0 : min(p.q.rows, (nf + 15) / 16 * 16 + 16);
  const int64_t plane = (int64_t)r * s.Hkv + hk;
  float sk, ik;
  plane_scale(p.pk.amax[plane * 2], sk, ik);
  uint8_t* base = p.q.data + plane * p.q.plane_bytes(CB);
#pragma unroll 1
  for (int f = blockIdx.x * 64 + half; f < min(last, (int)blockIdx.x * 64 + 64); f += 16) {   // whole 16s: the warp's halves go together
    const int t = s.by_G.of(f), h = hk * s.G + f - t * s.G;
    float x[4 * CB];
    const float* src = s.q.data + (f < nf ? token_offset<true>(s.q, r, h, sp.q_begin + t) : 0);
    uint32_t top = 0;
    bool odd = false;
#pragma unroll
    for (int b = 0; b < CB; ++b) {
      const int c = b * 64 + l16 * 4;
      if (p.vec_q) {
        float4 v = make_float4(0, 0, 0, 0);
        if (f < nf && c < s.D) v = *reinterpret_cast<const float4*>(src + c);
        x[4 * b] = v.x; x[4 * b + 1] = v.y; x[4 * b + 2] = v.z; x[4 * b + 3] = v.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * b + e] = f < nf && c + e < s.D ? src[c + e] : 0.0f;
      }
    }
#pragma unroll
    for (int e = 0; e < 4 * CB; ++e) {
      if (finite_bits(x[e])) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
      else { odd = true; x[e] = 0.0f; }
    }
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    odd = ((__ballot_sync(0xffffffffu, odd) >> (threadIdx.x & 16)) & 0xffffu) != 0;
    float sq, iq;
    plane_scale(top, sq, iq);
#pragma unroll
    for (int b = 0; b < CB; ++b) {
      uint2 hi, lo;
      split_f16(x[4 * b] * sq, x[4 * b + 1] * sq, hi.x, lo.x);
      split_f16(x[4 * b + 2] * sq, x[4 * b + 3] * sq, hi.y, lo.y);
      uint8_t* at = base + ((int64_t)b * 2 * p.q.rows + f) * 128 + ((((l16 >> 1) ^ (f & 7)) << 4) | ((l16 & 1) << 3));
      *reinterpret_cast<uint2*>(at) = hi;
      *reinterpret_cast<uint2*>(at + (int64_t)p.q.rows * 128) = lo;
    }
    if (l16 == 0) {
      p.factor[plane * p.q.rows + f] = s.scale * kLog2e * iq * ik;
      p.off[plane * p.q.rows + f] = f >= nf ? 0.0f : odd ? NAN : -p.lse[stat_offset<true>(s, r, h, sp.q_begin + t)] * kLog2e;
    }
  }
}

constexpr int kThreadsM = 640;   // 16 summing warps (four threads per key), the issuing warp 16, the copying warp 17

template <int DP>
__global__ void __launch_bounds__(kThreadsM, 1) stream_tc_mass_kernel(const __grid_constant__ MassTc p) {
  constexpr int CB = DP / 64;
  constexpr uint32_t TILE = CB * 32768u, OFF_Q = TILE, STATS = 3 * TILE, BARS = STATS + 2048, SUMS = BARS + 128;
  extern __shared__ uint8_t smem_raw[];
  const StreamRows& s = p.s;
  const int hk = blockIdx.y, r = blockIdx.z, k0 = blockIdx.x * 128;
  const RowSpan sp = row_span<true>(s, r);
  if (k0 >= sp.ctx) { pdl_wait(); return; }
  const int first = sp.ctx - sp.q_len, nf = sp.q_len * s.G;
  const int64_t plane = (int64_t)r * s.Hkv + hk;
  // the query rows that see a key of the tile
  const int64_t t_end = (s.window < 0 || k0 < s.sinks) ? sp.q_len : min((int64_t)sp.q_len, (int64_t)k0 + 128 + s.window - first);
  const int f_begin = (max(0, k0 - first) * s.G) & ~7, f_end = (int)max((int64_t)0, t_end) * s.G;
  const int n = f_end > f_begin ? (f_end - f_begin + 127) / 128 : 0;

  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + BARS, k_full = bars, tmem_slot = bars + 80;
  auto q_full = [&](int i) { return bars + 8u + 8u * i; };
  auto q_empty = [&](int i) { return bars + 24u + 8u * i; };
  auto s_full = [&](int i) { return bars + 40u + 8u * i; };
  auto s_empty = [&](int i) { return bars + 56u + 8u * i; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(k_full, 1);
    for (int i = 0; i < 2; ++i) { mbar_init(q_full(i), 1); mbar_init(q_empty(i), 1); mbar_init(s_full(i), 1); mbar_init(s_empty(i), 512); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 16) { tmem_alloc(tmem_slot, 256); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gen + BARS + 80);
  pdl_wait();
  auto rows16 = [&](int i) { return min(128, (f_end - f_begin - i * 128 + 15) & ~15); };

  if (warp == 17) {
    if (lane == 0 && n > 0) {
      const int keys = min(128, (sp.ctx - k0 + 15) & ~15);
      mbar_expect_tx(k_full, (uint32_t)CB * 2u * keys * 128u);
      const uint8_t* kp = p.pk.k.data + plane * p.pk.k.plane_bytes(CB) + (int64_t)k0 * 128;
#pragma unroll 1
      for (int b = 0; b < CB * 2; ++b) bulk_load(base + b * 16384, kp + (int64_t)b * p.pk.k.rows * 128, keys * 128, k_full);
      bool ok = true;
      for (int i = 0; i < n && ok; ++i) {
        // the tile has been multiplied, and its factors read
        if (i >= 2) ok = hold(q_empty(i & 1), ((i >> 1) - 1) & 1) && hold(s_empty(i & 1), ((i >> 1) - 1) & 1);
        if (!ok) break;
        const int rows = rows16(i), f = f_begin + i * 128;
        const uint32_t bar = q_full(i & 1), st = base + STATS + (i & 1) * 1024;
        mbar_expect_tx(bar, (uint32_t)CB * 2u * rows * 128u + 2u * rows * 4u);
        const uint8_t* qp = p.q.data + plane * p.q.plane_bytes(CB) + (int64_t)f * 128;
#pragma unroll 1
        for (int b = 0; b < CB * 2; ++b) bulk_load(base + OFF_Q + (i & 1) * TILE + b * 16384, qp + (int64_t)b * p.q.rows * 128, rows * 128, bar);
        bulk_load(st, p.factor + plane * p.q.rows + f, rows * 4, bar);
        bulk_load(st + 512, p.off + plane * p.q.rows + f, rows * 4, bar);
      }
      if (!ok)   // copies in flight land before the CTA goes
        for (int i = 0; i < 2; ++i) { hold(q_full(i), 0); hold(q_full(i), 1); }
      hold(k_full, 0);
    }
  } else if (warp == 16) {
    if (n > 0) {
      const uint32_t el = elect_lane();
      bool ok = hold_warp(k_full, 0);
      const uint64_t a = smem_desc_sw128(base);
      for (int i = 0; i < n && ok; ++i) {
        ok = hold_warp(q_full(i & 1), (i >> 1) & 1) && (i < 2 || hold_warp(s_empty(i & 1), ((i >> 1) - 1) & 1));
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + (i & 1) * 128, id = instr_desc_f16(128, rows16(i), 0);
        const uint64_t b = smem_desc_sw128(base + OFF_Q + (i & 1) * TILE);
#pragma unroll 2
        for (int ks = 0; ks < CB * 4; ++ks) {
          const uint32_t in = (ks >> 2) * 2048 + (ks & 3) * 2;
          umma_f16(el, d, a + in + 1024, b + in, id, ks > 0);
          umma_f16(el, d, a + in, b + in + 1024, id, 1);
        }
#pragma unroll 2
        for (int ks = 0; ks < CB * 4; ++ks) { const uint32_t in = (ks >> 2) * 2048 + (ks & 3) * 2; umma_f16(el, d, a + in, b + in, id, 1); }
        commit_by(el, s_full(i & 1));
        commit_by(el, q_empty(i & 1));
      }
      for (int i = max(0, n - 2); i < n && ok; ++i) ok = hold_warp(q_empty(i & 1), (i >> 1) & 1);   // nobody else waits for the last ones
    }
  } else if (warp < 16) {
    const int quarter = warp & 3, part = warp >> 2, row = quarter * 32 + lane, key = k0 + row;
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    bool live = key < sp.ctx;
    if (live && n > 0 && p.pk.odd[plane * 2] && (p.pk.flags_k[plane * p.pk.k.rows + key] & kAbsent) &&
        (key < ((s.sinks + 7) & ~7) || s.window < 0 || key >= ((max(0, first - s.window)) & ~7))) live = false;   // no such page: nobody sees it
    const int f_lo = max(0, key - first) * s.G;
    const int f_hi = !live ? 0 : (s.window < 0 || key < s.sinks) ? nf : (int)max((int64_t)0, min((int64_t)nf, ((int64_t)key + s.window + 1 - first) * s.G));
    bool ok = true;
    float sum = 0.0f;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int f0 = f_begin + i * 128 + part * 32;
      const uint32_t see = (uint32_t)(bits_below(f_hi - f0) & ~bits_below(f_lo - f0));
      const float* st = reinterpret_cast<const float*>(gen + STATS + (i & 1) * 1024) + part * 32;
      ok = ok && hold_warp(q_full(i & 1), (i >> 1) & 1) && hold_warp(s_full(i & 1), (i >> 1) & 1);
      __syncwarp();
      tc_fence_after();
      uint32_t y[32];
      tmem_ld32(lane_addr + (i & 1) * 128 + part * 32, y);
      tmem_ld_wait();
      float add = 0.0f;
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float w = exp2_fast(fmaf(__uint_as_float(y[e]), st[e], st[128 + e]));
        add += ((see >> e) & 1u) ? w : 0.0f;
      }
      sum += add;
      tc_fence_before();
      mbar_arrive(s_empty(i & 1));
    }
    float* sums = reinterpret_cast<float*>(gen + SUMS);
    sums[part * 128 + row] = ok ? sum : NAN;
    __syncwarp();
    asm volatile("bar.sync %0, 128;" ::"r"(1 + quarter) : "memory");
    if (part == 0 && key < sp.ctx) {
      const float total = (sums[row] + sums[128 + row]) + (sums[256 + row] + sums[384 + row]);
      const int64_t at = plane * s.width * s.page_size + key;
      p.mass_out[at] = (p.mass && key < first ? p.mass[at] : 0.0f) + total;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 16) tmem_dealloc(tmem, 256);
}

int64_t carve(const StreamRows& s, uint8_t* base, MassTc* m) {
  const int CB = s.D <= 64 ? 1 : 2;
  const int64_t planes = (int64_t)s.rows * s.Hkv;
  Carve c{base};
  m->q.rows = packed_rows((int64_t)s.max_query * s.G);
  m->q.data = c.take<uint8_t>(planes * m->q.plane_bytes(CB));
  m->factor = c.take<float>(planes * m->q.rows);
  m->off = c.take<float>(planes * m->q.rows);
  return c.used;
}

template <int DP>
int go(const MassTc& m, cudaStream_t st) {
  constexpr int kSmem = DP / 64 * 3 * 32768 + 2048 + 128 + 2048 + 1024;
  const StreamRows& s = m.s;
  static std::atomic<uint64_t> ready{0};
  GN_TRY(prepare_kernel(ready, reinterpret_cast<const void*>(stream_tc_mass_kernel<DP>), kSmem, kThreadsM, 0));
  GN_CUDA(launch_pdl(stream_mass_pack_kernel<DP / 64>, dim3(ceil_div(m.q.rows, 64), s.Hkv, s.rows), dim3(256), 0, st, m));
  GN_CUDA(launch_pdl(stream_tc_mass_kernel<DP>, dim3(ceil_div(s.max_context, 128), s.Hkv, s.rows), dim3(kThreadsM), kSmem, st, m));
  return GN_OK;
}

}  // namespace

int64_t stream_tc_mass_bytes(const StreamRows& s) {
  MassTc m{};
  return carve(s, nullptr, &m);
}
int stream_tc_mass(const StreamRows& s, const PackedKeys& pk, const float* lse, const float* mass, float* mass_out, void* workspace, cudaStream_t st) {
  MassTc m{};
  m.s = s; m.pk = pk; m.lse = lse; m.mass = mass; m.mass_out = mass_out; m.vec_q = vec_view(s.q, s.D);
  carve(s, static_cast<uint8_t*>(workspace), &m);
  return s.D <= 64 ? go<64>(m, st) : go<128>(m, st);
}

}  // namespace gn
