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

// Largest finite magnitude of every plane.  Bound: HBM; 9.7 us for 2 planes of 8704 keys (18 MB, too few CTAs in flight to reach it).
template <int CB, bool PAGED>
__global__ void __launch_bounds__(256) stream_amax_kernel(const __grid_constant__ StreamRows s, PackedKeys pk, int vec) {
  pdl_trigger();
  pdl_wait();
  const int hk = blockIdx.y, r = blockIdx.z >> 1, value = blockIdx.z & 1, half = threadIdx.x >> 4;
  const RowSpan sp = row_span<PAGED>(s, r);
  const int begin = first_needed<PAGED>(s, sp), j0 = blockIdx.x * kPackRows;
  if (j0 >= sp.ctx || (j0 + kPackRows <= begin && j0 >= s.sinks)) return;
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

// Keys and values times a power of two that brings the plane's largest to [2^14, 2^15), as f16 pairs in the layout that the tiles are copied in.
// With whole = 1 a plane is a cluster's (its CTAs take 16 keys in turn), which finds the largest magnitude itself.  Half a warp per row:
// 16-byte loads and whole 128-byte lines of stores.  Bound: HBM, 4 D bytes a row in and out; 25 us for 2 x 128 planes of up to 383 keys
// (37 MB read, 37 written; the meeting of the cluster and two readings in a row are its latency).
template <int CB, bool PAGED>
__global__ void __launch_bounds__(256) stream_pack_kernel(const __grid_constant__ StreamRows s, PackedKeys pk, uint32_t* norms, int vec, int whole) {
  pdl_trigger();
  pdl_wait();
  const int hk = blockIdx.y, r = blockIdx.z >> 1, value = blockIdx.z & 1, half = threadIdx.x >> 4, l16 = threadIdx.x & 15;
  const RowSpan sp = row_span<PAGED>(s, r);
  const int ctas = gridDim.x, step = whole ? 16 * ctas : 16;
  const int begin = first_needed<PAGED>(s, sp), j0 = blockIdx.x * (whole ? 16 : kPackRows);
  const Packed& dst = value ? pk.v : pk.k;
  const int last = min(dst.rows, (sp.ctx + 15) / 16 * 16 + 16);   // zero rows behind the sequence: a tile is copied in 16s
  if (!whole && (j0 >= last || (j0 + kPackRows <= begin && j0 >= s.sinks))) return;   // nothing that anyone sees
  const int64_t plane = (int64_t)r * s.Hkv + hk;
  __shared__ uint32_t found[3];   // of this CTA's rows: largest magnitude, whether one is odd, largest norm
  uint32_t largest;
  if (whole) {
    if (threadIdx.x < 3) found[threadIdx.x] = 0;
    __syncthreads();
    uint32_t top = 0;
#pragma unroll 4
    for (int j = j0 + half; j < sp.ctx; j += step) {
      if (!is_needed<PAGED>(s, sp, begin, j)) continue;
      float x[4 * CB];
      load_key<CB, PAGED>(s, value, vec, r, hk, j, x);
#pragma unroll
      for (int e = 0; e < 4 * CB; ++e) if (finite_bits(x[e])) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    }
    if (top) atomicMax(&found[0], top);
    cluster_meet();
    largest = cluster_largest(&found[0], ctas);
  } else {
    largest = pk.amax[plane * 2 + value];
  }
  uint8_t* base = dst.data + plane * dst.plane_bytes(CB);
  uint8_t* flags = (value ? pk.flags_v : pk.flags_k) + plane * dst.rows;
  float sc, inv;
  plane_scale(largest, sc, inv);
  float top = 0.0f;
  const int end = whole ? last : min(last, j0 + kPackRows);
  // backwards: what was read last is in a cache
#pragma unroll 4
  for (int j16 = j0 + (end - j0 + step - 1) / step * step - step; j16 >= j0; j16 -= step) {
    const int j = j16 + half;
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
    if (!needed && j < sp.ctx) continue;
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
      if (flag) { if (whole) found[1] = 1; else pk.odd[plane * 2 + value] = 1; }
    }
  }
  if (norms && value) {
    top = warp_max(top);
    if ((threadIdx.x & 31) == 0 && top > 0.0f) atomicMax(whole ? &found[2] : norms + plane, __float_as_uint(top));
  }
  if (whole) {
    cluster_meet();
    if (blockIdx.x == 0 && threadIdx.x < 32) {
      const uint32_t odd = cluster_largest(&found[1], ctas), norm = cluster_largest(&found[2], ctas);
      if (threadIdx.x == 0) {
        pk.amax[plane * 2 + value] = largest; pk.odd[plane * 2 + value] = odd;
        if (norms && value) norms[plane] = norm;
      }
    }
    cluster_meet();   // no CTA goes while its words are read
  }
}

// ------------------------------------------------------------------ forward
struct ForwardTc {
  StreamRows s;
  PackedKeys pk;
  gn_view out;
  float* lse;
  int vec_q, vec_out, tiles, splits;
  int planes, listed;   // listed: items are counted over the tiles that exist
  FastDiv by_planes, by_splits, by_Hkv;
  float* part_o; float* part_l;   // splits > 1: [plane][tile][split][128] rows of DP channels, and their log2-sum-exps
};

constexpr int kRowsT = 128;      // query rows of an item = keys of a tile = UMMA M and N
constexpr int kRowsListed = 511;
constexpr int kThreads = 768;    // four softmax warpgroups, one that fetches Q, one with the issuing and the copying warp
constexpr int kRegsSoftmax = 88, kRegsFetch = 80, kRegsOther = 48;   // shares of the launch's 6 x 80 (the fetching one keeps its)

// What a CTA works on next: 128 query rows of a plane against a range of their key tiles.
struct Item {
  int r, hk, tile, split, f0, nf, first, q_begin, j0, n;   // first: position of the row's first new token; n key tiles from j0
  bool inside;                                             // the rows exist (a padded batch's padding does)
  int64_t plane;
  KeyRuns runs;
  __device__ __forceinline__ int rows16(int j) const { return min(kRowsT, (runs.total - (j0 + j) * kRowsT + 15) & ~15); }   // keys of tile j, in 16s
};
// `before`: of a paged call with few enough rows, how many tiles of new tokens stand before each row's (shared memory).  Its items are
// counted over these, so that every CTA gets as many that exist.  (Two parts of chunks of 512, 0, 180 and 332 tokens, 8 x 8704 keys: the 128
// items that exist went to 94 of 148 CTAs when the 256 that could exist were dealt out.)
template <bool PAGED>
__device__ __forceinline__ Item get_item(const ForwardTc& p, const int* before, int w) {
  const StreamRows& s = p.s;
  Item it;
  if (PAGED && p.listed) {
    const int c = p.by_splits.of(w), t = p.by_Hkv.of(c);
    int low = 0, high = s.rows - 1;   // the last row with before[row] <= t
    while (low < high) {
      const int mid = (low + high + 1) >> 1;
      if (before[mid] <= t) low = mid; else high = mid - 1;
    }
    it.split = w - c * p.splits; it.hk = c - t * s.Hkv; it.r = low; it.tile = t - before[low];
    it.plane = (int64_t)low * s.Hkv + it.hk;
  } else {
    // the last tiles first: under a causal mask they are the longest.  Planes are turned by one from level to level, or a number of them
    // that divides the grid's would leave each to the same few CTAs
    const int level = p.by_planes.of(w), last = p.by_splits.of(level);
    int plane = w - level * p.planes + level - p.by_planes.of(level) * p.planes;
    if (plane >= p.planes) plane -= p.planes;
    it.plane = plane;
    it.split = level - last * p.splits; it.tile = p.tiles - 1 - last;
    it.r = p.by_Hkv.of(plane); it.hk = plane - it.r * s.Hkv;
  }
  const RowSpan sp = row_span<PAGED>(s, it.r);
  it.f0 = it.tile * kRowsT; it.nf = sp.q_len * s.G; it.first = sp.ctx - sp.q_len; it.q_begin = sp.q_begin;
  it.inside = it.f0 < (PAGED ? it.nf : s.seq * s.G);
  it.runs = KeyRuns{0, 0, 0};
  if (it.f0 < it.nf) it.runs = key_runs(s, it.first + s.by_G.of(it.f0), it.first + s.by_G.of(min(it.f0 + kRowsT - 1, it.nf - 1)));
  const int all = (it.runs.total + kRowsT - 1) / kRowsT, per = p.by_splits.of(all + p.splits - 1);
  it.j0 = it.split * per; it.n = max(0, min(all, it.j0 + per) - it.j0);
  return it;
}

// A persistent CTA per SM walks the items; no role waits for an item to end before it begins the next:
//   warps 0-15  four threads per query row, 32 keys of a tile and a quarter of the channels each: read S from tensor memory, take the
//               running maximum, and write 2^15 p as f16 pairs over the scores they came from: P is the A operand of O = P V
//               straight from tensor memory.  Each tile's O starts from zero and is added to float32 registers one tile later, where the
//               rescaling by the grown maximum costs nothing extra: sums over many keys are rounded, not cut off.  An item's
//               result is stored while the next one's Q is fetched and its first products run (behind the next item's first weights, where it
//               was before, it held up everything: 31 400 cycles an item of five tiles);
//   warps 16-19 fetch the next item's Q rows (raw float32), scale, split and leave them in tensor memory (A operand of S = Q K^T);
//   warps 20, 22  issue the instructions, 24 of 128 x 128 x 16 for a tile's S and 24 for its O: each a queue of its own, so that the
//               waits of one pass while the other's instructions run;
//   warp 21     copies K and V tiles (bulk copies of packed rows) through a ring of tile buffers.
// Tensor memory: two score / weight buffers of 128 columns, O 128, Q hi and lo 128.  Code is kept short: warps that run through
// long unrolled code once a tile wait for instructions most of the time.  Sixteen warps, because eight took 3360 cycles a tile
// (read 530, meet 250, weights 1650, O 850) against the 48 instructions of 64 cycles of the tensor pipe, which is the bound of a tile.  Every wait is
// bounded; a kernel whose wait ran out writes NaN.
// 4 x 8192 tokens, 8 heads on one, window 512 and 64 sinks: 253 us, tensor pipe busy 46 %; a tile takes about 3400 cycles, and between two
// items (O to memory in 6700, the next rows' bounds 2000) there are about three tiles' time.  Chunks over 8704 keys: 55 %.
template <int DP, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1) stream_tc_forward_kernel(const __grid_constant__ ForwardTc p) {
  constexpr int CB = DP / 64, QC = DP / 4, RING = DP == 64 ? 6 : 3;
  constexpr uint32_t TILE = CB * 32768u, BARS = RING * TILE, ROWC = BARS + 256, XCH = ROWC + 2048, STASH = XCH + 6144, BEFORE = STASH + 16384;
  constexpr uint32_t COL_O = 256, COL_Q = 384;
  extern __shared__ uint8_t smem_raw[];
  const StreamRows& s = p.s;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + BARS;
  auto full = [&](int i) { return bars + 8u * i; };
  auto empty = [&](int i) { return bars + 48u + 8u * i; };
  auto s_full = [&](int i) { return bars + 96u + 8u * i; };
  auto p_full = [&](int i) { return bars + 112u + 8u * i; };
  const uint32_t o_full = bars + 128, o_empty = bars + 136, q_free = bars + 152, tmem_slot = bars + 160;
  auto s_free = [&](int i) { return bars + 168u + 8u * i; };
  // Items' Q by turns on four barriers: with items of one key tile the fetcher gets two items ahead of a softmax thread that still stores
  // an earlier result, and a barrier that is two phases on looks like one that has not moved
  auto q_ready = [&](uint32_t item) { return bars + 184u + 8u * (item & 3); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < RING; ++i) { mbar_init(full(i), 1); mbar_init(empty(i), 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(s_full(i), 1); mbar_init(p_full(i), 512); mbar_init(s_free(i), 1); }
    mbar_init(o_full, 1); mbar_init(o_empty, 512); mbar_init(q_free, 1);
    for (int i = 0; i < 4; ++i) mbar_init(q_ready(i), 128);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 20) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  pdl_trigger();
  int* before = reinterpret_cast<int*>(gen + BEFORE);
  if (PAGED && p.listed) {
    for (int r = threadIdx.x; r < s.rows; r += kThreads) before[r] = (row_span<PAGED>(s, r).q_len * s.G + kRowsT - 1) / kRowsT;
    __syncthreads();
    if (warp == 0) {
      int sum = 0;
      for (int r = lane; r - lane < s.rows; r += 32) {
        const int x = r < s.rows ? before[r] : 0;
        int y = x;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) { const int z = __shfl_up_sync(0xffffffffu, y, d); if (lane >= d) y += z; }
        if (r < s.rows) before[r] = sum + y - x;
        sum += __shfl_sync(0xffffffffu, y, 31);
      }
      if (lane == 0) before[s.rows] = sum;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(gen + BARS + 160);
  const int items = PAGED && p.listed ? before[s.rows] * s.Hkv * p.splits : p.planes * p.tiles * p.splits;

  if (warp >= 20) {
    regs_dec<kRegsOther>();
    if (warp == 21 && lane == 0) {
      // ------------------------------------------------------------- copies: K_0, K_1, V_0, K_2, V_1, ... as they are used
      bool ok = true;
      int slot = 0; uint32_t turn = 0;
      pdl_wait();   // for the packed planes; the fetching warps wait later, for they read the caller's queries first
      for (int w = blockIdx.x; w < items && ok; w += gridDim.x) {
        const Item it = get_item<PAGED>(p, before, w);
        for (int m = 0; m < 2 * it.n && ok; ++m) {
          const bool value = m == 2 * it.n - 1 || (m > 0 && (m & 1) == 0);
          const int j = value ? (m == 2 * it.n - 1 ? it.n - 1 : (m >> 1) - 1) : (m + 1) >> 1;
          if (turn > 0) ok = hold(empty(slot), (turn - 1) & 1);
          if (!ok) break;
          const Packed& src = value ? p.pk.v : p.pk.k;
          const int c0 = (it.j0 + j) * kRowsT, rows = it.rows16(j), na = min(max(it.runs.a_len - c0, 0), rows), nb = rows - na;
          const uint8_t* from = src.data + it.plane * src.plane_bytes(CB) + (int64_t)c0 * 128;
          uint32_t dst = base + slot * TILE;
          mbar_expect_tx(full(slot), (uint32_t)CB * 2u * rows * 128u);
#pragma unroll 1
          for (int b = 0; b < CB * 2; ++b) {
            if (na) bulk_load(dst, from, na * 128, full(slot));
            if (nb) bulk_load(dst + na * 128, from + (int64_t)(na + it.runs.shift) * 128, nb * 128, full(slot));
            dst += 16384; from += (int64_t)src.rows * 128;
          }
          if (++slot == RING) { slot = 0; ++turn; }
        }
      }
      if (!ok)   // copies in flight land before the CTA goes
        for (int i = 0; i < RING; ++i) { hold(full(i), 0); hold(full(i), 1); }
    }
    if (warp == 20 || warp == 22) {
      // ------------------------------------------------------------- instructions
      const uint32_t el = elect_lane();
      const bool products = warp == 22;   // O = P V; the other warp S = Q K^T
      bool ok = true;
      uint32_t tile = 0, count = 0, ring = 0;   // tiles, items and copies so far
      Item it = get_item<PAGED>(p, before, blockIdx.x);   // may not exist
      for (int w = blockIdx.x; w < items && ok;) {
        const int n = it.n, last16 = n > 0 ? it.rows16(n - 1) : 0;
        w += gridDim.x;
        if (w < items) it = get_item<PAGED>(p, before, w);   // the next item's geometry is on its way while this one runs
        if (n == 0) continue;
        if (!products) ok = hold_warp(q_ready(count), (count >> 2) & 1);
        for (int j = 0; j < n && ok; ++j, ++tile) {
          const int rows = j + 1 == n ? last16 : kRowsT, b = tile & 1;
          const uint32_t m = ring + (products ? min(2 * j + 2, 2 * n - 1) : j == 0 ? 0 : 2 * j - 1), slot = m % RING;
          // A copy is waited for only when what stood in its slot before is known to have landed: it may have been the other warp's (K_j before V_j), which
          // this one does not wait for, and as long as it is on its way the parity of the phase before it lets a wait for this copy pass.  Scores of
          // tile j mean that K_j landed.  Before K_j stood a tile of keys, or V of three tiles back or more, whose products freed the buffer that the last
          // scores were issued into; only at an item's start it may be V of two tiles back, which the free buffer of these scores means.
          if (products) {
            ok = hold_warp(s_full(b), (tile >> 1) & 1) && hold_warp(full(slot), (m / RING) & 1) && hold_warp(p_full(b), (tile >> 1) & 1) &&
                 (tile == 0 || hold_warp(o_empty, (tile - 1) & 1));
          } else {
            auto free_scores = [&]() { return tile < 2 || hold_warp(s_free(b), ((tile >> 1) - 1) & 1); };
            ok = (j > 0 || free_scores()) && hold_warp(full(slot), (m / RING) & 1) && (j == 0 || free_scores());
          }
          if (!ok) break;
          tc_fence_after();
          if (products) {
            const uint32_t id = instr_desc_f16(128, DP, 1), wt = tmem + b * 128;
            const uint64_t v = smem_desc_mn(base + slot * TILE, 32768);
            const int slices = rows >> 4;
#pragma unroll 1
            for (int ks = 0; ks < slices; ++ks) {
              const uint32_t at = wt + (ks >> 1) * 32 + (ks & 1) * 8;
              umma_f16_ts(el, tmem + COL_O, at + 16, v + ks * 128, id, ks > 0);
              umma_f16_ts(el, tmem + COL_O, at, v + ks * 128 + 1024, id, 1);
            }
#pragma unroll 1
            for (int ks = 0; ks < slices; ++ks) umma_f16_ts(el, tmem + COL_O, wt + (ks >> 1) * 32 + (ks & 1) * 8, v + ks * 128, id, 1);
            commit_by(el, o_full);
            commit_by(el, s_free(b));
          } else {
            const uint32_t d = tmem + b * 128, id = instr_desc_f16(128, rows, 0);
            const uint64_t k = smem_desc_sw128(base + slot * TILE);
#pragma unroll 2
            for (int ks = 0; ks < CB * 4; ++ks) {
              const uint32_t at = tmem + COL_Q + (ks >> 1) * 32 + (ks & 1) * 8, in = (ks >> 2) * 2048 + (ks & 3) * 2;
              umma_f16_ts(el, d, at + 16, k + in, id, ks > 0);
              umma_f16_ts(el, d, at, k + in + 1024, id, 1);
            }
#pragma unroll 2
            for (int ks = 0; ks < CB * 4; ++ks) umma_f16_ts(el, d, tmem + COL_Q + (ks >> 1) * 32 + (ks & 1) * 8, k + (ks >> 2) * 2048 + (ks & 3) * 2, id, 1);
            commit_by(el, s_full(b));
            if (j + 1 == n) commit_by(el, q_free);   // the item's last scores
          }
          commit_by(el, empty(slot));
        }
        ++count;
        ring += 2 * n;
      }
      // What the instructions still signal, nobody else waits for: it has arrived before this CTA's shared memory goes to another
      if (products) {
        for (uint32_t t = tile < 2 ? 0 : tile - 2; t < tile && ok; ++t) ok = hold_warp(s_free(t & 1), (t >> 1) & 1);
      } else {
        for (uint32_t m = ring < RING ? 0 : ring - RING; m < ring && ok; ++m) ok = hold_warp(empty(m % RING), (m / RING) & 1);
        if (count > 0 && ok) hold_warp(q_free, (count - 1) & 1);
      }
    }
  } else if (warp >= 16) {
    // --------------------------------------------------------------- Q rows to tensor memory
    const int row = (warp & 3) * 32 + lane;
    const uint32_t q_addr = tmem + COL_Q + ((uint32_t)((warp & 3) * 32) << 16);
    float* rowc = reinterpret_cast<float*>(gen + ROWC);
    uint4* stash = reinterpret_cast<uint4*>(gen + STASH);   // each thread its own column
    bool ok = true;
    uint32_t count = 0;
    for (int w = blockIdx.x; w < items; w += gridDim.x) {
      const Item it = get_item<PAGED>(p, before, w);
      if (it.n == 0) continue;
      const int f = it.f0 + row, t = s.by_G.of(f), g = f - t * s.G;
      const bool live = f < it.nf;
      const float* src = live ? s.q.data + token_offset<PAGED>(s.q, it.r, it.hk * s.G + g, it.q_begin + t) : nullptr;
      // 32 channels of the row from ch on, all loads in flight at once (a row that is not there reads the tensor's first)
      auto load = [&](int ch, float (&x)[32]) {
        if (p.vec_q) {
          const float* row = src ? src : s.q.data;
          float4 v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = __ldg(reinterpret_cast<const float4*>(row + min(ch + 4 * k, s.D - 4)));
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const bool in = src && ch + 4 * k < s.D;
            x[4 * k] = in ? v[k].x : 0.0f; x[4 * k + 1] = in ? v[k].y : 0.0f; x[4 * k + 2] = in ? v[k].z : 0.0f; x[4 * k + 3] = in ? v[k].w : 0.0f;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) x[e] = src && ch + e < s.D ? src[ch + e] : 0.0f;
        }
      };
      // One pass: the scale comes from the first 32 channels, with 2^6 to spare for the others; a warp with a row that needs
      // more (or whose first channels are zeros) goes over its rows again.  While the last item's scores still read Q, the first
      // 32 channels wait in shared memory, the next in registers, and the others are on their way to L2.  One copy of the code serves all of
      // them: unrolled it was 7400 cycles from the last scores to Q, most of them spent waiting for instructions, its own and the other warps'.
      uint32_t top = 0;
      float sq = 1.0f, iq = 1.0f;
      if (p.vec_q && src)
#pragma unroll
        for (int ch = 64; ch < DP; ch += 32) if (ch < s.D) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + ch));
#pragma unroll 1
      for (int pass = 0; pass < 2; ++pass) {
#pragma unroll 1
        for (int h = 0; h < DP / 32; ++h) {
          float x[32];
          uint32_t y[32];
          load(h * 32, x);
          if (pass == 0) {
#pragma unroll
            for (int e = 0; e < 32; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);   // a row that is not finite has no result whatever its scale
            if (h == 0) { plane_scale(top, sq, iq); sq *= 0x1p-6f; iq *= 0x1p6f; }
          }
          const float by = s.scale < 0.0f ? -sq : sq;   // a negative scale goes into Q, so that larger products are larger scores
#pragma unroll
          for (int e = 0; e < 32; e += 2) split_f16(x[e] * by, x[e + 1] * by, y[e >> 1], y[16 + (e >> 1)]);
          if (h == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) stash[e * 128 + row] = make_uint4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
          } else {
            if (h == 1 && pass == 0 && count > 0) { ok = ok && hold_warp(q_free, (count - 1) & 1); tc_fence_after(); }
            __syncwarp();
            tmem_st32(q_addr + h * 32, y);
          }
        }
        uint32_t y[32];
#pragma unroll
        for (int e = 0; e < 8; ++e) { const uint4 v = stash[e * 128 + row]; y[4 * e] = v.x; y[4 * e + 1] = v.y; y[4 * e + 2] = v.z; y[4 * e + 3] = v.w; }
        __syncwarp();
        tmem_st32(q_addr, y);
        const float largest = __uint_as_float(top) * sq;
        const bool again = top != 0 && !(largest >= 0x1p7f && largest < 0x1p15f);
        if (pass == 1 || !__any_sync(0xffffffffu, again)) break;
        if (again) plane_scale(top, sq, iq);
      }
      float sk, ik;
      if (count == 0) pdl_wait();
      plane_scale(p.pk.amax[it.plane * 2], sk, ik);
      const float c = fmaxf(fabsf(s.scale) * kLog2e * iq * ik, 1e-30f);   // a vanishing scale stays a positive number
      rowc[(count & 3) * 128 + row] = c;   // four, as the barriers
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(q_ready(count));
      ++count;
    }
  } else {
    // --------------------------------------------------------------- softmax threads
    regs_inc<kRegsSoftmax>();
    pdl_wait();
    const int quarter = warp & 3, part = warp >> 2, row = quarter * 32 + lane;   // a warp reaches the tensor-memory lanes [32 * (warp % 4), +32)
    const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
    float* xch = reinterpret_cast<float*>(gen + XCH);   // [2][4 parts][128] maxima, then [4 parts][128] sums
    const float* rowc = reinterpret_cast<const float*>(gen + ROWC);
    auto meet = [&]() { __syncwarp(); asm volatile("bar.sync %0, 128;" ::"r"(1 + quarter) : "memory"); };   // the four warps of these 32 rows
    bool ok = true;
    uint32_t tiles = 0, count = 0;
    float m = -INFINITY, l = 0.0f, alpha = 0.0f;   // l of a poisoned row is not a number
    float o[QC];
    // where the row's result goes: out from this thread's channels on (null: nowhere), lse null in all but one of the row's threads
    struct Target { float* out; float* lse; float iv; } to{nullptr, nullptr, 1.0f};

    auto gather = [&]() {   // O of the last tile, against the maximum that it used
      ok = ok && hold_warp(o_full, (tiles - 1) & 1);
      tc_fence_after();
      uint32_t y[QC];
      if constexpr (QC == 32) tmem_ld32(lane_addr + COL_O + part * QC, y);
      else tmem_ld16(lane_addr + COL_O + part * QC, y);
      tmem_ld_wait();
      tc_fence_before();
      mbar_arrive(o_empty);
#pragma unroll
      for (int e = 0; e < QC; ++e) o[e] = fmaf(o[e], alpha, __uint_as_float(y[e]));
    };
    auto store = [&]() {
      float* mine = xch + 1024;
      mine[part * 128 + row] = ok ? l : NAN;
      meet();
      const float sum = (mine[row] + mine[128 + row]) + (mine[256 + row] + mine[384 + row]);
      const float z = sum == 0.0f ? 0.0f : to.iv / sum, L = sum == 0.0f ? -INFINITY : m - kWeightShift + log2f(sum);
      meet();
      if (to.lse) *to.lse = p.splits > 1 ? L : L * kLn2;
      const int left = (p.splits > 1 ? DP : s.D) - part * QC;
      if (p.vec_out) {
        constexpr int N = QC / 4;
#pragma unroll
        for (int e = 0; e < QC; ++e) o[e] *= z;
        transpose_blocks<N>(o);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          float* dst = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to.out), (lane & ~(N - 1)) + k));
          const int e = (lane & (N - 1)) * 4;
          if (dst && e < left) *reinterpret_cast<float4*>(dst + e) = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
        }
      } else if (to.out) {
#pragma unroll
        for (int e = 0; e < QC; ++e) if (e < left) to.out[e] = o[e] * z;
      }
    };

    for (int w = blockIdx.x; w < items; w += gridDim.x) {
      const Item it = get_item<PAGED>(p, before, w);
      if (!it.inside) continue;
      const int f = it.f0 + row, t = s.by_G.of(f), g = f - t * s.G, token = it.q_begin + t, pos = it.first + t;
      const bool live = f < it.nf;
      to = Target{nullptr, nullptr, 1.0f};
      if (p.splits > 1) {
        const int64_t at = ((it.plane * p.tiles + it.tile) * p.splits + it.split) * kRowsT + row;
        to.out = p.part_o + at * DP + part * QC;
        to.lse = p.part_l + at;
      } else {
        to.out = f < (PAGED ? it.nf : s.seq * s.G) ? p.out.data + token_offset<PAGED>(p.out, it.r, it.hk * s.G + g, token) + part * QC : nullptr;
        to.lse = p.lse + stat_offset<PAGED>(s, it.r, it.hk * s.G + g, token);
      }
      if (!to.out || part != 0) to.lse = nullptr;
      if (it.n == 0) {   // rows that see nothing: padding, or tokens before the cache
        if (to.lse) *to.lse = -INFINITY;
        if (to.out) for (int e = 0; e < min(QC, p.splits > 1 ? QC : s.D - part * QC); ++e) to.out[e] = 0.0f;
        continue;
      }
      float sv;
      plane_scale(p.pk.amax[it.plane * 2 + 1], sv, to.iv);
      // what the row sees, in virtual keys: [0, s_end) and [lo, hi]
      const int s_end = live ? max(0, min(s.sinks, pos + 1)) : 0;
      const int lo_key = live ? (s.window < 0 ? 0 : max(0, pos - s.window)) - it.runs.shift : 0, hi_key = live ? pos - it.runs.shift : -1;
      const bool odd_plane = (p.pk.odd[it.plane * 2] | p.pk.odd[it.plane * 2 + 1]) != 0;
      ok = ok && hold_warp(q_ready(count), (count >> 2) & 1);
      const float c = rowc[(count & 3) * 128 + row];
      ++count;
      m = -INFINITY; l = 0.0f;
#pragma unroll
      for (int e = 0; e < QC; ++e) o[e] = 0.0f;
#pragma unroll 1
      for (int j = 0; j < it.n; ++j) {
        const uint32_t buf = lane_addr + (tiles & 1) * 128 + part * 32;
        const int c0 = (it.j0 + j) * kRowsT + part * 32;
        uint32_t see = (uint32_t)(bits_below(s_end - c0) | (bits_below(hi_key + 1 - c0) & ~bits_below(lo_key - c0)));
        if (odd_plane) {
#pragma unroll 1
          for (int e = 0; e < 32; ++e)
            if ((see >> e) & 1u) {
              const int key = c0 + e < it.runs.a_len ? c0 + e : c0 + e + it.runs.shift;
              const uint8_t flag = p.pk.flags_k[it.plane * p.pk.k.rows + key] | p.pk.flags_v[it.plane * p.pk.v.rows + key];
              if (flag & kAbsent) see &= ~(1u << e);
              else if (flag & kOdd) l = NAN;
            }
        }
        ok = ok && hold_warp(s_full(tiles & 1), (tiles >> 1) & 1);
        tc_fence_after();
        uint32_t y[32];
        tmem_ld32(buf, y);
        tmem_ld_wait();
        if (!__all_sync(0xffffffffu, see == ~0u)) {
#pragma unroll
          for (int e = 0; e < 32; ++e) if (!((see >> e) & 1u)) y[e] = 0xff800000u;
        }
        float top = __uint_as_float(y[0]);
#pragma unroll
        for (int e = 1; e < 32; ++e) top = fmaxf(top, __uint_as_float(y[e]));
        float* mine = xch + (tiles & 1) * 512 + row;
        mine[part * 128] = top;
        meet();
        top = fmaxf(fmaxf(mine[0], mine[128]), fmaxf(mine[256], mine[384]));
        const float m_new = fmaxf(m, top == -INFINITY ? -INFINITY : top * c), m_use = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha_here = exp2_fast(m - m_use), off = kWeightShift - m_use;
        m = m_new;
        float sum = 0.0f;
        uint32_t z[32];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float a = exp2_fast(fmaf(__uint_as_float(y[e]), c, off)), b = exp2_fast(fmaf(__uint_as_float(y[e + 1]), c, off));
          sum += a + b;
          split_f16(a, b, z[e >> 1], z[16 + (e >> 1)]);
        }
        tmem_st32(buf, z);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(p_full(tiles & 1));
        l = fmaf(l, alpha_here, sum);
        if (j > 0) gather();
        alpha = alpha_here;
        ++tiles;
      }
      gather();
      store();
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 20) tmem_dealloc(tmem, 512);
}

// Joins the parts of a row's keys by their log-sum-exps: a warp per query row.  Bound: reading them; 8.5 us for 8192 rows in two parts.
template <int DP, bool PAGED>
__global__ void __launch_bounds__(256) stream_tc_combine_kernel(const __grid_constant__ ForwardTc p) {
  pdl_trigger();
  pdl_wait();
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
  int64_t seen = pl.max_k, ctas = std::max<int64_t>(1, pl.planes * pl.tiles);
  if (s.window >= 0) seen = std::min<int64_t>(seen, (int64_t)s.window + s.sinks + kRowsT / s.G + 1);
  if (s.paged()) ctas = std::min(ctas, s.Hkv * (ceil_div((int64_t)s.tokens * s.G, kRowsT) + (int64_t)s.rows));   // no more tiles exist
  // Parts of a tile's keys: the fewest rounds of 148 items, counted in key tiles with 3.5 for an item's start and end, 2 for the pass that
  // joins the parts and the partial results' way to memory and back (0.012 a part); no part below four tiles.  In one part and in two:
  // 12 planes x 49 tiles of 2049 keys 134 and 173 us, 1 x 128 of 2048 58 and 65, 2 x 32 of 1024 40 and 41, 16 x up to 4 of 4000 125 and 106.
  const double keys = (double)seen / kRowsT;
  double best = 0.0;
  pl.splits = 1;
  for (int parts = 1; parts <= 64 && (parts == 1 || keys / parts >= 4.0); ++parts) {
    const double cost = (double)((ctas * parts + 147) / 148) * (keys / parts + 3.5) + (parts > 1 ? 2.0 + 0.012 * (double)(ctas * parts) : 0.0);
    if (parts == 1 || cost < best) { best = cost; pl.splits = parts; }
  }
  return pl;
}
int64_t carve_forward(const StreamRows& s, const Plan& pl, void* workspace, ForwardTc* f) {
  Carve c{static_cast<uint8_t*>(workspace)};
  const int rows = packed_rows(pl.max_k);
  PackedKeys& pk = f->pk;
  pk.amax = c.take<uint32_t>(pl.planes * 4);   // amax and odd in one piece: cleared together
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
  const int vec = vec_keys(s), keys = pk.k.rows, ctas = pack_cluster(keys, 2ll * s.rows * s.Hkv);
  if (ctas) {
    GN_CUDA(launch_cluster(stream_pack_kernel<CB, PAGED>, dim3(ctas, s.Hkv, 2 * s.rows), 256, ctas, st, s, pk, norms, vec, 1));
  } else {
    GN_CUDA(cudaMemsetAsync(pk.amax, 0, (int64_t)s.rows * s.Hkv * 4 * sizeof(uint32_t), st));   // amax and odd
    if (norms) GN_CUDA(cudaMemsetAsync(norms, 0, (int64_t)s.rows * s.Hkv * sizeof(uint32_t), st));
    stream_amax_kernel<CB, PAGED><<<dim3(ceil_div(keys, kPackRows), s.Hkv, 2 * s.rows), 256, 0, st>>>(s, pk, vec);
    GN_LAUNCH_CHECK();
    GN_CUDA(launch_pdl(stream_pack_kernel<CB, PAGED>, dim3(ceil_div(keys, kPackRows), s.Hkv, 2 * s.rows), dim3(256), 0, st, s, pk, norms, vec, 0));
  }
  return GN_OK;
}

template <int DP, bool PAGED>
int forward_go(const StreamRows& s, const Plan& pl, ForwardTc& f, cudaStream_t st) {
  constexpr int kSmem = 6 * 32768 + 256 + 2048 + 6144 + 16384 + (kRowsListed + 1) * 4 + 1024;
  GN_TRY(stream_pack_keys(s, f.pk, nullptr, st));
  static std::atomic<uint64_t> ready{0};
  GN_TRY(prepare_kernel(ready, reinterpret_cast<const void*>(stream_tc_forward_kernel<DP, PAGED>), kSmem, kThreads, 512 * kRegsSoftmax + 128 * (kRegsFetch + kRegsOther)));
  const int64_t items = pl.planes * pl.tiles * pl.splits;
  GN_REQUIRE(items < (1ll << 31) - 1024, "attention: %lld tiles of query rows", (long long)items);
  GN_CUDA(launch_pdl(stream_tc_forward_kernel<DP, PAGED>, dim3((unsigned)std::min<int64_t>(items, num_sms())), dim3(kThreads), kSmem, st, f));
  if (pl.splits > 1) GN_CUDA(launch_pdl(stream_tc_combine_kernel<DP, PAGED>, dim3(ceil_div(pl.max_q * s.G, 8), s.Hkv, s.rows), dim3(256), 0, st, f));
  return GN_OK;
}

}  // namespace

int prepare_kernel(std::atomic<uint64_t>& ready, const void* kernel, int smem, int threads, int shared_out) {
  int device = 0;
  GN_CUDA(cudaGetDevice(&device));
  const uint64_t bit = 1ull << (device & 63);
  if (device < 64 && (ready.load(std::memory_order_acquire) & bit)) return GN_OK;
  cudaFuncAttributes a{};
  GN_CUDA(cudaFuncGetAttributes(&a, kernel));
  if (a.numRegs * threads < shared_out) {
    set_error("streaming attention: built with %d registers a thread, too few for the kernel's split", a.numRegs);
    return GN_ERR_UNSUPPORTED;
  }
  GN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (device < 64) ready.fetch_or(bit, std::memory_order_release);   // only now: a call that failed leaves the next one to try again
  return GN_OK;
}

int stream_pack_keys(const StreamRows& s, const PackedKeys& pk, uint32_t* norms, cudaStream_t st) {
  if (s.D <= 64) return s.paged() ? pack_go<1, true>(s, pk, norms, st) : pack_go<1, false>(s, pk, norms, st);
  return s.paged() ? pack_go<2, true>(s, pk, norms, st) : pack_go<2, false>(s, pk, norms, st);
}

int64_t stream_tc_forward_bytes(const StreamRows& s) {
  ForwardTc f{};
  return carve_forward(s, plan_forward(s), nullptr, &f);
}
int stream_tc_forward(const StreamRows& s, const gn_view& out, float* lse, void* workspace, cudaStream_t st, PackedKeys* packed) {
  const Plan pl = plan_forward(s);
  ForwardTc f{};
  f.s = s; f.out = out; f.lse = lse; f.tiles = pl.tiles; f.splits = pl.splits; f.planes = (int)pl.planes;
  f.listed = s.paged() && s.rows <= kRowsListed;
  f.by_planes = FastDiv(pl.planes); f.by_splits = FastDiv(pl.splits); f.by_Hkv = FastDiv(s.Hkv);
  carve_forward(s, pl, workspace, &f);
  if (packed) *packed = f.pk;
  f.vec_q = vec_view(s.q, s.D); f.vec_out = pl.splits > 1 || vec_view(out, s.D);
  if (pl.DP == 64) return s.paged() ? forward_go<64, true>(s, pl, f, st) : forward_go<64, false>(s, pl, f, st);
  return s.paged() ? forward_go<128, true>(s, pl, f, st) : forward_go<128, false>(s, pl, f, st);
}

}  // namespace gn
