// Streaming attention on the tensor cores: operands, tiles and instructions shared by its kernels.
//
// Precision.  kind::f16 multiplies at twice the rate of kind::tf32 with the same 11-bit significand, so a float32 operand x is
// held as two halves of s x, s a power of two: hi = f16(s x), lo = f16(s x - hi).  Together they keep 22 bits, as the tf32 pair
// does, in half the bytes.  What f16 lacks is range, hence s: the largest finite |x| of a plane (a sequence and key head; queries
// and dO have finer scales) lands in [2^14, 2^15), which leaves every x an absolute error of at most 2^-40 of that largest one (f16's smallest step is 2^-24) or
// 2^-22 of x, whichever is more.  A product is hi*lo + lo*hi + hi*hi in float32 (lo*lo is below 2^-22), the small terms first: the tensor core
// cuts each partial sum off instead of rounding it, and a cut of the small terms costs 2^-11 of one of the large ones.
//
// Layout.  A packed plane is [64-channel block][hi, lo][row][64 channels], rows of 128 bytes whose 16-byte chunk c sits at chunk
// c ^ (row % 8): the 128-byte swizzle that tcgen05 reads, laid out by the packing kernel, so that any run of rows from a multiple
// of 8 is one contiguous bulk copy (no tensor maps), and the same rows serve as K-major operand (contraction over channels) and as
// MN-major operand (contraction over rows).
#pragma once
#include <cuda_fp16.h>

#include "streaming.cuh"
#include "tcgen05.cuh"

namespace gn {

// Packed planes of one tensor: `rows` = rows of a plane as stored (a multiple of 16, 16 more than the longest sequence rounded up).
struct Packed {
  uint8_t* data = nullptr;
  int rows = 0;
  __host__ __device__ int64_t plane_bytes(int blocks) const { return (int64_t)blocks * 2 * rows * 128; }
};
static inline int packed_rows(int64_t n) { return (int)((n + 15) / 16 * 16 + 16); }

// Keys and values of every (row, kv head) plane, packed, and what the packing found.
struct PackedKeys {
  Packed k, v;
  uint32_t* amax = nullptr;    // [plane][2]: bits of the largest finite |k|, |v|
  int* odd = nullptr;          // [plane][2]: a key, a value is not finite or has no page
  uint8_t* flags_k = nullptr;  // [plane][k.rows]: kOdd: a component is not finite (stored as 0), kAbsent: no such page
  uint8_t* flags_v = nullptr;
};
constexpr uint8_t kOdd = 1, kAbsent = 2;

constexpr float kWeightShift = 15.0f;   // weights are held as 2^15 p (p <= 1): f16 pairs then reach 2^-40
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Carve {   // workspace layout; with a null base it only counts
  uint8_t* base; int64_t used = 0;
  template <typename T> T* take(int64_t n) {
    T* at = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += (n * (int64_t)sizeof(T) + 127) / 128 * 128;
    return at;
  }
};
// Allows a kernel its dynamic shared memory, once per device (`ready` holds a bit for each), and refuses one that was built with fewer
// registers than its warpgroups share out: the wait for registers would not end.
int prepare_kernel(std::atomic<uint64_t>& ready, const void* kernel, int smem, int threads, int shared_out);
// Whether float4 accesses fit a view of head_dim D.
static inline bool vec_view(const gn_view& v, int D) {
  return (reinterpret_cast<uintptr_t>(v.data) & 15) == 0 && D % 4 == 0 && v.batch_stride % 4 == 0 && v.head_stride % 4 == 0 && v.token_stride % 4 == 0;
}
// CTAs of a cluster that packs a plane of `rows` keys and finds its largest magnitude on the way (0: a launch of its own finds it).
// CTAs until the machine has four each, then until their rows (128 or fewer) still stand in a cache when they are read again.  Long planes of which
// there are few leave SMs idle that way.  A forward call with one launch and with two: 16 planes of 63 keys 14.3 and 17.4 us, 256 of 383 119 and 120
// (with the backward pass 401 and 409), 64 of 1024 94 and 91, 256 of 2000 334 and 329; 8 of 1280 63 and 57, 4 of 8704 233 and 145.
static inline int pack_cluster(int64_t rows, int64_t planes) {
  int ctas = 1;
  while (ctas < 8 && (rows >= 128 * ctas || (rows > 16 * ctas && planes * ctas < 592))) ctas *= 2;
  return rows <= 1280 || planes * ctas >= 296 ? ctas : 0;
}
// A call's first kernel waits for the stream as usual, and what the caller passed in is there from then on.  The others may set up while the one before
// still runs (launch_pdl).  Each CTA of such a kernel waits for the one before to be complete before it ends (and before it reads what that one
// writes), so that complete means complete with all before it.
// Clusters pack the keys, a call's first kernel or the one behind the new tokens' copy: launched in the ordinary way.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_cluster(void (*kernel)(KArgs...), dim3 grid, int threads, int ctas, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}
// Packs keys and values; amax and the 2 * planes words of odd stand in one piece.  norms: null, or [plane], which receives the bits
// of the largest squared norm of a scaled value row.
int stream_pack_keys(const StreamRows& s, const PackedKeys& pk, uint32_t* norms, cudaStream_t stream);

// tcgen05 forward of a call (streaming_tc.cu): the workspace it wants, and the launches.
int64_t stream_tc_forward_bytes(const StreamRows& s);
int stream_tc_forward(const StreamRows& s, const gn_view& out, float* lse, void* workspace, cudaStream_t stream, PackedKeys* packed = nullptr);
// The weights of a paged call's keys (streaming_tc_mass.cu), from the forward's packed keys and its log-sum-exps.
int64_t stream_tc_mass_bytes(const StreamRows& s);
int stream_tc_mass(const StreamRows& s, const PackedKeys& pk, const float* lse, const float* mass, float* mass_out, void* workspace, cudaStream_t stream);
// tcgen05 backward (streaming_tc_backward.cu), padded batches.
int64_t stream_tc_backward_bytes(const StreamRows& s);
int stream_tc_backward(const StreamRows& s, const gn_view& out, const gn_view& dout, const float* lse, const gn_view& dq, const gn_view& dk, const gn_view& dv,
                       int accumulate, void* workspace, cudaStream_t stream);

#ifdef __CUDACC__
namespace {

// Bounded wait of one thread in which the hardware holds it back (up to 2 us a try): sixteen warps that poll instead take the issue slots and the
// shared memory from the others, which made the fetching of Q four times slower.  False when the tries (up to about a second) ran out.
__device__ __forceinline__ bool hold(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < (1u << 19); ++i) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity), "r"(2000u) : "memory");
    if (ok) return true;
  }
  return false;
}
// The same for a whole warp, whose lanes may leave the loop on different tries: they meet before they go on, because warp-aligned instructions
// (tensor memory, named barriers) follow, and all of them take the same answer.
__device__ __forceinline__ bool hold_warp(uint32_t bar, uint32_t parity) {
  const bool ok = __all_sync(0xffffffffu, hold(bar, parity));
  __syncwarp();
  return ok;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// kind::f16, both operands f16, float32 accumulators: [4,6) D format 1, A and B formats 0, [17,23) N>>3, [24,29) M>>4, bit 16: B MN-major.
__device__ __forceinline__ uint32_t instr_desc_f16(int m, int n, int b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// A whole warp runs the issuing code, so that its operands stay in uniform registers (24 instructions of 64 cycles then issue in 1533
// cycles, against 1830 from one lane's branch); `el` is non-zero in the one lane that issues.
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t x;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(x));
  return x;
}
__device__ __forceinline__ void umma_f16(uint32_t el, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(el) : "memory");
}
// A in tensor memory: lane = row, a 32-bit column holds two consecutive elements of the contraction index.
__device__ __forceinline__ void umma_f16_ts(uint32_t el, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(el) : "memory");
}
__device__ __forceinline__ void commit_by(uint32_t el, uint32_t bar) { if (el) umma_commit(bar); }
// MN-major operand, 128-byte swizzle: 64 channels a row of 128 bytes, 8 contraction rows 1024 bytes (stride offset), the next 64
// channels `group` bytes on (leading offset).
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr, uint32_t group) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(group >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15])
      : "memory");
}
// Transposes N x N blocks of four floats among groups of N lanes (N 4 or 8): block k of lane i becomes block i of lane k.  With
// it a thread that owns a row moves its channels by whole 64- or 128-byte pieces: lanes i of a group access piece i of one row.
// (A warp whose lanes access 16 bytes of 32 rows each took 10 000 cycles to store a 64 KB tile.)
template <int N>
__device__ __forceinline__ void transpose_blocks(float (&x)[4 * N]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < N; d <<= 1) {
    const bool upper = lane & d;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (k & d) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = x[4 * k + e], b = x[4 * (k | d) + e], y = __shfl_xor_sync(0xffffffffu, upper ? a : b, d);
        x[4 * k + e] = upper ? y : a;
        x[4 * (k | d) + e] = upper ? b : y;
      }
    }
  }
}
// All threads of the cluster's CTAs meet; what each wrote to shared memory before is seen by the others after.
__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// The largest of the words that the cluster's CTAs hold where this one holds `mine` (shared memory; all of a warp's threads call).
__device__ __forceinline__ uint32_t cluster_largest(const uint32_t* mine, int ctas) {
  uint32_t x = 0;
  const int lane = threadIdx.x & 31;
  if (lane < ctas)
    asm volatile("{\n\t.reg .b32 at;\n\tmapa.shared::cluster.u32 at, %1, %2;\n\tld.shared::cluster.u32 %0, [at];\n\t}" : "=r"(x) : "r"(smem_u32(mine)), "r"(lane) : "memory");
  return __reduce_max_sync(0xffffffffu, x);
}
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ bool finite_bits(float x) { return (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u; }

// Two floats to hi and lo pairs (the first in the low half).
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
// The power of two that brings `amax` (bits of the largest finite magnitude) to [2^14, 2^15), and its inverse.
__device__ __forceinline__ int scale_exponent(uint32_t amax) { return amax == 0 ? 0 : 14 + 127 - max((int)(amax >> 23), 27); }
__device__ __forceinline__ void plane_scale(uint32_t amax, float& s, float& inverse) {
  const int e = max((int)(amax >> 23), 27) - 127;   // 0 and what is below 2^-100 scale like 2^-100
  s = amax == 0 ? 1.0f : __uint_as_float((uint32_t)(14 - e + 127) << 23);
  inverse = amax == 0 ? 1.0f : __uint_as_float((uint32_t)(e - 14 + 127) << 23);
}

// Registers move between warpgroups inside what the launch holds (prepare_kernel).
template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ uint64_t bits_below(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }

// The keys that the queries at positions pos0 .. pos1 see, as two runs: virtual key c is key c below a_len and key c + shift from
// there.  Runs start at multiples of 8.
struct KeyRuns { int a_len, shift, total; };
__device__ __forceinline__ KeyRuns key_runs(const StreamRows& s, int pos0, int pos1) {
  KeyRuns k{0, 0, 0};
  if (pos1 < 0) return k;
  const int begin = (s.window < 0 ? 0 : max(0, pos0 - s.window)) & ~7, sinks8 = (min(s.sinks, pos1 + 1) + 7) & ~7;
  if (sinks8 == 0) k.shift = begin;
  else if (begin > sinks8) { k.a_len = sinks8; k.shift = begin - sinks8; }
  k.total = pos1 + 1 - k.shift;
  return k;
}

}  // namespace
#endif

}  // namespace gn
