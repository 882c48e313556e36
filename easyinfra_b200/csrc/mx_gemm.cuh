// What the grouped GEMMs on microscaled operands share (grouped_gemm_mx.cu,
// grouped_gemm_mx_2sm.cu): instructions, the walk over experts, the activation scales and
// the epilogue's arithmetic.
#pragma once

#include <atomic>

#include "kernels.cuh"
#include "mx.cuh"

namespace b200moe {

constexpr int MXG_BK = 128;
constexpr int MXG_MAXP = 512;
constexpr int MXG_SF_BYTES = 512;  // scales of 128 rows x 128 columns
constexpr uint64_t kDrainNs = 1000000;
constexpr int MXG_BN = 256;        // weight rows of a full tile: 4 units
constexpr int MXG_UNIT = 64;
constexpr int MXG_UNIT_BYTES = MXG_UNIT * MXG_BK / 2;  // a unit's k-block in memory

// D[tmem] (+)= A * B^T with block scales from TMEM; e4m3 A, e2m1 B (padded form), fp32 D.
__device__ __forceinline__ void umma_mx(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void umma_mx_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}

// 512 bytes of scales (32 rows of 16 bytes) to 4 TMEM columns, repeated for the four
// lane quarters.
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// The same in both CTAs of a pair, each from its own shared memory.
__device__ __forceinline__ void tmem_cp_scales_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Unswizzled 32 x 16-byte matrix: 8-row groups of 128 contiguous bytes (stride 128).
__device__ __forceinline__ uint64_t make_scale_desc(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(1u) << 16) |
         (static_cast<uint64_t>(128u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46);
}

// Instruction descriptor of kind::mxf8f6f4: A e4m3 (0 at [7,10)), B e2m1 (5 at [10,13)),
// N >> 3 at [17,23), e8m0 scales (bit 23), M >> 4 at [24,29); the byte of the scale words
// for A at [29,31) and for B at [4,6).
__host__ __device__ constexpr uint32_t make_idesc_mx(int M, int N) {
  return (5u << 10) | (static_cast<uint32_t>(N >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(M >> 4) << 24);
}

// The same with the operands exchanged: A e2m1, B e4m3.
__host__ __device__ constexpr uint32_t make_idesc_mx_wm(int M, int N) {
  return (5u << 7) | (static_cast<uint32_t>(N >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(M >> 4) << 24);
}

// A wait gave up: loads of the ring may still be on their way into shared memory, which the
// CTA must not hand back before they land.
__device__ __forceinline__ void mx_drain() {
  const uint64_t t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < kDrainNs) __nanosleep(1000);
}

// Barrier of the four epilogue warps.
__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// silu(g) * u with the hardware exponential and reciprocal, whose documented errors are 2 +
// 1.17 |g| and 2 units in the last place of fp32: up to 8 units (2^-20) for |g| below 2, 2^-17 at
// g = -40, 2^-16 at -87, against the e4m3 rounding of 2^-4 that follows.  From g = -87.4 on
// the denominator is beyond 2^126, where the quotient is 0; the exact value is below
// 2^-119 |u| there.  The exact forms (expf, a
// rounded division) cost more than the epilogue has time for: 64 tokens x 8 of 128 experts
// of 1536 x 2048 took 55 us instead of 35, 16384 x 6 rows of 64 experts of 2816 x 2048 600
// instead of 451; and they flip no fewer codes (105 instead of 93 of 100.7 M, K = 4096),
// since those come from the order of the tensor cores' sums.
__device__ __forceinline__ float silu_mul_fast(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// Bounded wait for a barrier's phase.  The hardware suspends the thread for up to kSuspendNs
// at a time, so that waiting roles do not poll: the tensor-core instructions of the issuing
// warp share the path that polls go through (Mixtral SwiGLU on CTA pairs 3.4 ms polling,
// 2.5 ms suspended).  CLUSTER: the other CTA of the pair arrives, and its writes before that
// are visible after the wait.  The loop is out of line, the issuing role being unrolled over
// the ring.
constexpr uint32_t kSuspendNs = 20000;
template <bool CLUSTER>
__device__ __forceinline__ bool mx_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  if (CLUSTER)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(kSuspendNs)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(kSuspendNs)
        : "memory");
  return ok != 0;
}
template <bool CLUSTER>
static __device__ __noinline__ bool mx_wait_poll(uint32_t bar, uint32_t parity, volatile int* abort, int* status) {
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    if (mx_try_wait<CLUSTER>(bar, parity)) return true;
    if (*abort) return false;
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      *abort = 1;
      record_status(status, kStatusTimeout);
      return false;
    }
  }
}
template <bool CLUSTER = false>
__device__ __forceinline__ bool mx_wait(uint32_t bar, uint32_t parity, volatile int* abort, int* status) {
  return mx_try_wait<CLUSTER>(bar, parity) || mx_wait_poll<CLUSTER>(bar, parity, abort, status);
}

// Exclusive maximum (MAX, of values >= 0) or sum over the CTA's threads; shared: 2 * warps
// ints, alternating between the two calls so that one barrier each suffices.
template <int THREADS, bool MAX>
__device__ __forceinline__ int cta_scan_exclusive(int v, int* shared) {
  constexpr int WARPS = THREADS / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* part = shared + (MAX ? 0 : WARPS);
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl = MAX ? max(incl, t) : incl + t;
  }
  if (lane == 31) part[warp] = incl;
  int excl = __shfl_up_sync(0xffffffffu, incl, 1);
  if (lane == 0) excl = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w)
    if (w < warp) excl = MAX ? max(excl, part[w]) : excl + part[w];
  return excl;
}

// 32 bytes to global memory: one store where rows start at multiples of 32 bytes (whole
// sectors: 98304 x 2048 bf16 outputs 327 us with 16-byte stores, 288 with these).
__device__ __forceinline__ void store_32(uint8_t* dst, const uint32_t (&w)[8], bool wide) {
  if (wide) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// 64 accumulator columns of a row as bf16.
__device__ __forceinline__ void store_bf16_64(uint8_t* dst, const uint32_t (&lo)[32], const uint32_t (&hi)[32],
                                              bool wide) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = 16 * (q & 1) + 2 * j;
      w[j] = q < 2 ? pack_bf16x2(__uint_as_float(lo[c]), __uint_as_float(lo[c + 1]))
                   : pack_bf16x2(__uint_as_float(hi[c]), __uint_as_float(hi[c + 1]));
    }
    store_32(dst + 32 * q, w, wide);
  }
}

// Row offsets, forced into [0, rows_cap] and ascending, so that no tile addresses outside the
// activation rows whatever the caller's table holds (off [P+1]), and the work before each
// expert, m-tiles of `bma` rows times per_m (prefix [P+1]).  Every thread of the CTA holds
// consecutive entries; one load latency and two scans (one warp walking the table took
// 2 us at 128 experts).  The caller synchronises before reading either table.
template <int THREADS>
__device__ __forceinline__ void mx_tables(const MxGemmParams& p, int bma, int per_m, int* prefix, int32_t* off,
                                          int* scan) {
  constexpr int EPT = (MXG_MAXP + THREADS) / THREADS;
  const int e0 = threadIdx.x * EPT;
  int v[EPT], raw[EPT], c[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) raw[i] = e0 + i <= p.P ? p.expert_offsets[e0 + i] : 0;
  int run = 0;
#pragma unroll
  for (int i = 0; i < EPT; ++i) run = v[i] = max(run, min(max(raw[i], 0), p.rows_cap));
  const int before = cta_scan_exclusive<THREADS, true>(run, scan);
  bool bad = false;
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    v[i] = max(v[i], before);
    if (e0 + i <= p.P) {
      off[e0 + i] = v[i];
      bad |= v[i] != raw[i];
    }
  }
  if (bad) record_status(p.status, kStatusBadIndex);
  __syncthreads();
  run = 0;
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    c[i] = run;
    if (e0 + i < p.P) run += ((off[e0 + i + 1] - v[i] + bma - 1) / bma) * per_m;
  }
  const int sum = cta_scan_exclusive<THREADS, false>(run, scan);
#pragma unroll
  for (int i = 0; i < EPT; ++i)
    if (e0 + i <= p.P) prefix[e0 + i] = sum + c[i];
}

// The last expert whose work starts at or before `pos`, searched from `from`.
__device__ __forceinline__ int mx_find_expert(const int* prefix, int P, int pos, int from) {
  if (pos < prefix[from + 1]) return from;
  int lo = from + 1, hi = P - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= pos) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Lane l holds rows l, l + 32, ... of a tile of R * 32 rows; 16 bytes of a row are its scales
// of four k-blocks, and word j of the rows is lane l's 16 bytes of k-block j.
template <int R>
struct MxRowScales {
  const uint8_t* src[R];
  bool have[R];
  uint4 cur[R], next[R];

  __device__ __forceinline__ void start(const MxGemmParams& p, int row0, int rows, int lane) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      have[r] = r * 32 + lane < rows;
      src[r] = p.a_scales + static_cast<int64_t>(row0 + (have[r] ? r * 32 + lane : 0)) * p.lda;
      next[r] = have[r] ? *reinterpret_cast<const uint4*>(src[r]) : make_uint4(0, 0, 0, 0);
    }
  }
  // the four k-blocks from kb0; asks for the next four
  __device__ __forceinline__ void advance(int kb0, int num_kb) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      cur[r] = next[r];
      if (have[r] && kb0 + 4 < num_kb) next[r] = *reinterpret_cast<const uint4*>(src[r] + (kb0 + 4) * 4);
    }
  }
  __device__ __forceinline__ uint4 block(int j) const {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < R; ++r) w[r] = j == 0 ? cur[r].x : j == 1 ? cur[r].y : j == 2 ? cur[r].z : cur[r].w;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// One MX8 block of the SwiGLU output from 32 gates and ups: the packed elements, and the
// scale byte as result.
__device__ __forceinline__ uint32_t mx_swiglu_block(uint32_t (&g)[32], const uint32_t (&u)[32], uint32_t (&w)[8]) {
  uint32_t amax = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    g[j] = __float_as_uint(silu_mul_fast(__uint_as_float(g[j]), __uint_as_float(u[j])));
    amax = max(amax, g[j] & 0x7fffffffu);
  }
  const uint32_t byte = mx8_scale_byte(amax);
  const float inv = mx_inverse_scale(byte);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    w[j] = cvt_e4m3x4(__uint_as_float(g[4 * j]) * inv, __uint_as_float(g[4 * j + 1]) * inv,
                      __uint_as_float(g[4 * j + 2]) * inv, __uint_as_float(g[4 * j + 3]) * inv);
  return byte;
}

// 2D maps of the activations (rows of K bytes, boxes of box_rows x 128) and of the weights:
// the product layout is a matrix of rows of 128 4-bit elements, of which a unit's k-block is
// 64; the TMA spreads 16 elements over 16 bytes.
int make_mx_maps(CUtensorMap* ma, CUtensorMap* mb, const MxGemmLaunch& L, int box_rows);

// Lets a kernel use BYTES of dynamic shared memory, once per device.
template <int BYTES, auto KERN>
inline bool mx_set_smem() {
  static std::atomic<uint64_t> done{0};  // one bit per device ordinal
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return true;
  if (cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_release);
  return true;
}

// Weights as the MMA's A operand, for few rows per expert (grouped_gemm_mx_wm.cu), and the
// units of work of such a launch at most (31 bits).
int launch_grouped_mx_wm(const MxGemmLaunch& L, bool swiglu, cudaStream_t stream);
inline int64_t mx_wm_work(const MxGemmLaunch& L) {
  return ((static_cast<int64_t>(L.p.rows_cap) + 63) / 64 + L.p.P) * (L.p.w_rows / MXG_UNIT);
}

// CTA pairs (grouped_gemm_mx_2sm.cu); w_rows a multiple of 256.
int launch_grouped_mx_pair(const MxGemmLaunch& L, bool swiglu, cudaStream_t stream);

}  // namespace b200moe
