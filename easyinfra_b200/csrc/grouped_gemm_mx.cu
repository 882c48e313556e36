// Grouped expert GEMMs on microscaled operands: MX8 activation rows (e4m3) times MX4
// weights (e2m1), scaled and accumulated in fp32 inside the tensor cores
// (tcgen05.mma kind::mxf8f6f4 with block scales, mx.cuh for the formats):
//   swiglu  act = MX8(silu(x Wg^T) * (x Wu^T))     down  y = bf16(act Wd^T)
// for every expert e and its rows [off[e], off[e+1]).
//
// Every product of two elements and their scales is exact in fp32, so the result is the
// fp32 sum over K of the values that the rows and the weights stand for.
//
// Weights are laid out once (MX4 product layout):
//   elements  [P, w_rows, K/2] bytes; for swiglu the rows of gate and up are interleaved
//             by 32 (32 gate rows, then the 32 up rows of the same columns), so that any
//             64 accumulator columns hold 32 gates and their 32 ups, and one output block
//             of 32 (one MX8 scale) belongs to one thread
//   scales    [P, K/128, w_rows/128, 512] bytes: for 128 rows x 128 columns the 32 x 16
//             bytes that tcgen05.cp copies to TMEM (byte (r % 32) * 16 + (r / 32) * 4 + k
//             is row r's scale of its k-th 32 columns), n-tiles adjacent
// The scales of activation rows stay in the rows; a warp gathers 16 bytes a row (four
// k-blocks) and writes the same 512-byte form to shared memory.
//
// A tile is BMA activation rows of one expert times NU units of 64 weight rows (NU <= 4).
// Its parts:
//   warp 0     TMA: 128 K-columns of the rows (e4m3, 128 B a row) and of the weight rows
//              (64 B a row in memory; the TMA spreads 16 elements over 16 bytes, half of
//              them gap, which is the form the tensor cores take beside 8-bit operands),
//              and the weights' scale tiles
//   warp 1     tcgen05.cp of the stage's scales, then 4 MMAs of M = 128, N = 64 NU, K = 32
//   warp 2     activation scales
//   warps 4..7 epilogue from the fp32 accumulator in TMEM
// The MMA always has M = 128.  Rows that are not loaded are whatever shared memory holds;
// their accumulator rows are never read.
//
// One persistent CTA per SM, and two ways of giving out the work (MxTiles):
//   tiles   (expert, n-tile of 4 units, m-tile of 128 rows) round robin, m fastest, so that
//           the m-tiles of a weight n-tile run together and share it through L2
//   stream  few rows per expert: the weights are the traffic, and every CTA gets an equal,
//           contiguous share of all (expert, 64-row m-tile, unit) in that order, cut into
//           tiles of up to 4 units.  Whole n-tiles of 256 rows would leave the last round of
//           CTAs up to 17% short of work (896 tiles on 148 SMs at 8 experts of 28672 rows).
//
// TMEM: the scales of stage s have columns of their own, rewritten only after the MMAs
// that read them have committed.  Two accumulators of 256 columns follow that share OVL
// columns, and the next tile's MMAs start as soon as the epilogue has read those (it reads
// them first).
#include <atomic>
#include <cstdlib>

#include "kernels.cuh"
#include "mx.cuh"

namespace b200moe {

constexpr int MXG_BK = 128;
constexpr int MXG_MAXP = 512;
constexpr int MXG_SF_BYTES = 512;  // scales of 128 rows x 128 columns
constexpr uint64_t kDrainNs = 1000000;

constexpr int MXG_BN = 256;        // weight rows of a full tile: 4 units
constexpr int MXG_UNIT = 64;
constexpr int MXG_THREADS = 256;

template <int STAGES, bool STREAM>
struct MxGemmShape {
  static constexpr int BMA = STREAM ? 64 : 128;           // activation rows of a tile
  static constexpr int A_BOX = STREAM ? 32 : 128;         // rows a TMA load brings
  static constexpr int B_BOX = STREAM ? 1 : 2;            // weight units a TMA load brings
  static constexpr int A_SLOT = BMA * MXG_BK;             // bytes of a stage's activation rows
  static constexpr int B_SLOT = MXG_BN * MXG_BK;          // weights in shared memory (padded form)
  static constexpr int SFB_SLOT = 2 * MXG_SF_BYTES;
  static constexpr int SF_COLS = 12;                      // TMEM columns of a stage's scales: 4 + 2 * 4
  static constexpr int SF0 = 512 - SF_COLS * STAGES;
  static constexpr int ACC1 = SF0 - MXG_BN;               // accumulator 0 is at column 0
  static constexpr int OVL = MXG_BN - ACC1;               // columns both accumulators use
  // the last slot's MMA reads 128 rows from its start: that stays inside the weight ring
  static constexpr int OFF_B = STAGES * A_SLOT;
  static constexpr int OFF_SFA = OFF_B + STAGES * B_SLOT;
  static constexpr int OFF_SFB = OFF_SFA + STAGES * MXG_SF_BYTES;
  static constexpr int OFF_CTRL = OFF_SFB + STAGES * SFB_SLOT;
  static constexpr int CTRL_BYTES = 256 + 2 * (MXG_MAXP + 1) * 4;
  static constexpr int SMEM_BYTES = 1024 + OFF_CTRL + CTRL_BYTES;
  static_assert(OVL > 0 && OVL <= 64, "the shared columns lie in one chunk of 64");
  static_assert(SF0 % 4 == 0, "TMEM columns");
  static_assert(128 * MXG_BK <= A_SLOT + STAGES * B_SLOT, "the MMA's 128 rows stay in shared memory");
  static_assert((2 * STAGES + 3) * 8 + 16 <= 256, "barriers");
  static_assert(SMEM_BYTES <= 232448, "shared memory");
};

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

// 512 bytes of scales (32 rows of 16 bytes) to 4 TMEM columns, repeated for the four
// lane quarters.
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
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

// The tiles of a CTA, in order; every role walks its own copy.
template <bool STREAM>
struct MxTiles {
  static constexpr int BMA = STREAM ? 64 : 128;
  const int* prefix;    // [P + 1] tiles (stream: units) before each expert
  const int32_t* off;   // [P + 1] rows
  int P, units;         // units of 64 weight rows per expert
  int pos, end, step;
  int e, row0, rows;    // expert, first activation row, rows of the tile (at most BMA)
  int n0, nu;           // first unit, units

  __device__ __forceinline__ MxTiles(const int* prefix_, const int32_t* off_, int P_, int units_)
      : prefix(prefix_), off(off_), P(P_), units(units_) {
    const int total = prefix[P];
    if (STREAM) {
      pos = static_cast<int>(static_cast<int64_t>(total) * blockIdx.x / gridDim.x);
      end = static_cast<int>(static_cast<int64_t>(total) * (blockIdx.x + 1) / gridDim.x);
      step = 0;
    } else {
      pos = blockIdx.x;
      end = total;
      step = gridDim.x;
    }
  }

  __device__ __forceinline__ bool next() {
    if (pos >= end) return false;
    int lo = 0, hi = P - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] <= pos) lo = mid; else hi = mid - 1;
    }
    e = lo;
    const int local = pos - prefix[e];
    const int all = off[e + 1] - off[e];
    int m;
    if (STREAM) {
      m = local / units;
      n0 = local - m * units;
      // an odd first unit is the second half of a scale tile: the tile then ends at 3
      // units, so that it never touches more than two scale tiles
      nu = min(min(4 - (n0 & 1), units - n0), end - pos);
      pos += nu;
    } else {
      const int mt = (all + BMA - 1) / BMA;
      const int n = local / mt;
      m = local - n * mt;
      n0 = 4 * n;
      nu = min(4, units - n0);
      pos += step;
    }
    row0 = off[e] + m * BMA;
    rows = min(BMA, all - m * BMA);
    return true;
  }
};

// silu(g) * u with the hardware exponential and reciprocal: a few units in the last place
// of fp32, against the e4m3 rounding of 2^-4 that follows.  -g beyond 88 makes the
// exponential infinite and the result g * 0, as in the limit.
__device__ __forceinline__ float silu_mul_fast(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

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

template <int STAGES, bool SWIGLU, bool STREAM>
__global__ void __launch_bounds__(MXG_THREADS, 1)
    grouped_gemm_mx_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                           const __grid_constant__ MxGemmParams p) {
  using S = MxGemmShape<STAGES, STREAM>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sa = smem;
  uint8_t* sb = smem + S::OFF_B;
  uint8_t* ssfa = smem + S::OFF_SFA;
  uint8_t* ssfb = smem + S::OFF_SFB;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::OFF_CTRL);  // TMA bytes + the activation scales
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;   // [2] accumulator complete
  uint64_t* tread = tfull + 2;        // shared columns of the last tile read
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tread + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  int* prefix = reinterpret_cast<int*>(smem + S::OFF_CTRL + 256);  // [P+1] work before each expert
  int32_t* off = prefix + (MXG_MAXP + 1);                          // [P+1] row offsets, clamped

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int units = p.w_rows / MXG_UNIT;
  pdl_trigger();

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&tfull[0], 1);
    mbar_init(&tfull[1], 1);
    mbar_init(tread, 4);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  pdl_wait();  // inputs of this launch are complete and visible from here on
  if (warp == 2) {
    // row offsets, forced into [0, rows_cap] and ascending, so that no tile addresses
    // outside the activation rows whatever the caller's table holds
    int run = 0, bad = 0, last = 0;
    for (int base = 0; base <= p.P; base += 32) {
      const int e = base + lane;
      const int raw = e <= p.P ? p.expert_offsets[e] : 0x7fffffff;
      int v = min(max(raw, 0), p.rows_cap);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = max(v, t);
      }
      v = max(v, last);
      if (e <= p.P) {
        off[e] = v;
        bad |= v != raw;
      }
      last = __shfl_sync(0xffffffffu, v, 31);
    }
    if (bad) record_status(p.status, kStatusBadIndex);
    __syncwarp();
    const int per_m = STREAM ? units : (units + 3) / 4;
    for (int base = 0; base < p.P; base += 32) {
      const int e = base + lane;
      const int c = e < p.P ? ((off[e + 1] - off[e] + S::BMA - 1) / S::BMA) * per_m : 0;
      int incl = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (e < p.P) prefix[e] = run + incl - c;
      run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) prefix[p.P] = run;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const int num_kb = p.K / MXG_BK;
  MxTiles<STREAM> t(prefix, off, p.P, units);

  if (warp == 0) {
    if (elect_one()) {
      // ------------------------------------------------ TMA producer
      const int nt128 = p.w_rows / 128;
      const uint64_t stream_once = l2_policy_evict_first();
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      while (ok && t.next()) {
        const int a_loads = STREAM ? (t.rows + S::A_BOX - 1) / S::A_BOX : 1;
        const int row_b = t.e * p.w_rows + t.n0 * MXG_UNIT;
        const int sf0 = t.n0 >> 1;
        const uint32_t sf_bytes = static_cast<uint32_t>(((t.n0 + t.nu - 1) >> 1) - sf0 + 1) * MXG_SF_BYTES;
        const uint32_t tx = a_loads * (S::A_BOX * MXG_BK) + t.nu * (MXG_UNIT * MXG_BK / 2) + sf_bytes;
        const uint8_t* sf = p.w_scales + (static_cast<int64_t>(t.e) * num_kb * nt128 + sf0) * MXG_SF_BYTES;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, p.status)) { ok = false; break; }
          uint64_t* bar = &full[stage];
          mbar_arrive_expect_tx(bar, tx);
          uint8_t* dst = sb + stage * S::B_SLOT;
          for (int u = 0; u < t.nu; u += S::B_BOX) {
            if (STREAM)
              tma_load_2d_hint(dst + u * (MXG_UNIT * MXG_BK), &map_b, bar, kb * MXG_BK, row_b + u * MXG_UNIT, stream_once);
            else
              tma_load_2d(dst + u * (MXG_UNIT * MXG_BK), &map_b, bar, kb * MXG_BK, row_b + u * MXG_UNIT);
          }
          for (int i = 0; i < a_loads; ++i)
            tma_load_2d(sa + stage * S::A_SLOT + i * (S::A_BOX * MXG_BK), &map_a, bar, kb * MXG_BK,
                        t.row0 + i * S::A_BOX);
          bulk_load(ssfb + stage * S::SFB_SLOT, sf + static_cast<int64_t>(kb) * nt128 * MXG_SF_BYTES, sf_bytes, bar);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      // ------------------------------------------------ scales to TMEM, MMAs
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      bool ok = true;
      for (; ok && t.next(); ++it) {
        // the previous tile's shared columns are read (and with them, in the epilogue's
        // order, everything of the tile before it)
        if (it > 0 && !mbar_wait(tread, (it - 1) & 1, abort_flag, p.status)) break;
        tc_fence_after();
        const uint32_t idesc = make_idesc_mx(128, t.nu * MXG_UNIT);
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>((it & 1) * S::ACC1);
        const uint32_t sfb_half = static_cast<uint32_t>((t.n0 & 1) * 2);  // two of a scale tile's four columns
        const bool two = ((t.n0 + t.nu - 1) >> 1) != (t.n0 >> 1);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full[stage], phase, abort_flag, p.status)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sfa = tmem_base + static_cast<uint32_t>(S::SF0 + stage * S::SF_COLS);
          const uint32_t sfb = sfa + 4;
          const uint32_t sfb_smem = smem_u32(ssfb + stage * S::SFB_SLOT);
          tmem_cp_scales(sfa, make_scale_desc(smem_u32(ssfa + stage * MXG_SF_BYTES)));
          tmem_cp_scales(sfb, make_scale_desc(sfb_smem));
          if (two) tmem_cp_scales(sfb + 4, make_scale_desc(sfb_smem + MXG_SF_BYTES));
          const uint64_t adesc = make_sw128_kmajor_desc(smem_u32(sa + stage * S::A_SLOT));
          const uint64_t bdesc = make_sw128_kmajor_desc(smem_u32(sb + stage * S::B_SLOT));
#pragma unroll
          for (uint32_t k = 0; k < MXG_BK / MX_BLOCK; ++k)  // 32 bytes of K each; byte k of the scale words
            umma_mx(d_tmem, adesc + 2ull * k, bdesc + 2ull * k, idesc | (k << 29) | (k << 4), sfa, sfb + sfb_half,
                    (static_cast<uint32_t>(kb) | k) != 0 ? 1u : 0u);
          umma_commit(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        umma_commit(&tfull[it & 1]);
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // -------------------------------------------------- activation scales
    // Lane l holds rows l, l + 32, ... of the tile; 16 bytes of a row are its scales of
    // four k-blocks, and word j of the four rows is lane l's 16 bytes of k-block j.
    constexpr int R = S::BMA / 32;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    while (ok && t.next()) {
      const uint8_t* src[R];
      bool have[R];
      uint4 next[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        have[r] = r * 32 + lane < t.rows;
        src[r] = p.a_scales + static_cast<int64_t>(t.row0 + (have[r] ? r * 32 + lane : 0)) * p.lda;
        next[r] = have[r] ? *reinterpret_cast<const uint4*>(src[r]) : make_uint4(0, 0, 0, 0);
      }
      for (int kb0 = 0; ok && kb0 < num_kb; kb0 += 4) {
        uint4 cur[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          cur[r] = next[r];
          if (have[r] && kb0 + 4 < num_kb) next[r] = *reinterpret_cast<const uint4*>(src[r] + (kb0 + 4) * 4);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (kb0 + j < num_kb && ok) {
            int go = 0;
            if (lane == 0) go = mbar_wait(&empty[stage], phase ^ 1u, abort_flag, p.status) ? 1 : 0;
            ok = __shfl_sync(0xffffffffu, go, 0) != 0;
            if (ok) {
              uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
              for (int r = 0; r < R; ++r) w[r] = j == 0 ? cur[r].x : j == 1 ? cur[r].y : j == 2 ? cur[r].z : cur[r].w;
              *reinterpret_cast<uint4*>(ssfa + stage * MXG_SF_BYTES + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(&full[stage]);
              if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
          }
        }
      }
    }
  } else if (warp >= 4) {
    // -------------------------------------------------- epilogue
    const int quarter = warp & 3;          // TMEM lanes [32*quarter, 32*quarter + 32)
    const int r = quarter * 32 + lane;
    const bool wide = ((reinterpret_cast<uintptr_t>(p.out) | static_cast<uintptr_t>(p.ldo)) & 31u) == 0;
    for (int it = 0; t.next(); ++it) {
      const int acc = it & 1;
      const bool warp_has_rows = quarter * 32 < t.rows;
      bool valid = r < t.rows;
      int64_t orow = t.row0 + r;
      if (!SWIGLU && valid && p.out_row_map != nullptr) {
        orow = p.out_row_map[orow];
        if (orow < 0 || orow >= p.out_rows) {
          record_status(p.status, kStatusBadIndex);
          valid = false;
        }
      }
      int ok = 0;
      if (lane == 0) ok = mbar_wait(&tfull[acc], (it >> 1) & 1, abort_flag, p.status) ? 1 : 0;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      tc_fence_after();
      const uint32_t tbase =
          tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * S::ACC1);
      uint8_t* out_row = static_cast<uint8_t*>(p.out) + orow * p.ldo;  // ldo in bytes
#pragma unroll 1
      for (int i = 0; i < t.nu; ++i) {
        // the chunk with the shared columns first: the last one of accumulator 0, the
        // first of accumulator 1
        const int ch = acc != 0 ? i : i == 0 ? t.nu - 1 : i - 1;
        uint32_t lo[32], hi[32];
        if (warp_has_rows) {
          tmem_ld_32x32b_x32(tbase + ch * 64, lo);
          tmem_ld_32x32b_x32(tbase + ch * 64 + 32, hi);
          tmem_ld_wait();
        }
        if (i == 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(tread);
        }
        if (!valid) continue;
        if (SWIGLU) {
          // lo: 32 gates, hi: the ups of the same columns; one MX8 block
          const int col = (t.n0 + ch) * 32;
          uint32_t amax = 0;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float a = silu_mul_fast(__uint_as_float(lo[j]), __uint_as_float(hi[j]));
            lo[j] = __float_as_uint(a);
            amax = max(amax, lo[j] & 0x7fffffffu);
          }
          const uint32_t byte = mx8_scale_byte(amax);
          const float inv = mx_inverse_scale(byte);
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            w[j] = cvt_e4m3x4(__uint_as_float(lo[4 * j]) * inv, __uint_as_float(lo[4 * j + 1]) * inv,
                              __uint_as_float(lo[4 * j + 2]) * inv, __uint_as_float(lo[4 * j + 3]) * inv);
          store_32(out_row + col, w, wide);
          out_row[p.N + col / MX_BLOCK] = static_cast<uint8_t>(byte);
        } else {
          uint8_t* dst = out_row + (t.n0 + ch) * 128;
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
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // a wait gave up: loads of the ring may still be on their way into shared memory,
    // which the CTA must not hand back before they land
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < kDrainNs) __nanosleep(1000);
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// ------------------------------------------------------------------ host side
// 2D maps over rows of K elements: 8-bit (row stride ld bytes), or 4-bit packed (K/2
// bytes a row) spread by the TMA to 16 elements per 16 bytes.  Box: rows x 128.
static int make_mx_map(CUtensorMap* map, const void* base, int64_t rows, int64_t K, int64_t ld_bytes, int box_rows,
                       bool four_bit) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld_bytes)};
  const cuuint32_t box[2] = {MXG_BK, static_cast<cuuint32_t>(box_rows)};
  return encode_tma_map_2d(map, four_bit ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8, base,
                           dims, strides, box);
}

template <int STAGES, bool SWIGLU, bool STREAM>
static int run_mx(const MxGemmLaunch& L, int64_t work, cudaStream_t stream) {
  using S = MxGemmShape<STAGES, STREAM>;
  auto* kern = grouped_gemm_mx_kernel<STAGES, SWIGLU, STREAM>;
  CUtensorMap ma, mb;
  if (make_mx_map(&ma, L.a, L.p.rows_cap, L.p.K, L.p.lda, S::A_BOX, false) != 0) return -1;
  if (make_mx_map(&mb, L.w, static_cast<int64_t>(L.p.P) * L.p.w_rows, L.p.K, L.p.K / 2, S::B_BOX * MXG_UNIT, true) != 0)
    return -1;
  static_assert(S::SMEM_BYTES > 114 * 1024, "one CTA per SM: it holds all of the SM's TMEM");
  static std::atomic<uint64_t> attr_set_mask{0};  // one bit per device ordinal
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (!(attr_set_mask.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM_BYTES) != cudaSuccess)
      return -3;
    attr_set_mask.fetch_or(bit, std::memory_order_release);
  }
  const int limit = gemm_grid_limit();
  launch_kernel(kern, dim3(static_cast<unsigned>(work < limit ? work : limit)), dim3(MXG_THREADS), S::SMEM_BYTES,
                stream, ma, mb, L.p);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

template <bool SWIGLU>
static int pick_mx(const MxGemmLaunch& L, cudaStream_t stream) {
  if (L.p.P > MXG_MAXP) return -4;
  const int64_t rows = L.rows_hint > 0 ? L.rows_hint : L.p.rows_cap;
  const int64_t units = L.p.w_rows / MXG_UNIT;
  const int64_t stream_work = ((L.p.rows_cap + 63) / 64 + L.p.P) * units;
  const int64_t tile_work = ((L.p.rows_cap + 127) / 128 + L.p.P) * ((units + 3) / 4);
  static const int force = getenv("MXV") ? atoi(getenv("MXV")) : 0;
  if (force == 1 || (force == 0 && rows <= 32 * static_cast<int64_t>(L.p.P) && stream_work <= 0x7fffffff))
    return run_mx<5, SWIGLU, true>(L, stream_work, stream);
  if (tile_work > 0x7fffffff) return -5;
  return run_mx<4, SWIGLU, false>(L, tile_work, stream);
}

int launch_grouped_mx(const MxGemmLaunch& L, bool swiglu, cudaStream_t stream) {
  return swiglu ? pick_mx<true>(L, stream) : pick_mx<false>(L, stream);
}

}  // namespace b200moe
