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
// One persistent CTA per SM walks (expert, n-tile, m-tile) with m fastest:
//   warp 0     TMA: 128 K-columns of BMA rows (e4m3, 128 B a row) and of BN weight rows
//              (64 B a row in memory; the TMA spreads 16 elements over 16 bytes, half of
//              them gap, which is the form the tensor cores take beside 8-bit operands),
//              and the weights' scale tiles
//   warp 1     tcgen05.cp of the stage's scales, then 4 MMAs of M = 128, N = BN, K = 32
//   warp 2     activation scales
//   warps 4..  epilogue from the fp32 accumulator in TMEM
// The MMA always has M = 128.  With BMA < 128 only BMA rows are loaded and the others are
// whatever shared memory holds; their accumulator rows are never read.
//
// TMEM: the scales of stage s have columns of their own, rewritten only after the MMAs
// that read them have committed.  Two accumulators of BN columns follow; with BN = 256
// they share OVL columns, and the next tile's MMAs start as soon as the epilogue has read
// those (it reads them first).
#include <atomic>

#include "kernels.cuh"
#include "mx.cuh"

namespace b200moe {

constexpr int MXG_BK = 128;
constexpr int MXG_MAXP = 512;
constexpr int MXG_SF_BYTES = 512;  // scales of 128 rows x 128 columns
constexpr uint64_t kDrainNs = 1000000;

template <int BN, int BMA, int STAGES, bool SWIGLU, int EWG>
struct MxGemmShape {
  static constexpr int A_SLOT = BMA * MXG_BK;             // bytes of a stage's activation rows
  static constexpr int B_SLOT = BN * MXG_BK;              // weights in shared memory (padded form)
  static constexpr int B_TX = BN * MXG_BK / 2;            // bytes the TMA counts for them
  static constexpr int SFB_TILES = BN / 128 > 0 ? BN / 128 : 1;
  static constexpr int SFB_SLOT = SFB_TILES * MXG_SF_BYTES;
  static constexpr int SF_COLS = 4 + 4 * SFB_TILES;       // TMEM columns of a stage's scales
  static constexpr int SF_ALL = SF_COLS * STAGES;
  static constexpr int WANT = 2 * BN + SF_ALL;
  static constexpr int TMEM_COLS = WANT <= 128 ? 128 : WANT <= 256 ? 256 : 512;
  static constexpr int OVL = WANT > TMEM_COLS ? WANT - TMEM_COLS : 0;  // columns both accumulators use
  static constexpr int ACC1 = BN - OVL;
  static constexpr int SF0 = TMEM_COLS - SF_ALL;
  static constexpr int CHUNKS = BN / 64;
  static constexpr int THREADS = 128 + 128 * EWG;
  // the last slot's MMA reads 128 rows from its start: that stays inside the weight ring
  static constexpr int OFF_B = STAGES * A_SLOT;
  static constexpr int OFF_SFA = OFF_B + STAGES * B_SLOT;
  static constexpr int OFF_SFB = OFF_SFA + STAGES * MXG_SF_BYTES;
  static constexpr int OFF_CTRL = OFF_SFB + STAGES * SFB_SLOT;
  static constexpr int CTRL_BYTES = 512 + 2 * (MXG_MAXP + 1) * 4;
  static constexpr int SMEM_BYTES = 1024 + OFF_CTRL + CTRL_BYTES;
  static_assert(BN == 64 || BN == 128 || BN == 256, "BN");
  static_assert(BMA % 32 == 0 && BMA <= 128, "BMA");
  static_assert(OVL <= 64, "the shared columns lie in one chunk");
  static_assert(SF0 >= ACC1 + BN && SF0 % 4 == 0, "TMEM columns");
  static_assert(128 * MXG_BK <= A_SLOT + STAGES * B_SLOT, "the MMA's 128 rows stay in shared memory");
  static_assert((2 * STAGES + 4) * 8 + 16 <= 512, "barriers");
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

template <int BMA>
__device__ __forceinline__ void mx_decode_tile(const int* prefix, const int32_t* off, int P, int tile, int& e, int& m,
                                               int& n) {
  int lo = 0, hi = P - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= tile) lo = mid; else hi = mid - 1;
  }
  e = lo;
  const int local = tile - prefix[e];
  const int mt = (off[e + 1] - off[e] + BMA - 1) / BMA;
  n = local / mt;
  m = local - n * mt;
}

// silu(g) * u with the hardware exponential and reciprocal: a few units in the last place
// of fp32, against the e4m3 rounding of 2^-4 that follows.  -g beyond 88 makes the
// exponential infinite and the result g * 0, as in the limit.
__device__ __forceinline__ float silu_mul_fast(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

template <int BN, int BMA, int STAGES, bool SWIGLU, int EWG>
__global__ void __launch_bounds__(128 + 128 * EWG, 1)
    grouped_gemm_mx_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                           const __grid_constant__ MxGemmParams p) {
  using S = MxGemmShape<BN, BMA, STAGES, SWIGLU, EWG>;
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
  uint64_t* tempty = tfull + 2;       // [2] accumulator read (OVL: [0] alone, shared columns read)
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  int* prefix = reinterpret_cast<int*>(smem + S::OFF_CTRL + 512);  // [P+1] tiles before each expert
  int32_t* off = prefix + (MXG_MAXP + 1);                          // [P+1] row offsets, clamped

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nt = (p.w_rows + BN - 1) / BN;
  pdl_trigger();

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 4 * EWG);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, S::TMEM_COLS);
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
    for (int base = 0; base < p.P; base += 32) {
      const int e = base + lane;
      const int c = e < p.P ? ((off[e + 1] - off[e] + BMA - 1) / BMA) * nt : 0;
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
  const int total_tiles = prefix[p.P];
  const int num_kb = p.K / MXG_BK;
  const int nt128 = p.w_rows / 128;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < total_tiles; tile += gridDim.x) {
        int e, m, n;
        mx_decode_tile<BMA>(prefix, off, p.P, tile, e, m, n);
        const int row_a = off[e] + m * BMA;
        const int row_b = e * p.w_rows + n * BN;
        const uint8_t* sf = p.w_scales + (static_cast<int64_t>(e) * num_kb * nt128 + n * BN / 128) * MXG_SF_BYTES;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag, p.status)) { ok = false; break; }
          mbar_arrive_expect_tx(&full[stage], S::A_SLOT + S::B_TX + S::SFB_SLOT);
          tma_load_2d(sb + stage * S::B_SLOT, &map_b, &full[stage], kb * MXG_BK, row_b);
          tma_load_2d(sa + stage * S::A_SLOT, &map_a, &full[stage], kb * MXG_BK, row_a);
          bulk_load(ssfb + stage * S::SFB_SLOT, sf + static_cast<int64_t>(kb) * nt128 * MXG_SF_BYTES, S::SFB_SLOT,
                    &full[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      // ------------------------------------------------ scales to TMEM, MMAs
      constexpr uint32_t idesc = make_idesc_mx(128, BN);
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < total_tiles; tile += gridDim.x, ++it) {
        const int acc = it & 1;
        int e, m, n;
        mx_decode_tile<BMA>(prefix, off, p.P, tile, e, m, n);
        if (S::OVL > 0) {
          // the previous tile's shared columns are read (and with them, in the epilogue's
          // order, everything of the tile before it)
          if (it > 0 && !mbar_wait(&tempty[0], (it - 1) & 1, abort_flag, p.status)) break;
        } else {
          if (!mbar_wait(&tempty[acc], ((it >> 1) & 1) ^ 1u, abort_flag, p.status)) break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * S::ACC1);
        // a 64-row weight tile is one half of a 128-row scale tile: two of its four columns
        const uint32_t sfb_half = BN == 64 ? static_cast<uint32_t>((n & 1) * 2) : 0u;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full[stage], phase, abort_flag, p.status)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sfa = tmem_base + static_cast<uint32_t>(S::SF0 + stage * S::SF_COLS);
          const uint32_t sfb = sfa + 4;
          tmem_cp_scales(sfa, make_scale_desc(smem_u32(ssfa + stage * MXG_SF_BYTES)));
#pragma unroll
          for (int t = 0; t < S::SFB_TILES; ++t)
            tmem_cp_scales(sfb + 4 * t, make_scale_desc(smem_u32(ssfb + stage * S::SFB_SLOT + t * MXG_SF_BYTES)));
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
        umma_commit(&tfull[acc]);
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // -------------------------------------------------- activation scales
    // Lane l holds rows l, l + 32, ... of the tile; 16 bytes of a row are its scales of
    // four k-blocks, and word j of the four rows is lane l's 16 bytes of k-block j.
    constexpr int R = BMA / 32;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < total_tiles; tile += gridDim.x) {
      int e, m, n;
      mx_decode_tile<BMA>(prefix, off, p.P, tile, e, m, n);
      const uint8_t* src[R];
      bool have[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int row = off[e] + m * BMA + r * 32 + lane;
        have[r] = row < p.rows_cap;
        src[r] = p.a_scales + static_cast<int64_t>(have[r] ? row : 0) * p.lda;
      }
      uint4 next[R];
#pragma unroll
      for (int r = 0; r < R; ++r)
        next[r] = have[r] ? *reinterpret_cast<const uint4*>(src[r]) : make_uint4(0, 0, 0, 0);
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
    const int group = (warp - 4) >> 2;     // takes every EWG-th chunk of 64 columns
    int it = 0;
    for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x, ++it) {
      const int acc = it & 1;
      int e, m, n;
      mx_decode_tile<BMA>(prefix, off, p.P, tile, e, m, n);
      const int left = off[e + 1] - off[e] - m * BMA;   // rows of this tile
      const int r = quarter * 32 + lane;
      const bool warp_has_rows = quarter * 32 < min(left, BMA);
      bool valid = r < min(left, BMA);
      const int64_t grow = static_cast<int64_t>(off[e]) + m * BMA + r;
      int64_t orow = grow;
      if (!SWIGLU && valid && p.out_row_map != nullptr) {
        orow = p.out_row_map[grow];
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
      for (int i = group; i < S::CHUNKS; i += EWG) {
        // the chunk with the shared columns first: the last one of accumulator 0, the
        // first of accumulator 1
        const int ch = (S::OVL > 0 && acc == 0) ? (i == 0 ? S::CHUNKS - 1 : i - 1) : i;
        uint32_t lo[32], hi[32];
        if (warp_has_rows) {
          tmem_ld_32x32b_x32(tbase + ch * 64, lo);
          tmem_ld_32x32b_x32(tbase + ch * 64 + 32, hi);
          tmem_ld_wait();
        }
        if (S::OVL > 0 && i == group) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tempty[0]);
        }
        if (!valid) continue;
        if (SWIGLU) {
          // lo: 32 gates, hi: the ups of the same columns; one MX8 block
          const int col = n * (BN / 2) + ch * 32;
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
          uint4* dst = reinterpret_cast<uint4*>(out_row + col);
          dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
          dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
          out_row[p.N + col / MX_BLOCK] = static_cast<uint8_t>(byte);
        } else {
          uint4* dst = reinterpret_cast<uint4*>(out_row + (n * BN + ch * 64) * 2);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            dst[q] = make_uint4(pack_bf16x2(__uint_as_float(lo[8 * q]), __uint_as_float(lo[8 * q + 1])),
                                pack_bf16x2(__uint_as_float(lo[8 * q + 2]), __uint_as_float(lo[8 * q + 3])),
                                pack_bf16x2(__uint_as_float(lo[8 * q + 4]), __uint_as_float(lo[8 * q + 5])),
                                pack_bf16x2(__uint_as_float(lo[8 * q + 6]), __uint_as_float(lo[8 * q + 7])));
            dst[4 + q] = make_uint4(pack_bf16x2(__uint_as_float(hi[8 * q]), __uint_as_float(hi[8 * q + 1])),
                                    pack_bf16x2(__uint_as_float(hi[8 * q + 2]), __uint_as_float(hi[8 * q + 3])),
                                    pack_bf16x2(__uint_as_float(hi[8 * q + 4]), __uint_as_float(hi[8 * q + 5])),
                                    pack_bf16x2(__uint_as_float(hi[8 * q + 6]), __uint_as_float(hi[8 * q + 7])));
          }
        }
      }
      if (S::OVL == 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[acc]);
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
    tmem_dealloc(tmem_base, S::TMEM_COLS);
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

template <int BN, int BMA, int STAGES, bool SWIGLU, int EWG>
static int run_mx(const MxGemmLaunch& L, cudaStream_t stream) {
  using S = MxGemmShape<BN, BMA, STAGES, SWIGLU, EWG>;
  auto* kern = grouped_gemm_mx_kernel<BN, BMA, STAGES, SWIGLU, EWG>;
  CUtensorMap ma, mb;
  if (make_mx_map(&ma, L.a, L.p.rows_cap, L.p.K, L.p.lda, BMA, false) != 0) return -1;
  if (make_mx_map(&mb, L.w, static_cast<int64_t>(L.p.P) * L.p.w_rows, L.p.K, L.p.K / 2, BN, true) != 0) return -1;
  // at least half the SM's shared memory, so two CTAs never share one SM (each holds
  // its TMEM columns for its whole lifetime)
  const int smem = S::SMEM_BYTES > 120 * 1024 ? S::SMEM_BYTES : 120 * 1024;
  static std::atomic<uint64_t> attr_set_mask{0};  // one bit per device ordinal
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (!(attr_set_mask.load(std::memory_order_acquire) & bit)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -3;
    attr_set_mask.fetch_or(bit, std::memory_order_release);
  }
  const int nt = (L.p.w_rows + BN - 1) / BN;
  const int64_t bound = ((L.p.rows_cap + BMA - 1) / BMA + L.p.P) * static_cast<int64_t>(nt);
  if (bound > 0x7fffffff) return -5;
  const int limit = gemm_grid_limit();
  launch_kernel(kern, dim3(static_cast<unsigned>(bound < limit ? bound : limit)), dim3(S::THREADS), smem, stream, ma, mb,
                L.p);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

template <bool SWIGLU>
static int pick_mx(const MxGemmLaunch& L, cudaStream_t stream) {
  if (L.p.P > MXG_MAXP) return -4;
  const int64_t rows = L.rows_hint > 0 ? L.rows_hint : L.p.rows_cap;
  if (rows <= 32 * static_cast<int64_t>(L.p.P)) return run_mx<64, 32, 14, SWIGLU, 1>(L, stream);
  if (L.p.w_rows % 256 != 0) return run_mx<128, 128, 6, SWIGLU, 1>(L, stream);
  return run_mx<256, 128, 4, SWIGLU, 1>(L, stream);
}

int launch_grouped_mx(const MxGemmLaunch& L, bool swiglu, cudaStream_t stream) {
  return swiglu ? pick_mx<true>(L, stream) : pick_mx<false>(L, stream);
}

}  // namespace b200moe
