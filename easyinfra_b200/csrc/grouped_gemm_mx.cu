// Grouped expert GEMMs on microscaled operands: MX8 activation rows (e4m3) times MX4
// weights (e2m1), scaled and accumulated in fp32 inside the tensor cores
// (tcgen05.mma kind::mxf8f6f4 with block scales, mx.cuh for the formats):
//   swiglu  act = MX8(silu(x Wg^T) * (x Wu^T))     down  y = bf16(act Wd^T)
// for every expert e and its rows [off[e], off[e+1]).
//
// A product of two elements has at most six significant bits.  While the two scales' exponents
// add up to between -116 and 116 it is an exact normal number of fp32 with them, and the result
// is the fp32 sum over K of the values that the rows and the weights stand for.  Further out
// (rows or weights of about 2^-58 and 2^58 both) products leave fp32's range.
//
// Weights are laid out once (MX4 product layout), so that a CTA streams them in order:
//   elements  [P, w_rows/64, K/128, 64, 64] bytes: units of 64 weight rows, each its
//             k-blocks of 128 one after the other, 4 KB apiece; for swiglu the rows of
//             gate and up are interleaved by 32 first (32 gate rows, then the 32 up rows of
//             the same columns), so that a unit's 64 accumulator columns hold 32 gates and
//             their 32 ups, and one output block of 32 (one MX8 scale) belongs to one thread
//   scales    [P, K/128, w_rows/128, 512] bytes: for 128 rows x 128 columns the 32 x 16
//             bytes that tcgen05.cp copies to TMEM (byte (r % 32) * 16 + (r / 32) * 4 + k
//             is row r's scale of its k-th 32 columns); a tile's two are adjacent
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
// One persistent CTA per SM takes tiles (expert, n-tile of 4 units, m-tile of 128 rows) round
// robin, m fastest, so that the m-tiles of a weight n-tile run together and share it
// through L2.  This is the form for the middle: few rows per expert stream the weights
// through grouped_gemm_mx_wm.cu, many run on CTA pairs (grouped_gemm_mx_2sm.cu).
//
// TMEM: the scales of stage s have columns of their own, rewritten only after the MMAs
// that read them have committed.  Two accumulators of 256 columns follow that share OVL
// columns, and the next tile's MMAs start as soon as the epilogue has read those (it reads
// them first).
//
// Measured: SwiGLU of 6006 rows over 64 experts of 2816 x 2048 51 us (4.2 TB/s over the
// weights and rows, tensor pipe active 44% of the cycles; 57 us in a long run).  Neither is
// full, and which of the producer, the issuer and the epilogue the others wait for has not been
// counted.  Half of a stage's 32 KB of weights in shared memory is padding, which leaves room
// for four stages; rows are padded to 128.
#include <atomic>

#include "mx_gemm.cuh"

namespace b200moe {

template <int STAGES>
struct MxGemmShape {
  static constexpr int BMA = 128;                         // activation rows of a tile
  static constexpr int THREADS = 256;
  static constexpr int A_SLOT = BMA * MXG_BK;             // bytes of a stage's activation rows
  static constexpr int B_SLOT = MXG_BN * MXG_BK;          // weights in shared memory (padded form)
  static constexpr int SFB_SLOT = 2 * MXG_SF_BYTES;
  static constexpr int SF_COLS = 12;                      // TMEM columns of a stage's scales: 4 + 2 * 4
  static constexpr int SF0 = 512 - SF_COLS * STAGES;
  static constexpr int ACC1 = SF0 - MXG_BN;               // accumulator 0 is at column 0
  static constexpr int OVL = MXG_BN - ACC1;               // columns both accumulators use
  static constexpr int OFF_B = STAGES * A_SLOT;
  static constexpr int OFF_SFA = OFF_B + STAGES * B_SLOT;
  static constexpr int OFF_SFB = OFF_SFA + STAGES * MXG_SF_BYTES;
  static constexpr int OFF_CTRL = OFF_SFB + STAGES * SFB_SLOT;
  static constexpr int CTRL_BYTES = 256 + 2 * (MXG_MAXP + 1) * 4 + 2 * (THREADS / 32) * 4;
  static constexpr int SMEM_BYTES = 1024 + OFF_CTRL + CTRL_BYTES;
  static_assert(OVL > 0 && OVL <= 64, "the shared columns lie in one chunk of 64");
  static_assert(SF0 % 4 == 0, "TMEM columns");
  static_assert((2 * STAGES + 3) * 8 + 16 <= 256, "barriers");
  static_assert(SMEM_BYTES <= 232448, "shared memory");
};

// The tiles of a CTA, in order; every role walks its own copy.
struct MxTiles {
  const int* prefix;    // [P + 1] tiles before each expert
  const int32_t* off;   // [P + 1] rows
  int P, units;         // units of 64 weight rows per expert
  int pos, end;
  int e, row0, rows;    // expert, first activation row, rows of the tile (at most 128)
  int n0, nu;           // first unit, units

  __device__ __forceinline__ MxTiles(const int* prefix_, const int32_t* off_, int P_, int units_)
      : prefix(prefix_), off(off_), P(P_), units(units_), pos(blockIdx.x), end(prefix_[P_]), e(0) {}

  __device__ __forceinline__ bool next() {
    if (pos >= end) return false;
    e = mx_find_expert(prefix, P, pos, e);
    const int local = pos - prefix[e];
    const int all = off[e + 1] - off[e];
    const int mt = (all + 127) / 128;
    const int n = local / mt, m = local - n * mt;
    n0 = 4 * n;
    nu = min(4, units - n0);
    row0 = off[e] + m * 128;
    rows = min(128, all - m * 128);
    pos += gridDim.x;
    return true;
  }
};

template <int STAGES, bool SWIGLU>
__global__ void __launch_bounds__(256, 1)
    grouped_gemm_mx_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                           const __grid_constant__ MxGemmParams p) {
  using S = MxGemmShape<STAGES>;
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
  int* scan = off + (MXG_MAXP + 1);                                // [2 * warps]

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
  mx_tables<S::THREADS>(p, S::BMA, (units + 3) / 4, prefix, off, scan);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const int num_kb = p.K / MXG_BK;
  MxTiles t(prefix, off, p.P, units);

  if (warp == 0) {
    if (elect_one()) {
      // ------------------------------------------------ TMA producer
      const int nt128 = units / 2;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      while (ok && t.next()) {
        const int row_b = (t.e * units + t.n0) * num_kb * MXG_UNIT;
        const int sf0 = t.n0 >> 1;
        const uint32_t sf_bytes = (t.nu >> 1) * MXG_SF_BYTES;  // units are even in number
        const uint8_t* sf = p.w_scales + (static_cast<int64_t>(t.e) * num_kb * nt128 + sf0) * MXG_SF_BYTES;
        const uint32_t tx = S::A_SLOT + t.nu * MXG_UNIT_BYTES + sf_bytes;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mx_wait(smem_u32(&empty[stage]), phase ^ 1u, abort_flag, p.status)) { ok = false; break; }
          uint64_t* bar = &full[stage];
          mbar_arrive_expect_tx(bar, tx);
          uint8_t* dst = sb + stage * S::B_SLOT;
          for (int u = 0; u < t.nu; ++u)
            tma_load_2d(dst + u * (MXG_UNIT * MXG_BK), &map_b, bar, 0, row_b + (u * num_kb + kb) * MXG_UNIT);
          tma_load_2d(sa + stage * S::A_SLOT, &map_a, bar, kb * MXG_BK, t.row0);
          bulk_load(ssfb + stage * S::SFB_SLOT, sf + static_cast<int64_t>(kb) * nt128 * MXG_SF_BYTES, sf_bytes, bar);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      // ------------------------------------------------ scales to TMEM, MMAs
      // One loop over the k-blocks of all tiles, unrolled over the ring, so that every address
      // of a stage is a base plus a constant.
      const uint32_t full_a = smem_u32(full), empty_a = smem_u32(empty);
      const uint64_t a0 = make_sw128_kmajor_desc(smem_u32(sa)), b0 = make_sw128_kmajor_desc(smem_u32(sb));
      const uint64_t sfa0 = make_scale_desc(smem_u32(ssfa)), sfb0 = make_scale_desc(smem_u32(ssfb));
      const uint32_t sf_tmem = tmem_base + S::SF0;
      uint32_t phase = 0, idesc = 0, d_tmem = 0;
      bool two = false;
      int kb = 0, it = 0;
      bool more = t.next();
      while (more) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) {
          if (more && kb == 0) {
            // the previous tile's shared columns are read (and with them, in the epilogue's
            // order, everything of the tile before it)
            more = it == 0 || mx_wait(smem_u32(tread), (it - 1) & 1, abort_flag, p.status);
            tc_fence_after();
            idesc = make_idesc_mx(128, t.nu * MXG_UNIT);
            d_tmem = tmem_base + static_cast<uint32_t>((it & 1) * S::ACC1);
            two = t.nu > 2;
          }
          if (more && (more = mx_wait(full_a + 8 * s, phase, abort_flag, p.status))) {
            tc_fence_after();
            const uint32_t sfa = sf_tmem + s * S::SF_COLS, sfb = sfa + 4;
            tmem_cp_scales(sfa, sfa0 + s * (MXG_SF_BYTES >> 4));
            tmem_cp_scales(sfb, sfb0 + s * (S::SFB_SLOT >> 4));
            if (two) tmem_cp_scales(sfb + 4, sfb0 + (s * S::SFB_SLOT + MXG_SF_BYTES >> 4));
#pragma unroll
            for (uint32_t k = 0; k < MXG_BK / MX_BLOCK; ++k)  // 32 bytes of K each; byte k of the scale words
              umma_mx(d_tmem, a0 + s * (S::A_SLOT >> 4) + 2 * k, b0 + s * (S::B_SLOT >> 4) + 2 * k,
                      idesc | (k << 29) | (k << 4), sfa, sfb, k != 0 ? 1u : kb != 0 ? 1u : 0u);
            umma_commit_at(empty_a + 8 * s);
            if (++kb == num_kb) {
              umma_commit(&tfull[it & 1]);
              kb = 0;
              ++it;
              more = t.next();
            }
          }
        }
        phase ^= 1u;
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // -------------------------------------------------- activation scales
    MxRowScales<S::BMA / 32> sc;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    while (ok && t.next()) {
      sc.start(p, t.row0, t.rows, lane);
      for (int kb0 = 0; ok && kb0 < num_kb; kb0 += 4) {
        sc.advance(kb0, num_kb);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (kb0 + j < num_kb && ok) {
            int go = 0;
            if (lane == 0) go = mx_wait(smem_u32(&empty[stage]), phase ^ 1u, abort_flag, p.status) ? 1 : 0;
            ok = __shfl_sync(0xffffffffu, go, 0) != 0;
            if (ok) {
              *reinterpret_cast<uint4*>(ssfa + stage * MXG_SF_BYTES + lane * 16) = sc.block(j);
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
      if (lane == 0) ok = mx_wait(smem_u32(&tfull[acc]), (it >> 1) & 1, abort_flag, p.status) ? 1 : 0;
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
          uint32_t w[8];
          const uint32_t byte = mx_swiglu_block(lo, hi, w);
          store_32(out_row + col, w, wide);
          out_row[p.N + col / MX_BLOCK] = static_cast<uint8_t>(byte);
        } else {
          store_bf16_64(out_row + (t.n0 + ch) * 128, lo, hi, wide);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) mx_drain();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// ------------------------------------------------------------------ host side

int make_mx_maps(CUtensorMap* ma, CUtensorMap* mb, const MxGemmLaunch& L, int box_rows) {
  const cuuint64_t adims[2] = {static_cast<cuuint64_t>(L.p.K), static_cast<cuuint64_t>(L.p.rows_cap)};
  const cuuint64_t astr[1] = {static_cast<cuuint64_t>(L.p.lda)};
  const cuuint32_t abox[2] = {MXG_BK, static_cast<cuuint32_t>(box_rows)};
  const cuuint64_t bdims[2] = {MXG_BK, static_cast<cuuint64_t>(L.p.P) * L.p.w_rows * (L.p.K / MXG_BK)};
  const cuuint64_t bstr[1] = {MXG_BK / 2};
  const cuuint32_t bbox[2] = {MXG_BK, MXG_UNIT};
  if (encode_tma_map_2d(ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, L.a, adims, astr, abox) != 0) return -1;
  return encode_tma_map_2d(mb, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, L.p.w, bdims, bstr, bbox) != 0 ? -1 : 0;
}

template <int STAGES, bool SWIGLU>
static int run_mx(const MxGemmLaunch& L, int64_t work, cudaStream_t stream) {
  using S = MxGemmShape<STAGES>;
  constexpr auto* kern = grouped_gemm_mx_kernel<STAGES, SWIGLU>;
  CUtensorMap ma, mb;
  if (make_mx_maps(&ma, &mb, L, S::BMA) != 0) return -1;
  static_assert(S::SMEM_BYTES > 114 * 1024, "one CTA per SM: it holds all of the SM's TMEM");
  if (!mx_set_smem<S::SMEM_BYTES, kern>()) return -3;
  const int limit = gemm_grid_limit();
  launch_kernel(kern, dim3(static_cast<unsigned>(work < limit ? work : limit)), dim3(S::THREADS), S::SMEM_BYTES,
                stream, ma, mb, L.p);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

// Kernel by the average rows of an expert.  SwiGLU of 64 experts of 2816 x 2048, us in a long
// run, even routing (Zipf): weights as A / tiles at 16 rows 40 / 48 (43 / 48), 48 rows
// 43 / 50 (50 / 56), 56 rows 45 / 50 (54 / 56), 64 rows 56 / 51 (55 / 57), 96 rows 74 / 52
// (72 / 64); tiles / pairs at 256 rows 107 / 112, 768 rows 252 / 257 (256 / 254), 1536 rows
// 524 / 511 (528 / 482), and of 128 experts of 1536 x 2048 at 768 rows 291 / 288 (290 / 263).
constexpr int64_t kWmRows = 56, kPairRows = 768;

int launch_grouped_mx(const MxGemmLaunch& L, bool swiglu, cudaStream_t stream) {
  if (L.p.P > MXG_MAXP) return -4;
  const int64_t rows = L.rows_hint > 0 ? L.rows_hint : L.p.rows_cap;
  const int64_t P = L.p.P, nt = (L.p.w_rows + MXG_BN - 1) / MXG_BN;
  if (rows <= kWmRows * P && mx_wm_work(L) <= 0x7fffffff) return launch_grouped_mx_wm(L, swiglu, stream);
  const int64_t work = ((L.p.rows_cap + 127) / 128 + P) * nt;
  if (work > 0x7fffff00) return -5;  // a CTA's position passes the last tile by up to its stride, the grid
  if (rows >= kPairRows * P && L.p.w_rows % MXG_BN == 0) return launch_grouped_mx_pair(L, swiglu, stream);
  return swiglu ? run_mx<4, true>(L, work, stream) : run_mx<4, false>(L, work, stream);
}

}  // namespace b200moe
