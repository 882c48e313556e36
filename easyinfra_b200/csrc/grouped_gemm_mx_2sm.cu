// Grouped expert GEMMs on microscaled operands, prefill form on CTA pairs: the contract,
// formats and weight layout of grouped_gemm_mx.cu, with tcgen05.mma.cta_group::2.
//
// At prefill both operands come from L2, and a 128 x 256 tile pulls 32 KB a k-block into its
// SM (128 rows of 128 bytes, 256 weight rows of 64), about what an SM can draw.  A pair's
// tile is 256 activation rows x 256 weight rows: CTA r loads rows [128 r, 128 r + 128) of
// both, 24 KB a k-block, and the even CTA issues MMAs of M = 256, N = 256, K = 32 that read
// both CTAs' shared memory.  Each CTA holds the scales of its own activation rows and of all
// 256 weight rows in its TMEM; tcgen05.cp by the even CTA copies in both, each from its own
// shared memory.
//
// Roles (256 threads per CTA):
//   warp 0     TMA in both CTAs, completion on the even CTA's full barriers
//   warp 1     TMEM, and in the even CTA scales to TMEM and MMAs, whose commits arrive on the
//              barriers of both CTAs
//   warp 2     activation scales, in both CTAs
//   warps 4..7 epilogue of this CTA's 128 rows
// Accumulators share columns as in grouped_gemm_mx.cu.  Every wait is bounded.
//
// Bound by the tensor cores, at the power limit in a long run: SwiGLU of 32768 rows over 8
// experts of 28672 x 4096 2.48 ms after a pause (3.1 PFLOP/s) and 2.85 at the clock of a
// long run; 82% of the cycles have an MMA in the pipe with K = 4096.  With K = 1408 it is
// 63%: a tile's 11 k-blocks are 5.7 k clocks of MMAs, and the next tile waits about 1.3 k
// more for the shared columns (down of 98304 rows over 64 experts of 2048 x 1408: 272 us,
// 320 in a long run; 403 MB of output are stored in that time).
#include <atomic>

#include "mx_gemm.cuh"

namespace b200moe {

constexpr uint16_t MXP_PAIR_MASK = 0x3;

template <int STAGES>
struct MxPairShape {
  static constexpr int THREADS = 256;
  static constexpr int BMA = 256;                          // activation rows of a pair's tile
  static constexpr int A_SLOT = 128 * MXG_BK;
  static constexpr int B_SLOT = 128 * MXG_BK;              // this CTA's half of the weight rows, padded form
  static constexpr int SFB_SLOT = 2 * MXG_SF_BYTES;
  static constexpr int GROUPS = 3;                         // activation scales: slots of four k-blocks
  static constexpr int TX = 2 * (A_SLOT + 2 * MXG_UNIT_BYTES + SFB_SLOT);  // both CTAs' bytes of a stage
  static constexpr int SF_COLS = 12;
  static constexpr int SF0 = 512 - SF_COLS * STAGES;
  static constexpr int ACC1 = SF0 - MXG_BN;
  static constexpr int OVL = MXG_BN - ACC1;
  static constexpr int OFF_B = STAGES * A_SLOT;
  static constexpr int OFF_SFB = OFF_B + STAGES * B_SLOT;
  static constexpr int OFF_SFA = OFF_SFB + STAGES * SFB_SLOT;
  static constexpr int OFF_CTRL = OFF_SFA + GROUPS * 4 * MXG_SF_BYTES;
  static constexpr int CTRL_BYTES = 256 + 2 * (MXG_MAXP + 1) * 4 + 2 * (THREADS / 32) * 4;
  static constexpr int SMEM_BYTES = 1024 + OFF_CTRL + CTRL_BYTES;
  static_assert(OVL > 0 && OVL <= 64, "the shared columns lie in one chunk of 64");
  static_assert((2 * STAGES + 3 * GROUPS + 3) * 8 + 16 <= 256, "barriers");
  static_assert(SMEM_BYTES > 114 * 1024 && SMEM_BYTES <= 232448, "one CTA per SM");
};

// The tiles of a pair: (expert, n-tile, m-tile of 256 rows) round robin, m fastest.
struct MxPairTiles {
  const int* prefix;
  const int32_t* off;
  int P, pos, end, step;
  int e, row0, rows, n;  // first row and row count (0..128) of this CTA's half

  __device__ __forceinline__ MxPairTiles(const int* prefix_, const int32_t* off_, int P_)
      : prefix(prefix_), off(off_), P(P_), pos(blockIdx.x >> 1), end(prefix_[P_]), step(gridDim.x >> 1), e(0) {}

  __device__ __forceinline__ bool next(int crank) {
    if (pos >= end) return false;
    e = mx_find_expert(prefix, P, pos, e);
    const int local = pos - prefix[e];
    const int all = off[e + 1] - off[e];
    const int mt = (all + 255) / 256;
    n = local / mt;
    const int first = (local - n * mt) * 256 + crank * 128;
    row0 = off[e] + first;
    rows = max(0, min(128, all - first));
    pos += step;
    return true;
  }
};

template <int STAGES, bool SWIGLU>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(256, 1)
    grouped_gemm_mx_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                const __grid_constant__ CUtensorMap map_sfb, const __grid_constant__ MxGemmParams p) {
  using S = MxPairShape<STAGES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sa = smem;
  uint8_t* sb = smem + S::OFF_B;
  uint8_t* ssfb = smem + S::OFF_SFB;
  uint8_t* ssfa = smem + S::OFF_SFA;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::OFF_CTRL);  // even CTA: both CTAs' bytes of a stage
  uint64_t* empty = full + STAGES;                                   // both CTAs: the stage's MMAs are through
  uint64_t* sf_full = empty + STAGES;         // even CTA: both CTAs' activation scales of four k-blocks
  uint64_t* sf_empty = sf_full + S::GROUPS;   // both CTAs: their MMAs are through
  uint64_t* sf_mine = sf_empty + S::GROUPS;   // odd CTA: its own scales are written
  uint64_t* tfull = sf_mine + S::GROUPS;    // [2] both CTAs: accumulator complete
  uint64_t* tread = tfull + 2;        // even CTA: shared columns of the last tile read in both
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tread + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  int* prefix = reinterpret_cast<int*>(smem + S::OFF_CTRL + 256);
  int32_t* off = prefix + (MXG_MAXP + 1);
  int* scan = off + (MXG_MAXP + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int crank = __shfl_sync(0xffffffffu, static_cast<int>(cluster_ctarank()), 0);
  pdl_trigger();

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int g = 0; g < S::GROUPS; ++g) {
      mbar_init(&sf_full[g], 2);
      mbar_init(&sf_empty[g], 1);
      mbar_init(&sf_mine[g], 1);
    }
    mbar_init(&tfull[0], 1);
    mbar_init(&tfull[1], 1);
    mbar_init(tread, 8);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
    tma_prefetch_desc(&map_sfb);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_holder, 512);
    tmem_relinquish_pair();
  }
  cluster_sync_all();  // barriers of both CTAs initialised before any remote arrive or load
  pdl_wait();
  mx_tables<S::THREADS>(p, S::BMA, p.w_rows / MXG_BN, prefix, off, scan);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const int num_kb = p.K / MXG_BK;
  MxPairTiles t(prefix, off, p.P);

  if (warp == 0) {
    if (elect_one()) {
      // ------------------------------------------------ TMA producer (both CTAs)
      const uint32_t full0 = mapa_shared(smem_u32(full), 0);
      const int units = p.w_rows / MXG_UNIT;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      while (ok && t.next(crank)) {
        const int row_b = (t.e * units + 4 * t.n + 2 * crank) * num_kb * MXG_UNIT;
        const int row_sf = t.e * num_kb * (units / 2) + 2 * t.n;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mx_wait(smem_u32(&empty[stage]), phase ^ 1u, abort_flag, p.status)) { ok = false; break; }
          if (crank == 0) mbar_arrive_expect_tx(&full[stage], S::TX);
          const uint32_t fb = full0 + stage * 8;
          uint8_t* dst = sb + stage * S::B_SLOT;
          tma_load_2d_pair(sa + stage * S::A_SLOT, &map_a, fb, kb * MXG_BK, t.row0);
          tma_load_2d_pair(dst, &map_b, fb, 0, row_b + kb * MXG_UNIT);
          tma_load_2d_pair(dst + MXG_UNIT * MXG_BK, &map_b, fb, 0, row_b + (num_kb + kb) * MXG_UNIT);
          tma_load_2d_pair(ssfb + stage * S::SFB_SLOT, &map_sfb, fb, 0, row_sf + kb * (units / 2));
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1 && crank == 0) {
    if (elect_one()) {
      // ------------------------------------------------ scales to TMEM, MMAs (even CTA)
      constexpr uint32_t idesc = make_idesc_mx(256, MXG_BN);
      int stage = 0;
      uint32_t phase = 0;
      int group = 0;
      uint32_t gphase = 0;
      int it = 0;
      bool ok = true;
      for (; ok && t.next(crank); ++it) {
        if (it > 0 && !mx_wait<true>(smem_u32(tread), (it - 1) & 1, abort_flag, p.status)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>((it & 1) * S::ACC1);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mx_wait(smem_u32(&full[stage]), phase, abort_flag, p.status) ||
              ((kb & 3) == 0 && !mx_wait<true>(smem_u32(&sf_full[group]), gphase, abort_flag, p.status))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sfa = tmem_base + static_cast<uint32_t>(S::SF0 + stage * S::SF_COLS);
          const uint32_t sfb = sfa + 4;
          const uint32_t sfb_smem = smem_u32(ssfb + stage * S::SFB_SLOT);
          tmem_cp_scales_pair(sfa, make_scale_desc(smem_u32(ssfa + (group * 4 + (kb & 3)) * MXG_SF_BYTES)));
          tmem_cp_scales_pair(sfb, make_scale_desc(sfb_smem));
          tmem_cp_scales_pair(sfb + 4, make_scale_desc(sfb_smem + MXG_SF_BYTES));
          const uint64_t adesc = make_sw128_kmajor_desc(smem_u32(sa + stage * S::A_SLOT));
          const uint64_t bdesc = make_sw128_kmajor_desc(smem_u32(sb + stage * S::B_SLOT));
#pragma unroll
          for (uint32_t k = 0; k < MXG_BK / MX_BLOCK; ++k)
            umma_mx_pair(d_tmem, adesc + 2ull * k, bdesc + 2ull * k, idesc | (k << 29) | (k << 4), sfa, sfb,
                         (static_cast<uint32_t>(kb) | k) != 0 ? 1u : 0u);
          umma_commit_pair(&empty[stage], MXP_PAIR_MASK);
          if ((kb & 3) == 3 || kb == num_kb - 1) {
            umma_commit_pair(&sf_empty[group], MXP_PAIR_MASK);
            if (++group == S::GROUPS) { group = 0; gphase ^= 1u; }
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        umma_commit_pair(&tfull[it & 1], MXP_PAIR_MASK);
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // -------------------------------------------------- activation scales (both CTAs)
    // Written and signalled by fours.  The odd CTA's signal has to release at cluster scope,
    // which waits for all that its warp has outstanding, this warp's loads among it; warp 3,
    // which has nothing outstanding, passes it on (once a k-block and from here, the Mixtral
    // SwiGLU product took 5.4 ms instead of 3.0).
    MxRowScales<4> sc;
    int group = 0;
    uint32_t gphase = 0;
    bool ok = true;
    while (ok && t.next(crank)) {
      sc.start(p, t.rows > 0 ? t.row0 : 0, t.rows, lane);
      for (int kb0 = 0; ok && kb0 < num_kb; kb0 += 4) {
        sc.advance(kb0, num_kb);
        int go = 0;
        if (lane == 0) go = mx_wait(smem_u32(&sf_empty[group]), gphase ^ 1u, abort_flag, p.status) ? 1 : 0;
        ok = __shfl_sync(0xffffffffu, go, 0) != 0;
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint4*>(ssfa + (group * 4 + j) * MXG_SF_BYTES + lane * 16) = sc.block(j);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(crank == 0 ? &sf_full[group] : &sf_mine[group]);
        if (++group == S::GROUPS) { group = 0; gphase ^= 1u; }
      }
    }
  } else if (warp == 3 && crank == 1) {
    if (elect_one()) {
      // ------------------------------------------------ the odd CTA's scales are there
      const uint32_t sf_full0 = mapa_shared(smem_u32(sf_full), 0);
      int group = 0;
      uint32_t gphase = 0;
      bool ok = true;
      while (ok && t.next(crank)) {
        for (int kb0 = 0; kb0 < num_kb; kb0 += 4) {
          if (!mx_wait(smem_u32(&sf_mine[group]), gphase, abort_flag, p.status)) { ok = false; break; }
          mbar_arrive_remote(sf_full0 + group * 8);
          if (++group == S::GROUPS) { group = 0; gphase ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // -------------------------------------------------- epilogue (both CTAs)
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t tread0 = mapa_shared(smem_u32(tread), 0);
    const bool wide = ((reinterpret_cast<uintptr_t>(p.out) | static_cast<uintptr_t>(p.ldo)) & 31u) == 0;
    for (int it = 0; t.next(crank); ++it) {
      const int acc = it & 1;
      const bool warp_has_rows = quarter * 32 < t.rows;
      bool valid = r < t.rows;
      int64_t orow = static_cast<int64_t>(t.row0) + r;
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
      uint8_t* out_row = static_cast<uint8_t*>(p.out) + orow * p.ldo;
      uint32_t bytes = 0;
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        const int ch = acc != 0 ? i : (i + 3) & 3;  // the chunk with the shared columns first
        uint32_t lo[32], hi[32];
        if (warp_has_rows) {
          tmem_ld_32x32b_x32(tbase + ch * 64, lo);
          tmem_ld_32x32b_x32(tbase + ch * 64 + 32, hi);
          tmem_ld_wait();
        }
        if (i == 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote_relaxed(tread0);
        }
        if (!valid) continue;
        if (SWIGLU) {
          uint32_t w[8];
          bytes |= mx_swiglu_block(lo, hi, w) << (8 * ch);
          store_32(out_row + (4 * t.n + ch) * 32, w, wide);
        } else {
          store_bf16_64(out_row + (4 * t.n + ch) * 128, lo, hi, wide);
        }
      }
      if (SWIGLU && valid) *reinterpret_cast<uint32_t*>(out_row + p.N + 4 * t.n) = bytes;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*abort_flag) mx_drain();
  cluster_sync_all();  // neither CTA frees TMEM or exits while the pair still works
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

template <int STAGES, bool SWIGLU>
static int run_mx_pair(const MxGemmLaunch& L, cudaStream_t stream) {
  using S = MxPairShape<STAGES>;
  constexpr auto* kern = grouped_gemm_mx_pair_kernel<STAGES, SWIGLU>;
  CUtensorMap ma, mb, msf;
  if (make_mx_maps(&ma, &mb, L, 128) != 0) return -1;
  // scale tiles as rows of 128 words
  const cuuint64_t dims[2] = {128, static_cast<cuuint64_t>(L.p.P) * (L.p.K / MXG_BK) * (L.p.w_rows / 128)};
  const cuuint64_t strides[1] = {MXG_SF_BYTES};
  const cuuint32_t box[2] = {128, 2};
  if (encode_tma_map_2d(&msf, CU_TENSOR_MAP_DATA_TYPE_UINT32, L.p.w_scales, dims, strides, box,
                        CU_TENSOR_MAP_SWIZZLE_NONE) != 0)
    return -1;
  if (!mx_set_smem<S::SMEM_BYTES, kern>()) return -3;
  const int64_t work = ((L.p.rows_cap + 255) / 256 + L.p.P) * static_cast<int64_t>(L.p.w_rows / MXG_BN);
  if (work > 0x7fffffff) return -5;
  const int limit = gemm_grid_limit() / 2;
  const unsigned pairs = static_cast<unsigned>(work < limit ? work : limit);
  launch_kernel(kern, dim3(2 * pairs), dim3(S::THREADS), S::SMEM_BYTES, stream, ma, mb, msf, L.p);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int launch_grouped_mx_pair(const MxGemmLaunch& L, bool swiglu, cudaStream_t stream) {
  return swiglu ? run_mx_pair<5, true>(L, stream) : run_mx_pair<5, false>(L, stream);
}

}  // namespace b200moe
