// Grouped expert GEMMs on microscaled operands, few rows per expert (decode): the contract,
// formats and weight layout of grouped_gemm_mx.cu with the operands exchanged.  The weights
// are the MMA's A (M = 128 weight rows), the tokens its B, so that the tensor cores do
// N = 16..64 columns of work per 128 weight rows instead of 128 rows of mostly nothing:
// Qwen3's 64-token SwiGLU product takes 37 us in a long run, and 50 with the tokens as A
// (grouped_gemm_mx.cu, forced by the row hint).
//
// The launch is bound by the stream of weights from HBM.  A stage holds one k-block (128
// columns) of up to 4 units of 64 weight rows, 16 KB in memory and twice that in shared
// memory (padded 4-bit form), and of up to 64 tokens; five stages are in flight.  Every CTA
// gets an equal, contiguous share of all (expert, 64-row m-tile, unit) in that order, cut
// into even tiles of up to 4 units: whole n-tiles of 256 rows would leave the last round of
// CTAs up to 17% short of work (896 tiles on 148 SMs at 8 experts of 28672 rows).
//
// Measured: 64 tokens x 8 of 128 experts of 1536 x 2048 35 us (4.8 TB/s of weights; the
// copy rate would take 25.5), 64 tokens x 2 of 8 experts of 28672 x 4096 85 us (5.9 TB/s;
// 76.4).  About 7 us of every launch pass before the stream of weights is at its rate and
// after the last tile.  Taking work out of a copy shows how little else is left: without
// the epilogue 33.0 us, with half of the MMAs 33.8.
//
// Roles (256 threads): warp 0 TMA, warp 1 scales to TMEM and MMAs, warp 2 token scales,
// warps 4..7 epilogue.  Accumulator lanes are weight rows: 16 tokens at a time go through
// shared memory as [128 rows][16 tokens], so that a thread gets consecutive output columns
// of one token; the four threads that share an MX8 block find its largest value by
// shuffles.  TMEM: two accumulators of 2 x 64 columns, and 16 columns of scales a stage.
#include <atomic>

#include "mx_gemm.cuh"
#include "mx_share.cuh"

namespace b200moe {

template <int STAGES>
struct MxWmShape {
  static constexpr int THREADS = 256;
  static constexpr int TOK = 64;                           // tokens of a tile
  static constexpr int X_BOX = 16;                         // tokens a TMA load brings
  static constexpr int W_SLOT = MXG_BN * MXG_BK;           // weights of a stage (padded form)
  static constexpr int X_SLOT = TOK * MXG_BK;
  static constexpr int SFW_SLOT = 3 * MXG_SF_BYTES;        // 4 units touch up to 3 scale tiles
  static constexpr int SF_COLS = 16;                       // 3 * 4 + 4
  static constexpr int SF0 = 512 - SF_COLS * STAGES;
  static constexpr int STG_LD = 17;                        // floats between staged weight rows
  static constexpr int OFF_X = STAGES * W_SLOT;
  static constexpr int OFF_SFW = OFF_X + STAGES * X_SLOT;
  static constexpr int OFF_SFX = OFF_SFW + STAGES * SFW_SLOT;
  static constexpr int OFF_STG = OFF_SFX + STAGES * MXG_SF_BYTES;
  static constexpr int OFF_CTRL = OFF_STG + 128 * STG_LD * 4;
  static constexpr int CTRL_BYTES = 256 + 2 * (MXG_MAXP + 1) * 4 + 2 * (THREADS / 32) * 4;
  static constexpr int SMEM_BYTES = 1024 + OFF_CTRL + CTRL_BYTES;
  static_assert(SF0 >= 4 * TOK, "TMEM columns");
  static_assert((2 * STAGES + 4) * 8 + 16 <= 256, "barriers");
  static_assert(SMEM_BYTES > 114 * 1024 && SMEM_BYTES <= 232448, "one CTA per SM: it holds all of the SM's TMEM");
};

// The tiles of a CTA, in order; every role walks its own copy.
struct MxWmTiles {
  const int* prefix;    // [P + 1] units before each expert
  const int32_t* off;   // [P + 1] rows
  int P, units;         // units of 64 weight rows per expert
  int pos, end;
  int e, row0, rows;    // expert, first token row, rows of the tile (at most 64)
  int n0, nu;           // first unit, units
  int left, part, more; // of this CTA's share in the m-tile: units to come, parts of `part` units, `more` of part + 1

  // Called by whole warps.
  __device__ __forceinline__ MxWmTiles(const int* prefix_, const int32_t* off_, int P_, int units_)
      : prefix(prefix_), off(off_), P(P_), units(units_), e(0), n0(0), nu(0), left(0), part(0), more(0) {
    const MxShare s = mx_share(prefix[P], units, gridDim.x, blockIdx.x);
    pos = s.pos;
    end = s.end;
    // the first expert: two ballots instead of a chain of dependent reads
    const int lane = threadIdx.x & 31, step = (P + 31) / 32;
    const unsigned coarse = __ballot_sync(0xffffffffu, lane * step < P && prefix[min(lane * step, P)] <= pos);
    const int lo = max(31 - __clz(coarse), 0) * step;
    const unsigned fine = __ballot_sync(0xffffffffu, lane < step && lo + lane < P && prefix[min(lo + lane, P)] <= pos);
    e = min(lo + max(31 - __clz(fine), 0), P - 1);
  }

  __device__ __forceinline__ bool next() {
    if (left == 0) {
      if (pos >= end) return false;
      e = mx_find_expert(prefix, P, pos, e);
      const int local = pos - prefix[e];
      const int m = local / units;
      n0 = local - m * units;
      row0 = off[e] + m * 64;
      rows = min(64, off[e + 1] - row0);
      // even parts of at most 4 units: a last tile of one unit would keep a quarter of the
      // bytes in flight
      left = min(units - n0, end - pos);
      const int parts = (left + 3) >> 2;
      part = left / parts;
      more = left - part * parts;
    } else {
      n0 += nu;
    }
    nu = part + (more > 0 ? 1 : 0);
    --more;
    left -= nu;
    pos += nu;
    return true;
  }
};

template <int STAGES, bool SWIGLU>
__global__ void __launch_bounds__(256, 1)
    grouped_gemm_mx_wm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                              const __grid_constant__ MxGemmParams p) {
  using S = MxWmShape<STAGES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sw = smem;
  uint8_t* sx = smem + S::OFF_X;
  uint8_t* ssfw = smem + S::OFF_SFW;
  uint8_t* ssfx = smem + S::OFF_SFX;
  float* stg = reinterpret_cast<float*>(smem + S::OFF_STG);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::OFF_CTRL);  // TMA bytes + the token scales
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;   // [2] accumulator complete
  uint64_t* tread = tfull + 2;        // [2] accumulator read
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tread + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  volatile int* tile_ok = reinterpret_cast<volatile int*>(tmem_holder + 2);
  int* prefix = reinterpret_cast<int*>(smem + S::OFF_CTRL + 256);
  int32_t* off = prefix + (MXG_MAXP + 1);
  int* scan = off + (MXG_MAXP + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int units = p.w_rows / MXG_UNIT;
  pdl_trigger();

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tread[a], 4);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_w);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, 512);
    tmem_relinquish();
  }
  pdl_wait();  // inputs of this launch are complete and visible from here on
  mx_tables<S::THREADS>(p, S::TOK, units, prefix, off, scan);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const int num_kb = p.K / MXG_BK;
  MxWmTiles t(prefix, off, p.P, units);

  if (warp == 0) {
    if (elect_one()) {
      // ------------------------------------------------ TMA producer
      const uint64_t stream_once = l2_policy_evict_first();
      const int nt128 = units / 2;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      while (ok && t.next()) {
        const int x_loads = (t.rows + S::X_BOX - 1) / S::X_BOX;
        const int row_w = (t.e * units + t.n0) * num_kb * MXG_UNIT;
        const int sf0 = t.n0 >> 1;
        const uint32_t sf_bytes = (((t.n0 + t.nu - 1) >> 1) - sf0 + 1) * MXG_SF_BYTES;
        const uint8_t* sf = p.w_scales + (static_cast<int64_t>(t.e) * num_kb * nt128 + sf0) * MXG_SF_BYTES;
        const uint32_t tx = x_loads * (S::X_BOX * MXG_BK) + t.nu * MXG_UNIT_BYTES + sf_bytes;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mx_wait(smem_u32(&empty[stage]), phase ^ 1u, abort_flag, p.status)) { ok = false; break; }
          uint64_t* bar = &full[stage];
          mbar_arrive_expect_tx(bar, tx);
          uint8_t* dst = sw + stage * S::W_SLOT;
          for (int u = 0; u < t.nu; ++u)
            tma_load_2d_hint(dst + u * (MXG_UNIT * MXG_BK), &map_w, bar, 0, row_w + (u * num_kb + kb) * MXG_UNIT,
                             stream_once);
          for (int i = 0; i < x_loads; ++i)
            tma_load_2d(sx + stage * S::X_SLOT + i * (S::X_BOX * MXG_BK), &map_x, bar, kb * MXG_BK,
                        t.row0 + i * S::X_BOX);
          bulk_load(ssfw + stage * S::SFW_SLOT, sf + static_cast<int64_t>(kb) * nt128 * MXG_SF_BYTES, sf_bytes, bar);
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
      const uint64_t w0 = make_sw128_kmajor_desc(smem_u32(sw)), x0 = make_sw128_kmajor_desc(smem_u32(sx));
      const uint64_t sfw0 = make_scale_desc(smem_u32(ssfw)), sfx0 = make_scale_desc(smem_u32(ssfx));
      const uint32_t sf_tmem = tmem_base + S::SF0;
      uint32_t phase = 0, idesc = 0, d_tmem = 0, half = 0;
      int sf_tiles = 0;
      bool two = false;
      int kb = 0, it = 0;
      bool more = t.next();
      while (more) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) {
          if (more && kb == 0) {
            // the accumulator's last tile (two tiles ago) is read
            more = it < 2 || mx_wait(smem_u32(&tread[it & 1]), ((it >> 1) - 1) & 1, abort_flag, p.status);
            tc_fence_after();
            idesc = make_idesc_mx_wm(128, (t.rows + 15) & ~15);
            d_tmem = tmem_base + static_cast<uint32_t>((it & 1) * 2 * S::TOK);
            half = static_cast<uint32_t>((t.n0 & 1) * 2);  // an odd first unit: second half of a scale tile
            sf_tiles = ((t.n0 + t.nu - 1) >> 1) - (t.n0 >> 1) + 1;
            two = t.nu > 2;  // two blocks of 128 weight rows
          }
          if (more && (more = mx_wait(full_a + 8 * s, phase, abort_flag, p.status))) {
            tc_fence_after();
            const uint32_t sfx = sf_tmem + s * S::SF_COLS, sfw = sfx + 4;
            tmem_cp_scales(sfx, sfx0 + s * (MXG_SF_BYTES >> 4));
            tmem_cp_scales(sfw, sfw0 + s * (S::SFW_SLOT >> 4));
            if (sf_tiles > 1) tmem_cp_scales(sfw + 4, sfw0 + ((s * S::SFW_SLOT + MXG_SF_BYTES) >> 4));
            if (sf_tiles > 2) tmem_cp_scales(sfw + 8, sfw0 + ((s * S::SFW_SLOT + 2 * MXG_SF_BYTES) >> 4));
#pragma unroll
            for (uint32_t k = 0; k < MXG_BK / MX_BLOCK; ++k) {  // 32 bytes of K each; byte k of the scale words
              const uint32_t id = idesc | (k << 29) | (k << 4);
              const uint32_t acc = k != 0 ? 1u : kb != 0 ? 1u : 0u;
              const uint64_t wk = w0 + s * (S::W_SLOT >> 4) + 2 * k, xk = x0 + s * (S::X_SLOT >> 4) + 2 * k;
              umma_mx(d_tmem, wk, xk, id, sfw + half, sfx, acc);
              if (two) umma_mx(d_tmem + S::TOK, wk + (128 * MXG_BK >> 4), xk, id, sfw + 4 + half, sfx, acc);
            }
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
    // -------------------------------------------------- token scales
    MxRowScales<S::TOK / 32> sc;
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
              *reinterpret_cast<uint4*>(ssfx + stage * MXG_SF_BYTES + lane * 16) = sc.block(j);
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
    const int e = threadIdx.x - 128;
    const bool wide = ((reinterpret_cast<uintptr_t>(p.out) | static_cast<uintptr_t>(p.ldo)) & 31u) == 0;
    for (int it = 0; t.next(); ++it) {
      const int acc = it & 1;
      // one thread waits; all four warps learn the outcome at the barrier, so that none is
      // left waiting at a later one
      if (e == 0) *tile_ok = mx_wait(smem_u32(&tfull[acc]), (it >> 1) & 1, abort_flag, p.status) ? 1 : 0;
      epi_sync();
      if (*tile_ok == 0) break;
      tc_fence_after();
      const int chunks = (t.rows + 15) >> 4, blocks = (t.nu + 1) >> 1;
      for (int h = 0; h < blocks; ++h) {
        for (int c = 0; c < chunks; ++c) {
          uint32_t v[16];
          tmem_ld_32x32b_x16(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                                 static_cast<uint32_t>((acc * 2 + h) * S::TOK + c * 16),
                             v);
          tmem_ld_wait();
          if (h == blocks - 1 && c == chunks - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tread[acc]);
          }
          float* mine = stg + e * S::STG_LD;
#pragma unroll
          for (int j = 0; j < 16; ++j) mine[j] = __uint_as_float(v[j]);
          epi_sync();
          if (SWIGLU) {
            // (unit, token, quarter of the block): 8 columns of one token's MX8 block
            const int u = quarter >> 1, tok = (quarter & 1) * 8 + (lane & 7), s = lane >> 3;
            const float* g = stg + (64 * u + 8 * s) * S::STG_LD + tok;
            float a[8];
            uint32_t amax = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              a[j] = silu_mul_fast(g[j * S::STG_LD], g[(32 + j) * S::STG_LD]);
              amax = max(amax, __float_as_uint(a[j]) & 0x7fffffffu);
            }
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 8));
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 16));
            const uint32_t byte = mx8_scale_byte(amax);
            const float inv = mx_inverse_scale(byte);
            if (2 * h + u < t.nu && c * 16 + tok < t.rows) {
              uint8_t* row = static_cast<uint8_t*>(p.out) + static_cast<int64_t>(t.row0 + c * 16 + tok) * p.ldo;
              const int blk = t.n0 + 2 * h + u;
              *reinterpret_cast<uint2*>(row + blk * 32 + 8 * s) =
                  make_uint2(cvt_e4m3x4(a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv),
                             cvt_e4m3x4(a[4] * inv, a[5] * inv, a[6] * inv, a[7] * inv));
              if (s == 0) row[p.N + blk] = static_cast<uint8_t>(byte);
            }
          } else {
            // (token, 16 columns)
            const int tok = e & 15, seg = e >> 4;
            if (2 * h + (seg >> 2) < t.nu && c * 16 + tok < t.rows) {
              int64_t orow = t.row0 + c * 16 + tok;
              if (p.out_row_map != nullptr) orow = p.out_row_map[orow];
              if (orow >= 0 && orow < p.out_rows) {
                const float* f = stg + seg * 16 * S::STG_LD + tok;
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = pack_bf16x2(f[2 * j * S::STG_LD], f[(2 * j + 1) * S::STG_LD]);
                store_32(static_cast<uint8_t*>(p.out) + orow * p.ldo + ((t.n0 + 2 * h) * 64 + seg * 16) * 2, w, wide);
              } else {
                record_status(p.status, kStatusBadIndex);
              }
            }
          }
          epi_sync();  // the staging buffer and tile_ok are rewritten next
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

template <int STAGES, bool SWIGLU>
static int run_mx_wm(const MxGemmLaunch& L, cudaStream_t stream) {
  using S = MxWmShape<STAGES>;
  constexpr auto* kern = grouped_gemm_mx_wm_kernel<STAGES, SWIGLU>;
  CUtensorMap mx, mw;
  if (make_mx_maps(&mx, &mw, L, S::X_BOX) != 0) return -1;
  if (!mx_set_smem<S::SMEM_BYTES, kern>()) return -3;
  const int64_t work = mx_wm_work(L);
  const int limit = gemm_grid_limit();
  launch_kernel(kern, dim3(static_cast<unsigned>(work < limit ? work : limit)), dim3(S::THREADS), S::SMEM_BYTES,
                stream, mx, mw, L.p);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int launch_grouped_mx_wm(const MxGemmLaunch& L, bool swiglu, cudaStream_t stream) {
  return swiglu ? run_mx_wm<5, true>(L, stream) : run_mx_wm<5, false>(L, stream);
}

}  // namespace b200moe
