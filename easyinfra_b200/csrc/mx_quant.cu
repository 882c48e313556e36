// Quantisation to the MX formats (mx.cuh) and back, and the block prologue with an
// 8-bit output.
//
// All of it is bound by HBM: a block of 32 elements is held by 4 lanes (bf16) or 8
// (fp32) with one 16-byte load each, so that loads and stores of a warp are whole
// lines; the block's largest magnitude is a butterfly of 2 or 3 shuffles.
#include "kernels.cuh"
#include "mx.cuh"
#include "norm_row.cuh"

namespace b200moe {

constexpr int MXQ_THREADS = 256;
constexpr int MXQ_UNROLL = 4;                            // 16-byte vectors in flight per thread
constexpr int MXQ_TILE = MXQ_THREADS * MXQ_UNROLL;       // vectors a CTA holds at a time

template <typename E>
struct MxVec {
  static constexpr int V = 16 / sizeof(E);         // elements per 16-byte vector
  static constexpr int LANES = MX_BLOCK / V;       // lanes that share a block
};

template <typename E>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[MxVec<E>::V]) {
  const E* e = reinterpret_cast<const E*>(&v);
#pragma unroll
  for (int j = 0; j < MxVec<E>::V; ++j) f[j] = to_f<E>(e[j]);
}

// Largest |x| of the lane's vector, as fp32 bits, over the lanes of its block (all 32
// lanes take part).  bf16 pairs are compared as 16-bit integers, two at a time.
template <typename E>
__device__ __forceinline__ uint32_t block_amax_bits(const uint4& v) {
  uint32_t m;
  if (sizeof(E) == 2) {
    const uint32_t k = 0x7fff7fffu;
    m = __vmaxu2(__vmaxu2(v.x & k, v.y & k), __vmaxu2(v.z & k, v.w & k));
#pragma unroll
    for (int o = MxVec<E>::LANES / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    return max(m << 16, m & 0xffff0000u);
  }
  const uint32_t k = 0x7fffffffu;
  m = max(max(v.x & k, v.y & k), max(v.z & k, v.w & k));
#pragma unroll
  for (int o = MxVec<E>::LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// The lane's elements, scaled and rounded, at dst (V bytes of MX8 or V/2 of MX4).
template <typename E, bool FOUR>
__device__ __forceinline__ void store_elements(uint8_t* dst, const uint4& v, float inv) {
  constexpr int V = MxVec<E>::V;
  float f[V];
  unpack<E>(v, f);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] *= inv;
  if (FOUR) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < V; j += 2) w |= cvt_e2m1x2(f[j], f[j + 1]) << (4 * j);
    if (V == 8)
      *reinterpret_cast<uint32_t*>(dst) = w;
    else
      *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(w);
  } else {
    uint32_t w[V / 4];
#pragma unroll
    for (int j = 0; j < V; j += 4) w[j / 4] = cvt_e4m3x4(f[j], f[j + 1], f[j + 2], f[j + 3]);
    if (V == 8)
      *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[V / 4 - 1]);
    else
      *reinterpret_cast<uint32_t*>(dst) = w[0];
  }
}

// V elements of 4 or 8 bits to one 16-byte vector of E.
template <typename E, bool FOUR>
__device__ __forceinline__ uint4 load_values(const uint2& w, uint32_t byte) {
  constexpr int V = MxVec<E>::V;
  const float scale = mx_scale_value(byte);
  uint4 o;
  E* oe = reinterpret_cast<E*>(&o);
#pragma unroll
  for (int j = 0; j < V; j += 2) {
    const float2 t = FOUR ? e2m1x2_to_float2((w.x >> (4 * j)) & 0xffu)
                          : e4m3x2_to_float2(((j < 4 ? w.x : w.y) >> (8 * (j % 4))) & 0xffffu);
    oe[j] = from_f<E>(t.x * scale);
    oe[j + 1] = from_f<E>(t.y * scale);
  }
  return o;
}

template <int BYTES>
__device__ __forceinline__ uint2 load_packed(const uint8_t* src) {
  uint2 w = make_uint2(0, 0);
  if (BYTES == 8) w = __ldg(reinterpret_cast<const uint2*>(src));
  if (BYTES == 4) w.x = __ldg(reinterpret_cast<const uint32_t*>(src));
  if (BYTES == 2) w.x = __ldg(reinterpret_cast<const uint16_t*>(src));
  return w;
}

// Contiguous matrices (FLAT) are one long row, a tile of vectors a CTA.  Others give a
// CTA whole rows (rows_cta of them, together at most a tile, or one longer row walked tile
// by tile); a vector's row inside the CTA is idx * magic >> 32 with magic =
// ceil(2^32 / vectors a row), exact for idx below a tile.
struct MxWalk {
  uint32_t per_row, magic;
  int rows_cta;
  int64_t total;  // FLAT: vectors
};

// Vector u of this thread in pass `base` of the CTA; false past the end.
template <bool FLAT>
__device__ __forceinline__ bool walk_at(const MxWalk& w, int64_t rows, uint32_t base, int u, int64_t& row,
                                        int64_t& col) {
  const uint32_t idx = base + u * MXQ_THREADS + threadIdx.x;
  if (FLAT) {
    row = 0;
    col = static_cast<int64_t>(blockIdx.x) * MXQ_TILE + idx;
    return col < w.total;
  }
  const uint32_t r = w.rows_cta > 1 ? __umulhi(idx, w.magic) : 0u;
  col = idx - r * w.per_row;
  row = static_cast<int64_t>(blockIdx.x) * w.rows_cta + r;
  return r < static_cast<uint32_t>(w.rows_cta) && idx < w.rows_cta * w.per_row && row < rows;
}

template <typename E, bool FOUR, bool FLAT>
__global__ void __launch_bounds__(MXQ_THREADS, FLAT ? 8 : 5)
    mx_quantize_kernel(const __grid_constant__ MxQuantParams p, const __grid_constant__ MxWalk w) {
  constexpr int V = MxVec<E>::V;
  constexpr int LANES = MxVec<E>::LANES;
  pdl_trigger();
  pdl_wait();
  const uint32_t end = FLAT ? MXQ_TILE : w.rows_cta * w.per_row;
  for (uint32_t base = 0; base < end; base += MXQ_TILE) {
    uint4 in[MXQ_UNROLL];
#pragma unroll
    for (int u = 0; u < MXQ_UNROLL; ++u) {
      int64_t row, col;
      in[u] = make_uint4(0, 0, 0, 0);
      if (walk_at<FLAT>(w, p.rows, base, u, row, col))
        in[u] = __ldg(reinterpret_cast<const uint4*>(static_cast<const E*>(p.x) + row * p.ldx) + col);
    }
#pragma unroll
    for (int u = 0; u < MXQ_UNROLL; ++u) {
      const uint32_t amax = block_amax_bits<E>(in[u]);
      int64_t row, col;
      if (!walk_at<FLAT>(w, p.rows, base, u, row, col)) continue;
      const uint32_t byte = FOUR ? mx4_scale_byte(amax) : mx8_scale_byte(amax);
      store_elements<E, FOUR>(p.data + row * p.ld_data + col * (FOUR ? V / 2 : V), in[u], mx_inverse_scale(byte));
      if (col % LANES == 0) {
        uint8_t* s = p.scales + row * p.ld_scales + col / LANES;
        *s = static_cast<uint8_t>(byte);
        if (!FOUR && col + LANES == w.per_row)
          for (int i = 1; i <= p.pad; ++i) s[i] = 0;
      }
    }
  }
}

template <typename E, bool FOUR, bool FLAT>
__global__ void __launch_bounds__(MXQ_THREADS, FLAT ? 8 : 5)
    mx_dequantize_kernel(const __grid_constant__ MxDequantParams p, const __grid_constant__ MxWalk w) {
  constexpr int V = MxVec<E>::V;
  constexpr int LANES = MxVec<E>::LANES;
  constexpr int BYTES = FOUR ? V / 2 : V;
  pdl_trigger();
  pdl_wait();
  const uint32_t end = FLAT ? MXQ_TILE : w.rows_cta * w.per_row;
  for (uint32_t base = 0; base < end; base += MXQ_TILE) {
    uint2 in[MXQ_UNROLL];
    uint32_t byte[MXQ_UNROLL];
#pragma unroll
    for (int u = 0; u < MXQ_UNROLL; ++u) {
      int64_t row, col;
      if (walk_at<FLAT>(w, p.rows, base, u, row, col)) {
        in[u] = load_packed<BYTES>(p.data + row * p.ld_data + col * BYTES);
        byte[u] = __ldg(p.scales + row * p.ld_scales + col / LANES);
      }
    }
#pragma unroll
    for (int u = 0; u < MXQ_UNROLL; ++u) {
      int64_t row, col;
      if (walk_at<FLAT>(w, p.rows, base, u, row, col))
        *(reinterpret_cast<uint4*>(static_cast<E*>(p.out) + row * p.ldo) + col) = load_values<E, FOUR>(in[u], byte[u]);
    }
  }
}

// Grid of a matrix of rows x vectors a row; 0 when it does not fit one.
static unsigned mx_walk(MxWalk* w, int64_t rows, int64_t per_row, bool flat) {
  w->total = rows * per_row;
  int64_t grid;
  if (flat) {
    w->per_row = w->magic = 0;
    w->rows_cta = 1;
    grid = (w->total + MXQ_TILE - 1) / MXQ_TILE;
  } else {
    w->per_row = static_cast<uint32_t>(per_row);
    w->magic = static_cast<uint32_t>(((1ull << 32) + per_row - 1) / per_row);
    w->rows_cta = per_row <= MXQ_TILE ? static_cast<int>(MXQ_TILE / per_row) : 1;
    grid = (rows + w->rows_cta - 1) / w->rows_cta;
  }
  return grid > 0x7fffffff ? 0u : static_cast<unsigned>(grid);
}

template <typename E>
static int quantize(const MxQuantParams& p, bool four_bit, cudaStream_t stream) {
  const bool flat = four_bit && p.ldx == p.K && p.ld_data == p.K / 2 && p.ld_scales == p.K / MX_BLOCK;
  MxWalk w;
  const unsigned grid = mx_walk(&w, p.rows, p.K / MxVec<E>::V, flat);
  if (grid == 0) return -1;
  auto* kern = !four_bit ? mx_quantize_kernel<E, false, false>
               : flat    ? mx_quantize_kernel<E, true, true>
                         : mx_quantize_kernel<E, true, false>;
  launch_kernel(kern, dim3(grid), dim3(MXQ_THREADS), 0, stream, p, w);
  return 0;
}

template <typename E>
static int dequantize(const MxDequantParams& p, bool four_bit, cudaStream_t stream) {
  const bool flat = four_bit && p.ldo == p.K && p.ld_data == p.K / 2 && p.ld_scales == p.K / MX_BLOCK;
  MxWalk w;
  const unsigned grid = mx_walk(&w, p.rows, p.K / MxVec<E>::V, flat);
  if (grid == 0) return -1;
  auto* kern = !four_bit ? mx_dequantize_kernel<E, false, false>
               : flat    ? mx_dequantize_kernel<E, true, true>
                         : mx_dequantize_kernel<E, true, false>;
  launch_kernel(kern, dim3(grid), dim3(MXQ_THREADS), 0, stream, p, w);
  return 0;
}

int launch_mx_quantize(const MxQuantParams& p, int dtype, bool four_bit, cudaStream_t stream) {
  return dtype == kDtypeBF16 ? quantize<__nv_bfloat16>(p, four_bit, stream) : quantize<float>(p, four_bit, stream);
}

int launch_mx_dequantize(const MxDequantParams& p, int dtype, bool four_bit, cudaStream_t stream) {
  return dtype == kDtypeBF16 ? dequantize<__nv_bfloat16>(p, four_bit, stream) : dequantize<float>(p, four_bit, stream);
}

// ------------------------------------------------------------------ prologue with MX8 rows
// residual_out = residual + hidden; normed = weight * rmsnorm(residual_out) with the
// rounding points of add_rmsnorm_row (norm_row.cuh); the MX8 row is quantised from the
// normed values, rounded to the activation type as every other reader of them sees them.
//
// A value next to a rounding border of bf16 (and then of e4m3) flips with the last bits of
// 1/rms, and one loud channel may hold most of a row's square: so every square is taken and
// summed in 64 bits, and so is the reciprocal root, which is rounded to fp32 once (sums of a
// thread's squares in fp32 take 100 us instead of 105 at 16384 x 4096 bf16, with 1/rms off by
// up to 2^-20).  The squares of finite values leave fp32's range from 2^64 and 2^-75 on; where
// the mean is that far out, the row is scaled by a power of two before the product, so that
// neither factor leaves fp32's normal range.
//
// One CTA per token, VPT 16-byte vectors a thread in registers between the two passes.
template <typename E, int VPT>
__global__ void __launch_bounds__(512, VPT == 4 ? 2 : VPT == 2 ? 3 : 4)
    add_rmsnorm_mx8_kernel(const __grid_constant__ AddNormParams p, uint8_t* q, int64_t ldq, double inv_h) {
  constexpr int V = MxVec<E>::V;
  __shared__ double red[16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  if (blockIdx.x == 0) prefetch_l2_lines(p.weight, static_cast<int64_t>(p.H) * sizeof(E));
  pdl_wait();
  const int64_t t = blockIdx.x;
  const uint4* res = reinterpret_cast<const uint4*>(static_cast<const E*>(p.residual) + t * p.ld);
  const uint4* hid = p.hidden ? reinterpret_cast<const uint4*>(static_cast<const E*>(p.hidden) + t * p.ld) : nullptr;
  uint4* rout = reinterpret_cast<uint4*>(static_cast<E*>(p.residual_out) + t * p.ld);
  const int nvec = p.H / V;
  uint4 keep[VPT], add[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = threadIdx.x + i * blockDim.x;
    keep[i] = add[i] = make_uint4(0, 0, 0, 0);
    if (vi < nvec) {
      keep[i] = res[vi];
      if (hid) add[i] = hid[vi];
    }
  }
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = threadIdx.x + i * blockDim.x;
    E* oe = reinterpret_cast<E*>(&keep[i]);
    if (hid) {
      const E* be = reinterpret_cast<const E*>(&add[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) oe[j] = from_f<E>(to_f<E>(oe[j]) + to_f<E>(be[j]));
    }
    if (vi < nvec) rout[vi] = keep[i];
    float f[V];
    unpack<E>(keep[i], f);
    double part = 0.0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double d = f[j];
      part = fma(d, d, part);
    }
    sum += part;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) red[warp] = sum;
  uint4 wv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = threadIdx.x + i * blockDim.x;
    wv[i] = vi < nvec ? __ldg(static_cast<const uint4*>(p.weight) + vi) : make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  double mean = red[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) mean += red[w];
  mean = fma(mean, inv_h, static_cast<double>(p.eps));
  // 1/rms from 2^-60 to 2^60 is taken as it is; beyond, scale * inv stands for it
  const bool huge = mean > 0x1p120, tiny = mean < 0x1p-120;
  const float scale = huge ? 0x1p-64f : tiny ? 0x1p64f : 1.f;
  const float inv = static_cast<float>(rsqrt(mean) * (huge ? 0x1p64 : tiny ? 0x1p-64 : 1.0));
  uint4* nout = p.normed ? reinterpret_cast<uint4*>(static_cast<E*>(p.normed) + t * p.ld_normed) : nullptr;
  uint8_t* qrow = q + t * ldq;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int vi = threadIdx.x + i * blockDim.x;
    const E* ae = reinterpret_cast<const E*>(&keep[i]);
    const E* we = reinterpret_cast<const E*>(&wv[i]);
    uint4 o;
    E* oe = reinterpret_cast<E*>(&o);
#pragma unroll
    for (int j = 0; j < V; ++j) oe[j] = from_f<E>(to_f<E>(we[j]) * to_f<E>(from_f<E>(to_f<E>(ae[j]) * scale * inv)));
    const uint32_t byte = mx8_scale_byte(block_amax_bits<E>(o));  // every lane takes part
    if (vi < nvec) {
      if (nout) nout[vi] = o;
      store_elements<E, false>(qrow + vi * V, o, mx_inverse_scale(byte));
      if (lane % MxVec<E>::LANES == 0) qrow[p.H + vi / MxVec<E>::LANES] = static_cast<uint8_t>(byte);
    }
  }
  const int nb = p.H / MX_BLOCK;
  if (threadIdx.x < (16 - nb % 16) % 16) qrow[p.H + nb + threadIdx.x] = 0;  // padding
}

template <typename E, int VPT>
static void run_add_rmsnorm_mx8(const AddNormParams& p, int nvec, uint8_t* q, int64_t ldq, cudaStream_t stream) {
  const int threads = ((nvec + VPT - 1) / VPT + 31) / 32 * 32;
  launch_kernel(add_rmsnorm_mx8_kernel<E, VPT>, dim3(p.T), dim3(threads), 0, stream, p, q, ldq, 1.0 / p.H);
}

template <typename E>
static int add_rmsnorm_mx8(const AddNormParams& p, uint8_t* q, int64_t ldq, cudaStream_t stream) {
  const int nvec = p.H / MxVec<E>::V;
  if (nvec > 512 * 4) return -1;
  // Batches of many waves: fewer threads with more loads each, so that more rows are on an
  // SM and one's loads cover another's reduction (16384 x 4096 bf16: 126 us with one vector a
  // thread, 109 with two, 105 with four and at most 64 registers; without the add 109, 92 and
  // 90; fp32 177, 177 and 171).  Few rows: every load of a row at once (1024 x 2048 bf16: 5.4,
  // 6.3, 6.9 us).
  int vpt = p.T <= 8 * num_sms() ? 1 : 4;
  while (nvec > 512 * vpt) vpt *= 2;
  if (vpt == 1)
    run_add_rmsnorm_mx8<E, 1>(p, nvec, q, ldq, stream);
  else if (vpt == 2)
    run_add_rmsnorm_mx8<E, 2>(p, nvec, q, ldq, stream);
  else
    run_add_rmsnorm_mx8<E, 4>(p, nvec, q, ldq, stream);
  return 0;
}

int launch_add_rmsnorm_mx8(const AddNormParams& p, void* q, int64_t ldq, cudaStream_t stream) {
  if (p.T == 0) return 0;
  return p.dtype == kDtypeBF16 ? add_rmsnorm_mx8<__nv_bfloat16>(p, static_cast<uint8_t*>(q), ldq, stream)
                               : add_rmsnorm_mx8<float>(p, static_cast<uint8_t*>(q), ldq, stream);
}

}  // namespace b200moe
