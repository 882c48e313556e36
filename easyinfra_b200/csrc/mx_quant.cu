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
constexpr int MXQ_UNROLL = 4;  // 16-byte loads in flight per thread

template <typename E>
struct MxVec {
  static constexpr int V = 16 / sizeof(E);         // elements per 16-byte vector
  static constexpr int LANES = MX_BLOCK / V;       // lanes that share a block
};

// Largest |x| of the lane's vector, as bits, over the lanes of its block.
template <typename E>
__device__ __forceinline__ uint32_t block_amax_bits(const float (&f)[MxVec<E>::V]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < MxVec<E>::V; ++j) m = max(m, __float_as_uint(f[j]) & 0x7fffffffu);
#pragma unroll
  for (int o = MxVec<E>::LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

template <typename E>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[MxVec<E>::V]) {
  const E* e = reinterpret_cast<const E*>(&v);
#pragma unroll
  for (int j = 0; j < MxVec<E>::V; ++j) f[j] = to_f<E>(e[j]);
}

// The lane's elements, scaled and rounded, at dst (V bytes of MX8 or V/2 of MX4).
template <typename E, bool FOUR>
__device__ __forceinline__ void store_elements(uint8_t* dst, const float (&f)[MxVec<E>::V], float inv) {
  constexpr int V = MxVec<E>::V;
  if (FOUR) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < V; j += 2) w |= cvt_e2m1x2(f[j] * inv, f[j + 1] * inv) << (4 * j);
    if (V == 8)
      *reinterpret_cast<uint32_t*>(dst) = w;
    else
      *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(w);
  } else {
    uint32_t w[V / 4];
#pragma unroll
    for (int j = 0; j < V; j += 4) w[j / 4] = cvt_e4m3x4(f[j] * inv, f[j + 1] * inv, f[j + 2] * inv, f[j + 3] * inv);
    if (V == 8)
      *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[V / 4 - 1]);
    else
      *reinterpret_cast<uint32_t*>(dst) = w[0];
  }
}

// Flat over the vectors of all rows; the row of a vector is a 32-bit division when the
// matrix is small enough, and there is none for one row (the host flattens contiguous
// MX4 matrices to that).
__device__ __forceinline__ void split_row(int64_t v, int64_t per_row, bool one_row, int64_t& row, int64_t& col) {
  if (one_row) {
    row = 0;
    col = v;
  } else if (((v | per_row) >> 32) == 0) {
    row = static_cast<uint32_t>(v) / static_cast<uint32_t>(per_row);
    col = v - row * per_row;
  } else {
    row = v / per_row;
    col = v - row * per_row;
  }
}

template <typename E, bool FOUR>
__global__ void __launch_bounds__(MXQ_THREADS) mx_quantize_kernel(const __grid_constant__ MxQuantParams p) {
  constexpr int V = MxVec<E>::V;
  pdl_trigger();
  pdl_wait();
  const int64_t per_row = p.K / V;
  const int64_t total = p.rows * per_row;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (MXQ_THREADS * MXQ_UNROLL) + threadIdx.x;
  uint4 in[MXQ_UNROLL];
  int64_t row[MXQ_UNROLL], col[MXQ_UNROLL];
#pragma unroll
  for (int u = 0; u < MXQ_UNROLL; ++u) {
    const int64_t v = base + u * MXQ_THREADS;
    in[u] = make_uint4(0, 0, 0, 0);
    if (v < total) {
      split_row(v, per_row, p.rows == 1, row[u], col[u]);
      in[u] = __ldg(reinterpret_cast<const uint4*>(static_cast<const E*>(p.x) + row[u] * p.ldx) + col[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < MXQ_UNROLL; ++u) {
    float f[V];
    unpack<E>(in[u], f);
    const uint32_t amax = block_amax_bits<E>(f);  // every lane takes part
    if (base + u * MXQ_THREADS >= total) continue;
    const uint32_t byte = FOUR ? mx4_scale_byte(amax) : mx8_scale_byte(amax);
    const float inv = mx_inverse_scale(byte);
    store_elements<E, FOUR>(p.data + row[u] * p.ld_data + col[u] * V / (FOUR ? 2 : 1), f, inv);
    if (threadIdx.x % MxVec<E>::LANES == 0) {
      uint8_t* s = p.scales + row[u] * p.ld_scales;
      const int64_t b = col[u] / MxVec<E>::LANES;
      s[b] = static_cast<uint8_t>(byte);
      if (!FOUR && b == p.K / MX_BLOCK - 1)
        for (int i = 1; i <= p.pad; ++i) s[b + i] = 0;
    }
  }
}

template <typename E, bool FOUR>
__global__ void __launch_bounds__(MXQ_THREADS) mx_dequantize_kernel(const __grid_constant__ MxDequantParams p) {
  constexpr int V = MxVec<E>::V;  // elements per 16-byte output vector
  pdl_trigger();
  pdl_wait();
  const int64_t per_row = p.K / V;
  const int64_t total = p.rows * per_row;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (MXQ_THREADS * MXQ_UNROLL) + threadIdx.x;
  constexpr int BYTES = FOUR ? V / 2 : V;  // packed bytes of a vector: 2, 4 or 8
  uint32_t w[MXQ_UNROLL][2];
  uint32_t sb[MXQ_UNROLL];
  int64_t row[MXQ_UNROLL], col[MXQ_UNROLL];
#pragma unroll
  for (int u = 0; u < MXQ_UNROLL; ++u) {
    const int64_t v = base + u * MXQ_THREADS;
    if (v < total) {
      split_row(v, per_row, p.rows == 1, row[u], col[u]);
      const uint8_t* src = p.data + row[u] * p.ld_data + col[u] * BYTES;
      if (BYTES == 8) {
        const uint2 t = __ldg(reinterpret_cast<const uint2*>(src));
        w[u][0] = t.x;
        w[u][1] = t.y;
      } else if (BYTES == 4) {
        w[u][0] = __ldg(reinterpret_cast<const uint32_t*>(src));
      } else {
        w[u][0] = __ldg(reinterpret_cast<const uint16_t*>(src));
      }
      sb[u] = __ldg(p.scales + row[u] * p.ld_scales + col[u] / MxVec<E>::LANES);
    }
  }
#pragma unroll
  for (int u = 0; u < MXQ_UNROLL; ++u) {
    if (base + u * MXQ_THREADS >= total) continue;
    const float scale = mx_scale_value(sb[u]);
    uint4 o;
    E* oe = reinterpret_cast<E*>(&o);
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 t = FOUR ? e2m1x2_to_float2((w[u][0] >> (4 * j)) & 0xffu)
                            : e4m3x2_to_float2((w[u][j / 4] >> (8 * (j % 4))) & 0xffffu);
      oe[j] = from_f<E>(t.x * scale);
      oe[j + 1] = from_f<E>(t.y * scale);
    }
    *(reinterpret_cast<uint4*>(static_cast<E*>(p.out) + row[u] * p.ldo) + col[u]) = o;
  }
}

static int64_t quant_grid(int64_t vectors) {
  return (vectors + MXQ_THREADS * MXQ_UNROLL - 1) / (MXQ_THREADS * MXQ_UNROLL);
}

int launch_mx_quantize(const MxQuantParams& p0, int dtype, bool four_bit, cudaStream_t stream) {
  MxQuantParams p = p0;
  if (four_bit && p.ldx == p.K && p.ld_data == p.K / 2 && p.ld_scales == p.K / MX_BLOCK) {
    p.K *= p.rows;  // contiguous: one long row
    p.rows = 1;
  }
  const int64_t grid = quant_grid(p.rows * p.K / (dtype == kDtypeBF16 ? 8 : 4));
  if (grid > 0x7fffffff) return -1;
  auto* kern = dtype == kDtypeBF16
                   ? (four_bit ? mx_quantize_kernel<__nv_bfloat16, true> : mx_quantize_kernel<__nv_bfloat16, false>)
                   : (four_bit ? mx_quantize_kernel<float, true> : mx_quantize_kernel<float, false>);
  launch_kernel(kern, dim3(static_cast<unsigned>(grid)), dim3(MXQ_THREADS), 0, stream, p);
  return 0;
}

int launch_mx_dequantize(const MxDequantParams& p0, int dtype, bool four_bit, cudaStream_t stream) {
  MxDequantParams p = p0;
  if (four_bit && p.ldo == p.K && p.ld_data == p.K / 2 && p.ld_scales == p.K / MX_BLOCK) {
    p.K *= p.rows;
    p.rows = 1;
  }
  const int64_t grid = quant_grid(p.rows * p.K / (dtype == kDtypeBF16 ? 8 : 4));
  if (grid > 0x7fffffff) return -1;
  auto* kern = dtype == kDtypeBF16 ? (four_bit ? mx_dequantize_kernel<__nv_bfloat16, true>
                                               : mx_dequantize_kernel<__nv_bfloat16, false>)
                                   : (four_bit ? mx_dequantize_kernel<float, true> : mx_dequantize_kernel<float, false>);
  launch_kernel(kern, dim3(static_cast<unsigned>(grid)), dim3(MXQ_THREADS), 0, stream, p);
  return 0;
}

// ------------------------------------------------------------------ prologue with MX8 rows
// residual_out = residual + hidden; normed = weight * rmsnorm(residual_out) with the
// rounding points of add_rmsnorm_row (norm_row.cuh) and its summation order, so residual
// and normed have the same bits as there; the MX8 row is quantised from the normed
// values, rounded to the activation type as every other reader of them sees them.
template <typename E>
__global__ void __launch_bounds__(NORM_THREADS)
    add_rmsnorm_mx8_kernel(const __grid_constant__ AddNormParams p, uint8_t* q, int64_t ldq) {
  constexpr int V = MxVec<E>::V;
  __shared__ float red[NORM_THREADS / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  if (blockIdx.x == 0) prefetch_l2_lines(p.weight, static_cast<int64_t>(p.H) * sizeof(E));
  pdl_wait();
  const int64_t t = blockIdx.x;
  const E* res = static_cast<const E*>(p.residual) + t * p.ld;
  const E* hid = p.hidden ? static_cast<const E*>(p.hidden) + t * p.ld : nullptr;
  E* rout = static_cast<E*>(p.residual_out) + t * p.ld;
  const int nvec = p.H / V;
  uint4 keep[NORM_MAXV];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NORM_MAXV; ++i) {
    const int vi = threadIdx.x + i * NORM_THREADS;
    keep[i] = make_uint4(0, 0, 0, 0);
    if (vi < nvec) {
      uint4 o = *reinterpret_cast<const uint4*>(res + vi * V);
      if (hid) {
        const uint4 b = *reinterpret_cast<const uint4*>(hid + vi * V);
        E* oe = reinterpret_cast<E*>(&o);
        const E* be = reinterpret_cast<const E*>(&b);
#pragma unroll
        for (int j = 0; j < V; ++j) oe[j] = from_f<E>(to_f<E>(oe[j]) + to_f<E>(be[j]));
      }
      float f[V];
      unpack<E>(o, f);
#pragma unroll
      for (int j = 0; j < V; ++j) ss = fmaf(f[j], f[j], ss);
      *reinterpret_cast<uint4*>(rout + vi * V) = o;
      keep[i] = o;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (lane == 0) red[warp] = ss;
  __syncthreads();
  float tot = 0.f;
#pragma unroll
  for (int w = 0; w < NORM_THREADS / 32; ++w) tot += red[w];
  const float inv = rsqrtf(tot / static_cast<float>(p.H) + p.eps);
  const E* wrow = static_cast<const E*>(p.weight);
  E* nout = p.normed ? static_cast<E*>(p.normed) + t * p.ld_normed : nullptr;
  uint8_t* qrow = q + t * ldq;
#pragma unroll
  for (int i = 0; i < NORM_MAXV; ++i) {
    if (i * NORM_THREADS >= nvec) break;  // the same for every thread: all take part in the shuffles
    const int vi = threadIdx.x + i * NORM_THREADS;
    const bool in = vi < nvec;
    uint4 o = make_uint4(0, 0, 0, 0);
    if (in) {
      const uint4 wv = *reinterpret_cast<const uint4*>(wrow + vi * V);
      const E* ae = reinterpret_cast<const E*>(&keep[i]);
      const E* we = reinterpret_cast<const E*>(&wv);
      E* oe = reinterpret_cast<E*>(&o);
#pragma unroll
      for (int j = 0; j < V; ++j) oe[j] = from_f<E>(to_f<E>(we[j]) * to_f<E>(from_f<E>(to_f<E>(ae[j]) * inv)));
    }
    float f[V];
    unpack<E>(o, f);
    const uint32_t byte = mx8_scale_byte(block_amax_bits<E>(f));
    if (in) {
      if (nout) *reinterpret_cast<uint4*>(nout + vi * V) = o;
      store_elements<E, false>(qrow + vi * V, f, mx_inverse_scale(byte));
      if (lane % MxVec<E>::LANES == 0) qrow[p.H + vi / MxVec<E>::LANES] = static_cast<uint8_t>(byte);
    }
  }
  const int nb = p.H / MX_BLOCK;
  if (threadIdx.x < (16 - nb % 16) % 16) qrow[p.H + nb + threadIdx.x] = 0;  // padding
}

int launch_add_rmsnorm_mx8(const AddNormParams& p, void* q, int64_t ldq, cudaStream_t stream) {
  if (p.T == 0) return 0;
  const int vec = 16 / (p.dtype == kDtypeBF16 ? 2 : 4);
  if (p.H / vec > NORM_THREADS * NORM_MAXV) return -1;
  auto* kern = p.dtype == kDtypeBF16 ? add_rmsnorm_mx8_kernel<__nv_bfloat16> : add_rmsnorm_mx8_kernel<float>;
  launch_kernel(kern, dim3(p.T), dim3(NORM_THREADS), 0, stream, p, static_cast<uint8_t*>(q), ldq);
  return 0;
}

}  // namespace b200moe
