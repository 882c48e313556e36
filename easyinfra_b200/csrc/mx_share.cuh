// The share of one CTA in a launch of weight units (grouped_gemm_mx_wm.cu).  Without CUDA
// types, so that the host can be asked for every CTA's share.
#pragma once

#ifdef __CUDACC__
#define MX_SHARE_FN __host__ __device__ __forceinline__
#else
#define MX_SHARE_FN inline
#endif

namespace b200moe {

struct MxShare {
  unsigned pos, end;  // units [pos, end) of all
};

// Where part i of `parts` equal parts of n begins: i * n / parts, without the product, which
// passes 32 bits where an expert has more than 2^32 / parts units.
MX_SHARE_FN unsigned mx_part_begin(unsigned n, unsigned parts, unsigned i) {
  const unsigned q = n / parts;
  return i * q + i * (n - q * parts) / parts;
}

// CTA b of `grid`: an equal share of all `total` units; or, where that costs at most an eighth
// more units in the largest one, equal parts of every segment of `u` units (one expert's, for
// one m-tile), so that no share crosses into the next one and leaves two short tiles, each
// with few bytes in flight.
MX_SHARE_FN MxShare mx_share(unsigned total, unsigned u, unsigned grid, unsigned b) {
  const unsigned share = total / grid, rest = total - share * grid;
  const unsigned segs = total / u, parts = segs > 0 ? grid / segs : 0, largest = share + (rest > 0 ? 1 : 0);
  MxShare s;
  if (parts > 0 && (u + parts - 1) / parts <= largest + largest / 8) {
    const unsigned seg = b / parts, i = b - seg * parts;
    s.pos = seg < segs ? seg * u + mx_part_begin(u, parts, i) : total;
    s.end = seg < segs ? seg * u + mx_part_begin(u, parts, i + 1) : total;
  } else {
    s.pos = b * share + (b < rest ? b : rest);
    s.end = s.pos + share + (b < rest ? 1 : 0);
  }
  return s;
}

}  // namespace b200moe
