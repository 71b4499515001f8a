// FP4 page pool: layout arithmetic and conversions shared by the FP4 kernels.
#pragma once

#include "iak_internal.cuh"

namespace iak {

constexpr int kFp4MaxPage = 16384;
constexpr int kFp4ScaleMin = 127 - 14, kFp4ScaleMax = 127 + 13;   // scale bytes an append writes

struct Fp4Pool {
  uint8_t* data;
  int64_t num_pages;
  int PS, D;
};

// Scale byte of a block with largest magnitude amax: the smallest e with 6 * 2^e >= amax.  amax = m * 2^k,
// 1 <= m < 2, and 6 = 1.5 * 4, so e = k - 2 for m <= 1.5 and k - 1 above, where the addend carries into the exponent;
// subnormals end at the lower bound, infinity at the upper.
__device__ __forceinline__ int fp4_scale_byte(float amax) {
  const int b = static_cast<int>((__float_as_uint(amax) + 0x3fffffu) >> 23) - 2;
  return min(max(b, kFp4ScaleMin), kFp4ScaleMax);
}

__device__ __forceinline__ float fp4_inv_scale(int byte) { return __uint_as_float((254 - byte) << 23); }

// eight E2M1 codes, x[i] in bits 4i..: nearest, ties to the even code, saturating at 6
__device__ __forceinline__ unsigned fp4_pack8(const float (&x)[8]) {
  unsigned r;
  asm("{\n.reg .b8 b0, b1, b2, b3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      "mov.b32 %0, {b0, b1, b2, b3};\n}"
      : "=r"(r) : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return r;
}

// the four bytes of w as half pairs (bits 0..3 of a byte in the low half)
__device__ __forceinline__ void fp4_unpack4(unsigned w, unsigned (&h)[4]) {
  asm("{\n.reg .b8 b0, b1, b2, b3;\nmov.b32 {b0, b1, b2, b3}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\ncvt.rn.f16x2.e2m1x2 %1, b1;\n"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\ncvt.rn.f16x2.e2m1x2 %3, b3;\n}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}

// Four scale bytes e + 127 -> the upper bytes of the halves 2^e (the lower ones are 0).  A half's exponent, e + 15, is the
// byte - 112 in five bits: the byte's low five with bit 4 turned.  Nothing carries from one to the next: the byte of a row
// that was never written may be anything (0 in a zeroed pool), its neighbour keeps its scale.
__device__ __forceinline__ unsigned fp4_half_tops(unsigned bytes) { return (bytes * 4u ^ 0x40404040u) & 0x7c7c7c7cu; }
// the half pair 2^e of bytes I (low) and J
template <int I, int J>
__device__ __forceinline__ unsigned fp4_scale_pair(unsigned tops) {
  return __byte_perm(tops, 0, J << 12 | 4 << 8 | I << 4 | 4);
}

// A group of 16 rows: byte offsets (the public header has the layout in words).
template <int NB>
struct Fp4Group {
  static constexpr int kPW = NB < 4 ? NB : 4;          // words of a lane's piece
  static constexpr int kSet = 128 * NB;                // 8 rows of K, or of V
  static constexpr int kV = 2 * kSet, kKs = 4 * kSet, kVs = kKs + 16 * NB;
  static constexpr int kBytes = 544 * NB;
  static __host__ __device__ constexpr int word(int lane, int w) { return ((w / kPW) * 32 + lane) * kPW + w % kPW; }
  static __device__ __forceinline__ int k_scale(int r, int b) { return kKs + ((r & 7) * 2 + (r >> 3)) * NB + b; }
  static __device__ __forceinline__ int v_scale(int r, int b) {
    return kVs + (b * 4 + ((r & 7) >> 1)) * 4 + (r & 1) + 2 * (r >> 3);
  }
};

int check_fp4_pool(const iak_fp4_pool* pool, const char* what);

}  // namespace iak
