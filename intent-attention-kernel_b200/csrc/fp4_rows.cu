// FP4 page pool: quantise-on-write of new rows (iak_fp4_append) and reading rows back (iak_fp4_read).
//
// Both are copies: per row and channel they move 2 * (element size + 17/32) bytes, which bounds them for long
// prompts; a decode step's few rows are bound by the launch.  A warp owns 8 aligned rows of K and V, its lanes what the
// attention kernel's lanes read of them: lane 4 g + t has row g's channels 32 b + 8 t .. + 7 of K (all blocks b) and
// channels 4 NB g .. of rows 2 t and 2 t + 1 of V.  Codes move as one run of 512 bytes (D 128) per plane, dense rows as
// 64-byte runs and more.  A V byte whose other row is not part of the call keeps that row's half.
// 8 x 8 x 32768 rows of D 128 read as bf16: 211 us, 6.4 TB/s; 4 ragged prompts of up to 8187 rows, 8 heads, fp16: 27 us to
// write (5.1 TB/s), 28 to read.
#include "fp4.cuh"

namespace iak {
namespace {

struct RowsParams {
  Fp4Pool pool;
  void* k; void* v; int dtype;
  int64_t k_sb, k_sh, k_sn, v_sb, v_sh, v_sn;
  int B, Ht, N;
  const int32_t* pt; int64_t pt_sb, pt_sh; int W;
  const int32_t* positions; const int32_t* counts; int32_t* dropped;
  int64_t octets;     // runs of 8 aligned rows that a (b, h) can touch
};

constexpr int kRowThreads = 256;

// How dense rows are read: 16 bytes at a time by type, or an element at a time (any type, any alignment).
enum { kAny = -1 };

// Eight neighbouring channels of a row as they were read.
template <int KIND>
struct Eight {
  static constexpr int kWords = KIND == IAK_DT_F16 || KIND == IAK_DT_BF16 ? 4 : 8;
  unsigned w[kWords];
  __device__ __forceinline__ void load(const void* base, int dtype, int64_t at, bool real) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
    if (!real) return;
    if constexpr (KIND == kAny) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(load_as_float(base, dtype, at + i));
    } else if constexpr (KIND == IAK_DT_F32) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + at);
      const uint4 a = __ldg(p), b = __ldg(p + 1);
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    } else {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at));
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    }
  }
  // the larger magnitude of a and b, of both halves for 16-bit types; the sign is of no use; NaN where there is one
  static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
    unsigned r;
    if constexpr (KIND == IAK_DT_F16) asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else if constexpr (KIND == IAK_DT_BF16) asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ __forceinline__ unsigned largest() const {
    unsigned m = larger(w[0], w[1]);
#pragma unroll
    for (int i = 2; i < kWords; ++i) m = larger(m, w[i]);
    return m;
  }
  // the magnitude that `largest` (or several of them, joined by `larger`) stands for
  static __device__ __forceinline__ float magnitude(unsigned m) {
    if constexpr (kWords == 8) return fabsf(__uint_as_float(m));
    m = larger(m, m >> 16 | m << 16) & 0x7fffu;
    if constexpr (KIND == IAK_DT_F16) return __half2float(__ushort_as_half(static_cast<unsigned short>(m)));
    return __uint_as_float(m << 16);
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (kWords == 8) return __uint_as_float(w[i]);
    const unsigned u = w[i / 2];
    if constexpr (KIND == IAK_DT_F16) {
      const __half2 h = *reinterpret_cast<const __half2*>(&u);
      return i % 2 ? __high2float(h) : __low2float(h);
    }
    return __uint_as_float(i % 2 ? u & 0xffff0000u : u << 16);
  }
  // NaN -> 0
  __device__ __forceinline__ void clean() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (kWords == 8) {
        if ((w[i] & 0x7fffffffu) > 0x7f800000u) w[i] = 0;
      } else {
        const unsigned inf = KIND == IAK_DT_F16 ? 0x7c00u : 0x7f80u;
        if ((w[i] & 0x7fffu) > inf) w[i] &= 0xffff0000u;
        if ((w[i] >> 16 & 0x7fffu) > inf) w[i] &= 0xffffu;
      }
    }
  }
};

// Where a warp works: 8 rows of one (b, h), tokens 8 k .. 8 k + 7.  Row j is row i0 + j of the call's.
struct Place {
  int b, h;
  int64_t i0;             // negative where the rows begin before the call's
  int n;                  // rows of the call that are real: counts[b], at most N
  int id;                 // page, or -1: no such table entry
  int64_t tok_in_page;
  int hi;                 // which 8 of the group's 16 rows
  __device__ __forceinline__ bool in(const RowsParams& p, int j) const { return i0 + j >= 0 && i0 + j < p.N; }
  __device__ __forceinline__ bool real(int j) const { return i0 + j >= 0 && i0 + j < n; }
};

template <int NB>
__device__ __forceinline__ bool find_place(const RowsParams& p, Place& w) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (kRowThreads / 32) + (threadIdx.x >> 5);
  const int64_t bh = at / p.octets;
  if (bh >= static_cast<int64_t>(p.B) * p.Ht) return false;
  w.b = static_cast<int>(bh / p.Ht);
  w.h = static_cast<int>(bh - static_cast<int64_t>(w.b) * p.Ht);
  const int64_t pos = p.positions ? p.positions[w.b] : 0;
  w.n = p.counts ? min(max(p.counts[w.b], 0), p.N) : p.N;
  const int64_t tok0 = (pos & ~int64_t(7)) + 8 * (at - bh * p.octets);
  w.i0 = tok0 - pos;
  w.hi = static_cast<int>(tok0 >> 3) & 1;    // page sizes are multiples of 16: so are pages' first tokens
  w.id = -1;
  w.tok_in_page = 0;
  if (tok0 >= 0 && w.i0 < w.n) {
    const int64_t slot = tok0 / p.pool.PS;
    w.tok_in_page = tok0 - slot * p.pool.PS;
    if (slot < p.W) w.id = p.pt[w.b * p.pt_sb + w.h * p.pt_sh + slot];
  }
  return w.i0 < p.N;
}

// the 16 rows' bytes, or null: no such page
template <int NB>
__device__ __forceinline__ uint8_t* group_of(const RowsParams& p, const Place& w) {
  if (w.id < 0 || w.id >= p.pool.num_pages) return nullptr;
  return p.pool.data + ((static_cast<int64_t>(w.id) * p.pool.PS + w.tok_in_page) >> 4) * Fp4Group<NB>::kBytes;
}

template <int NB>
__device__ __forceinline__ void put_words(uint8_t* set, int lane, const unsigned (&w)[NB]) {
  using Gr = Fp4Group<NB>;
  if constexpr (NB == 2) {
    *reinterpret_cast<uint2*>(set + 4 * Gr::word(lane, 0)) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < NB; i += 4)
      *reinterpret_cast<uint4*>(set + 4 * Gr::word(lane, i)) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  }
}
template <int NB>
__device__ __forceinline__ void get_words(const uint8_t* set, int lane, unsigned (&w)[NB]) {
  using Gr = Fp4Group<NB>;
  if constexpr (NB == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(set + 4 * Gr::word(lane, 0));
    w[0] = v.x; w[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < NB; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(set + 4 * Gr::word(lane, i));
      w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
    }
  }
}

template <int NB, int KIND>
__global__ void __launch_bounds__(kRowThreads) fp4_append_kernel(const RowsParams p) {
  using Gr = Fp4Group<NB>;
  using E = Eight<KIND>;
  Place w;
  if (!find_place<NB>(p, w)) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  constexpr int VC = NB / 2;                  // runs of 8 channels that a lane has of a V row
  const bool k_real = w.real(g), v_real0 = w.real(2 * t), v_real1 = w.real(2 * t + 1);
  // the rows are on their way while the page id is
  E k[NB], v[2][VC];
  const int64_t kat = w.b * p.k_sb + w.h * p.k_sh + (w.i0 + g) * p.k_sn + t * 8;
  const int64_t vat = w.b * p.v_sb + w.h * p.v_sh + (w.i0 + 2 * t) * p.v_sn + g * (4 * NB);
#pragma unroll
  for (int b = 0; b < NB; ++b) k[b].load(p.k, p.dtype, kat + 32 * b, k_real);
#pragma unroll
  for (int c = 0; c < VC; ++c) {
    v[0][c].load(p.v, p.dtype, vat + 8 * c, v_real0);
    v[1][c].load(p.v, p.dtype, vat + p.v_sn + 8 * c, v_real1);
  }
  uint8_t* group = group_of<NB>(p, w);
  if (!group) {
    if (p.dropped) {
      const int n = __popc(__ballot_sync(~0u, lane < 8 && w.real(lane)));
      if (lane == 0 && n) atomicAdd(p.dropped, n);
    }
    return;
  }
  // largest magnitudes: of K's blocks over the row's 4 lanes, of V's over 8 / NB neighbouring g
  float k_max[NB], v_max[2];
  auto measure = [&]() {
    bool nan = false;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      unsigned m = k[b].largest();
      m = E::larger(m, __shfl_xor_sync(~0u, m, 1));
      m = E::larger(m, __shfl_xor_sync(~0u, m, 2));
      k_max[b] = E::magnitude(m);
      nan = nan || k_max[b] != k_max[b];
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      unsigned m = v[r][0].largest();
#pragma unroll
      for (int c = 1; c < VC; ++c) m = E::larger(m, v[r][c].largest());
      if (NB <= 4) m = E::larger(m, __shfl_xor_sync(~0u, m, 4));
      if (NB <= 2) m = E::larger(m, __shfl_xor_sync(~0u, m, 8));
      v_max[r] = E::magnitude(m);
      nan = nan || v_max[r] != v_max[r];
    }
    return __any_sync(~0u, nan);
  };
  if (measure()) {                            // a NaN among the rows
#pragma unroll
    for (int b = 0; b < NB; ++b) k[b].clean();
#pragma unroll
    for (int c = 0; c < VC; ++c) {
      v[0][c].clean();
      v[1][c].clean();
    }
    measure();
  }
  unsigned word[NB];
  int byte[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    byte[b] = fp4_scale_byte(k_max[b]);
    const float inv = fp4_inv_scale(byte[b]);             // a power of two: the products are exact
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = k[b].value(i) * inv;
    word[b] = fp4_pack8(x);
  }
  if (k_real) {
    put_words<NB>(group + w.hi * Gr::kSet, lane, word);
    if (t == 0) {
      uint8_t* to = group + Gr::k_scale(8 * w.hi + g, 0);
#pragma unroll
      for (int b = 0; b < NB; b += 2)
        *reinterpret_cast<uint16_t*>(to + b) = static_cast<uint16_t>(byte[b] | byte[b + 1] << 8);
    }
  }
  if (!v_real0 && !v_real1) return;
  const int b0 = fp4_scale_byte(v_max[0]), b1 = fp4_scale_byte(v_max[1]);
  const float inv0 = fp4_inv_scale(b0), inv1 = fp4_inv_scale(b1);
#pragma unroll
  for (int j = 0; j < NB; ++j) {              // byte of a channel: both rows' codes
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = 4 * j + i;
      x[2 * i] = v[0][c / 8].value(c % 8) * inv0;
      x[2 * i + 1] = v[1][c / 8].value(c % 8) * inv1;
    }
    word[j] = fp4_pack8(x);
  }
  uint8_t* set = group + Gr::kV + w.hi * Gr::kSet;
  if (!(v_real0 && v_real1)) {                // the other row's half stays as it is
    unsigned old[NB];
    get_words<NB>(set, lane, old);
    const unsigned mine = v_real0 ? 0x0f0f0f0fu : 0xf0f0f0f0u;
#pragma unroll
    for (int j = 0; j < NB; ++j) word[j] = (word[j] & mine) | (old[j] & ~mine);
  }
  put_words<NB>(set, lane, word);
  if (g % (8 / NB) == 0) {
    uint8_t* to = group + Gr::v_scale(8 * w.hi + 2 * t, g * NB / 8);
    if (v_real0) to[0] = static_cast<uint8_t>(b0);
    if (v_real1) to[1] = static_cast<uint8_t>(b1);
  }
}

// the pool's values are halves, so the products are exact
__device__ __forceinline__ unsigned mul2(unsigned a, unsigned b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const unsigned*>(&r);
}
// 8 values held as half pairs, as 16-bit values of the type
__device__ __forceinline__ uint4 as_16bit(const unsigned* h, int dtype) {
  if (dtype == IAK_DT_F16) return make_uint4(h[0], h[1], h[2], h[3]);
  unsigned u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    const __nv_bfloat162 v = __floats2bfloat162_rn(f.x, f.y);
    u[i] = *reinterpret_cast<const unsigned*>(&v);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ uint4 as_floats(const unsigned* h) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h[0]));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&h[1]));
  return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
}
// Two lanes that differ in bit XOR and write the same row have 32 bytes each, a and b; every store of the pair fills a
// whole 32-byte sector: first the lower lane's, then the upper's.  `to`: this lane's 32 bytes, `gap`: to the other's.
template <int XOR>
__device__ __forceinline__ void store_sectors(char* to, int gap, uint4 a, uint4 b, bool write) {
  const bool upper = threadIdx.x & XOR;
  const uint4 send = upper ? a : b;
  uint4 got;
  got.x = __shfl_xor_sync(~0u, send.x, XOR);
  got.y = __shfl_xor_sync(~0u, send.y, XOR);
  got.z = __shfl_xor_sync(~0u, send.z, XOR);
  got.w = __shfl_xor_sync(~0u, send.w, XOR);
  if (!write) return;
  __stcs(reinterpret_cast<uint4*>(upper ? to - gap + 16 : to), upper ? got : a);
  __stcs(reinterpret_cast<uint4*>(upper ? to + 16 : to + gap), upper ? b : got);
}

// KIND: IAK_DT_F32, IAK_DT_F16 (either 16-bit type) or kAny
template <int NB, int KIND>
__global__ void __launch_bounds__(kRowThreads) fp4_read_kernel(const RowsParams p) {
  using Gr = Fp4Group<NB>;
  Place w;
  if (!find_place<NB>(p, w)) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint8_t* group = group_of<NB>(p, w);
  unsigned kw[NB] = {}, vw[NB] = {}, ks[NB / 2] = {}, vs = 0;
  if (group) {
    get_words<NB>(group + w.hi * Gr::kSet, lane, kw);
    get_words<NB>(group + Gr::kV + w.hi * Gr::kSet, lane, vw);
    const uint16_t* from = reinterpret_cast<const uint16_t*>(group + Gr::k_scale(8 * w.hi + g, 0));
#pragma unroll
    for (int b = 0; b < NB / 2; ++b) ks[b] = from[b];
    vs = *reinterpret_cast<const uint16_t*>(group + Gr::v_scale(8 * w.hi + 2 * t, g * NB / 8));
  }
  const int64_t kat = w.b * p.k_sb + w.h * p.k_sh + (w.i0 + g) * p.k_sn + t * 8;
  const int64_t vat = w.b * p.v_sb + w.h * p.v_sh + (w.i0 + 2 * t) * p.v_sn + g * (4 * NB);
  // rows from counts[b] on are zeros, whatever the page holds behind the sequence
  const bool k_real = group && w.real(g);
  const bool k_in = w.in(p, g);
  constexpr int SIZE = KIND == IAK_DT_F32 ? 4 : 2;
  auto put = [&](void* base, int64_t at, const unsigned* h, bool write) {      // one element at a time
    if (!write) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
      store_from_float(base, p.dtype, at + 2 * i, f.x);
      store_from_float(base, p.dtype, at + 2 * i + 1, f.y);
    }
  };
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    unsigned h[4];
    fp4_unpack4(kw[b], h);
    const unsigned tops = fp4_half_tops(ks[b / 2]), s = b % 2 ? fp4_scale_pair<1, 1>(tops) : fp4_scale_pair<0, 0>(tops);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = k_real ? mul2(h[i], s) : 0;
    char* to = static_cast<char*>(p.k) + (kat + 32 * b) * SIZE;
    if constexpr (KIND == kAny) put(p.k, kat + 32 * b, h, k_in);
    else if constexpr (KIND == IAK_DT_F32) store_sectors<1>(to, 32, as_floats(h), as_floats(h + 2), k_in);
    else if (k_in) __stcs(reinterpret_cast<uint4*>(to), as_16bit(h, p.dtype));
  }
  const bool real0 = group && w.real(2 * t), real1 = group && w.real(2 * t + 1);
  const bool in[2] = {w.in(p, 2 * t), w.in(p, 2 * t + 1)};
  const unsigned s = fp4_scale_pair<0, 1>(fp4_half_tops(vs));
  unsigned v[2][2 * NB];                      // the rows' channels as half pairs
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    unsigned h[4];
    fp4_unpack4(vw[j], h);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = mul2(h[i], s);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[0][2 * j + i] = real0 ? __byte_perm(h[2 * i], h[2 * i + 1], 0x5410) : 0;
      v[1][2 * j + i] = real1 ? __byte_perm(h[2 * i], h[2 * i + 1], 0x7632) : 0;
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t at = vat + r * p.v_sn;
    char* to = static_cast<char*>(p.v) + at * SIZE;
    constexpr int gap = 4 * NB * SIZE;        // bytes to the next g's channels
#pragma unroll
    for (int c = 0; c < NB / 2; ++c) {        // runs of 8 channels
      const unsigned* h = v[r] + 4 * c;
      if constexpr (KIND == kAny) put(p.v, at + 8 * c, h, in[r]);
      else if constexpr (KIND == IAK_DT_F32) store_sectors<4>(to + 32 * c, gap, as_floats(h), as_floats(h + 2), in[r]);
      else if constexpr (NB == 2) {
        if (in[r]) __stcs(reinterpret_cast<uint4*>(to), as_16bit(h, p.dtype));
      } else if (c % 2 == 0) {
        store_sectors<4>(to + 16 * c, gap, as_16bit(h, p.dtype), as_16bit(h + 4, p.dtype), in[r]);
      }
    }
  }
}

template <int NB>
int launch_rows(const RowsParams& p, bool append, bool vec, cudaStream_t s) {
  const int64_t per = kRowThreads / 32;
  const int64_t blocks = (static_cast<int64_t>(p.B) * p.Ht * p.octets + per - 1) / per;
  if (blocks > 0x7fffffffLL) return fail(IAK_ERR_UNSUPPORTED, "iak_fp4 rows: too many rows for one launch");
  const unsigned g = static_cast<unsigned>(blocks);
  if (append) {
    if (!vec) fp4_append_kernel<NB, kAny><<<g, kRowThreads, 0, s>>>(p);
    else if (p.dtype == IAK_DT_F32) fp4_append_kernel<NB, IAK_DT_F32><<<g, kRowThreads, 0, s>>>(p);
    else if (p.dtype == IAK_DT_F16) fp4_append_kernel<NB, IAK_DT_F16><<<g, kRowThreads, 0, s>>>(p);
    else fp4_append_kernel<NB, IAK_DT_BF16><<<g, kRowThreads, 0, s>>>(p);
  } else {
    if (!vec) fp4_read_kernel<NB, kAny><<<g, kRowThreads, 0, s>>>(p);
    else if (p.dtype == IAK_DT_F32) fp4_read_kernel<NB, IAK_DT_F32><<<g, kRowThreads, 0, s>>>(p);
    else fp4_read_kernel<NB, IAK_DT_F16><<<g, kRowThreads, 0, s>>>(p);
  }
  return check_cuda(cudaGetLastError(), append ? "fp4_append launch" : "fp4_read launch");
}

int rows_call(const iak_fp4_pool* pool, const iak_fp4_rows_args* a, bool append, void* stream) {
  const char* what = append ? "iak_fp4_append" : "iak_fp4_read";
  if (!pool || !a) return fail(IAK_ERR_INVALID_ARG, "%s: null arguments", what);
  if (int st = check_fp4_pool(pool, what)) return st;
  if (a->batch < 0 || a->num_table_heads < 0 || a->num_rows < 0 || a->table_width < 0)
    return fail(IAK_ERR_INVALID_ARG, "%s: negative size", what);
  if (a->dtype < IAK_DT_F32 || a->dtype > IAK_DT_BF16) return fail(IAK_ERR_INVALID_ARG, "%s: bad dtype", what);
  if (a->batch == 0 || a->num_table_heads == 0 || a->num_rows == 0) return IAK_OK;
  if (!a->k || !a->v || (a->table_width > 0 && !a->page_table))
    return fail(IAK_ERR_INVALID_ARG, "%s: null k, v or page_table", what);
  RowsParams p;
  p.pool = {static_cast<uint8_t*>(pool->data), pool->num_pages, pool->page_size, pool->head_dim};
  p.k = a->k; p.v = a->v; p.dtype = a->dtype;
  p.k_sb = a->k_stride_b; p.k_sh = a->k_stride_h; p.k_sn = a->k_stride_n;
  p.v_sb = a->v_stride_b; p.v_sh = a->v_stride_h; p.v_sn = a->v_stride_n;
  p.B = a->batch; p.Ht = a->num_table_heads; p.N = a->num_rows;
  p.pt = a->page_table; p.pt_sb = a->pt_stride_b; p.pt_sh = a->pt_stride_h; p.W = a->table_width;
  p.positions = a->positions; p.counts = a->counts; p.dropped = a->dropped;
  p.octets = (static_cast<int64_t>(a->num_rows) + 14) / 8;
  // 16-byte accesses need every row start on 16 bytes
  const int64_t per16 = a->dtype == IAK_DT_F32 ? 4 : 8;
  bool vec = reinterpret_cast<uintptr_t>(a->k) % 16 == 0 && reinterpret_cast<uintptr_t>(a->v) % 16 == 0;
  for (int64_t st : {p.k_sb, p.k_sh, p.k_sn, p.v_sb, p.v_sh, p.v_sn}) vec = vec && st % per16 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (pool->head_dim == 64) return launch_rows<2>(p, append, vec, s);
  if (pool->head_dim == 128) return launch_rows<4>(p, append, vec, s);
  return launch_rows<8>(p, append, vec, s);
}

}  // namespace

int check_fp4_pool(const iak_fp4_pool* pool, const char* what) {
  if (pool->head_dim != 64 && pool->head_dim != 128 && pool->head_dim != 256)
    return fail(IAK_ERR_UNSUPPORTED, "%s: head_dim %d is not 64, 128 or 256", what, pool->head_dim);
  if (pool->page_size <= 0 || pool->page_size % 16 || pool->page_size > kFp4MaxPage)
    return fail(IAK_ERR_UNSUPPORTED, "%s: page_size %d is not a multiple of 16 up to %d", what, pool->page_size, kFp4MaxPage);
  if (pool->num_pages < 0 || pool->num_pages > 0x7fffffffLL)
    return fail(IAK_ERR_INVALID_ARG, "%s: num_pages out of range", what);
  if (!pool->data && pool->num_pages > 0) return fail(IAK_ERR_INVALID_ARG, "%s: null pool data", what);
  if (reinterpret_cast<uintptr_t>(pool->data) % 16)
    return fail(IAK_ERR_INVALID_ARG, "%s: pool data must be 16-byte aligned", what);
  return IAK_OK;
}

}  // namespace iak

extern "C" int iak_fp4_append(const iak_fp4_pool* pool, const iak_fp4_rows_args* args, void* stream) {
  return iak::rows_call(pool, args, true, stream);
}

extern "C" int iak_fp4_read(const iak_fp4_pool* pool, const iak_fp4_rows_args* args, void* stream) {
  return iak::rows_call(pool, args, false, stream);
}
