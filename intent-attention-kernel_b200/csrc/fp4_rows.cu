// FP4 page pool: quantise-on-write of new rows (iak_fp4_append) and reading rows back (iak_fp4_read).
//
// Both are copies: per row and channel they move 2 * (element size + 17/32) bytes, which bounds them for long
// prompts; a decode step's few rows are bound by the launch.  A warp owns 8 aligned rows of K and V, its lanes what the
// attention kernel's lanes read of them: lane 4 g + t has row g's channels 32 b + 8 t .. + 7 of K (all blocks b) and
// channels 4 NB g .. of rows 2 t and 2 t + 1 of V.  Codes move as one run of 512 bytes (D 128) per plane, dense rows as
// 64-byte runs and more.  A V byte whose other row is not part of the call keeps that row's half.
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

template <bool VEC>
__device__ __forceinline__ void load8(const void* base, int dtype, int64_t at, float (&x)[8]) {
  if (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = load_as_float(base, dtype, at + i);
    return;
  }
  if (dtype == IAK_DT_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    const float4 a = __ldcs(p), b = __ldcs(p + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    return;
  }
  const uint4 w = __ldcs(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at));
  const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dtype == IAK_DT_F16) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x; x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = __uint_as_float(u[i] << 16); x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
}

template <bool VEC>
__device__ __forceinline__ void store8(void* base, int dtype, int64_t at, const float (&x)[8]) {
  if (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) store_from_float(base, dtype, at + i, x[i]);
    return;
  }
  if (dtype == IAK_DT_F32) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
    __stcs(p, make_float4(x[0], x[1], x[2], x[3]));
    __stcs(p + 1, make_float4(x[4], x[5], x[6], x[7]));
    return;
  }
  unsigned u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dtype == IAK_DT_F16) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      u[i] = *reinterpret_cast<const unsigned*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      u[i] = *reinterpret_cast<const unsigned*>(&h);
    }
  }
  __stcs(reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at), make_uint4(u[0], u[1], u[2], u[3]));
}

// Where a warp works: 8 rows of one (b, h), tokens 8 k .. 8 k + 7.  Row j is row i0 + j of the call's.
struct Place {
  int b, h;
  int64_t i0;             // negative where the rows begin before the call's
  int n;                  // rows of the call that are real: counts[b], at most N
  uint8_t* group;         // the 16 rows' bytes, or null: no such page
  int hi;                 // which 8 of them
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
  w.group = nullptr;
  if (tok0 >= 0 && w.i0 < w.n) {
    const int64_t slot = tok0 / p.pool.PS;
    if (slot < p.W) {
      const int id = p.pt[w.b * p.pt_sb + w.h * p.pt_sh + slot];
      if (id >= 0 && id < p.pool.num_pages)
        w.group = p.pool.data + ((static_cast<int64_t>(id) * p.pool.PS + (tok0 - slot * p.pool.PS)) >> 4) * Fp4Group<NB>::kBytes;
    }
  }
  return w.i0 < p.N;
}

__device__ __forceinline__ float largest8(float (&x)[8]) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = x[i] != x[i] ? 0.f : x[i];
    amax = fmaxf(amax, fabsf(x[i]));
  }
  return amax;
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

template <int NB, bool VEC>
__global__ void __launch_bounds__(kRowThreads) fp4_append_kernel(const RowsParams p) {
  using Gr = Fp4Group<NB>;
  Place w;
  if (!find_place<NB>(p, w)) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (!w.group) {
    if (p.dropped) {
      const int n = __popc(__ballot_sync(~0u, lane < 8 && w.real(lane)));
      if (lane == 0 && n) atomicAdd(p.dropped, n);
    }
    return;
  }
  constexpr int VC = NB / 2;                  // runs of 8 channels that a lane has of a V row
  const bool k_real = w.real(g), v_real0 = w.real(2 * t), v_real1 = w.real(2 * t + 1);
  float kx[NB][8], vx[2][VC][8];
  const int64_t kat = w.b * p.k_sb + w.h * p.k_sh + (w.i0 + g) * p.k_sn + t * 8;
  const int64_t vat = w.b * p.v_sb + w.h * p.v_sh + (w.i0 + 2 * t) * p.v_sn + g * (4 * NB);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) kx[b][i] = 0.f;
    if (k_real) load8<VEC>(p.k, p.dtype, kat + 32 * b, kx[b]);
  }
#pragma unroll
  for (int c = 0; c < VC; ++c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) vx[0][c][i] = vx[1][c][i] = 0.f;
    if (v_real0) load8<VEC>(p.v, p.dtype, vat + 8 * c, vx[0][c]);
    if (v_real1) load8<VEC>(p.v, p.dtype, vat + p.v_sn + 8 * c, vx[1][c]);
  }
  // K: a block's largest magnitude spans the row's 4 lanes
  unsigned word[NB];
  uint8_t scale[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    float amax = largest8(kx[b]);
    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
    scale[b] = static_cast<uint8_t>(fp4_scale_byte(amax));
    const float inv = fp4_inv_scale(scale[b]);            // a power of two: the product is exact
    word[b] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) word[b] |= fp4_pack2(kx[b][2 * i] * inv, kx[b][2 * i + 1] * inv) << (8 * i);
  }
  if (k_real) {
    put_words<NB>(w.group + w.hi * Gr::kSet, lane, word);
    if (t == 0) {
      uint8_t* to = w.group + Gr::k_scale(8 * w.hi + g, 0);
#pragma unroll
      for (int b = 0; b < NB; b += 2)
        *reinterpret_cast<uint16_t*>(to + b) = static_cast<uint16_t>(scale[b] | scale[b + 1] << 8);
    }
  }
  // V: a block spans 8 / NB neighbouring g
  int byte[2];
  float inv[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < VC; ++c) amax = fmaxf(amax, largest8(vx[r][c]));
    if (NB <= 4) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 4));
    if (NB <= 2) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 8));
    byte[r] = fp4_scale_byte(amax);
    inv[r] = fp4_inv_scale(byte[r]);
  }
  if (!v_real0 && !v_real1) return;
#pragma unroll
  for (int j = 0; j < NB; ++j) {              // byte of a channel: both rows' codes
    word[j] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = 4 * j + i;
      word[j] |= fp4_pack2(vx[0][c / 8][c % 8] * inv[0], vx[1][c / 8][c % 8] * inv[1]) << (8 * i);
    }
  }
  uint8_t* set = w.group + Gr::kV + w.hi * Gr::kSet;
  if (!(v_real0 && v_real1)) {                // the other row's half stays as it is
    unsigned old[NB];
    get_words<NB>(set, lane, old);
    const unsigned mine = v_real0 ? 0x0f0f0f0fu : 0xf0f0f0f0u;
#pragma unroll
    for (int j = 0; j < NB; ++j) word[j] = (word[j] & mine) | (old[j] & ~mine);
  }
  put_words<NB>(set, lane, word);
  if (g % (8 / NB) == 0) {
    uint8_t* to = w.group + Gr::v_scale(8 * w.hi + 2 * t, g * NB / 8);
    if (v_real0) to[0] = static_cast<uint8_t>(byte[0]);
    if (v_real1) to[1] = static_cast<uint8_t>(byte[1]);
  }
}

// scale byte (bytes) -> half 2^e in both halves (one in each): the pool's values are halves, so the products are exact
__device__ __forceinline__ unsigned half_scales(unsigned lo, unsigned hi) {
  return (lo | hi << 16) * 1024u - 112u * 1024u * 65537u;
}
__device__ __forceinline__ unsigned mul2(unsigned a, unsigned b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const unsigned*>(&r);
}
// 8 values held as half pairs
template <bool VEC>
__device__ __forceinline__ void store_halves(void* base, int dtype, int64_t at, const unsigned* h) {
  if (VEC && dtype == IAK_DT_F16) {
    __stcs(reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at), make_uint4(h[0], h[1], h[2], h[3]));
    return;
  }
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
  store8<VEC>(base, dtype, at, x);
}

template <int NB, bool VEC>
__global__ void __launch_bounds__(kRowThreads) fp4_read_kernel(const RowsParams p) {
  using Gr = Fp4Group<NB>;
  Place w;
  if (!find_place<NB>(p, w)) return;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  unsigned kw[NB] = {}, vw[NB] = {}, ks[NB / 2] = {}, vs = 0;
  if (w.group) {
    get_words<NB>(w.group + w.hi * Gr::kSet, lane, kw);
    get_words<NB>(w.group + Gr::kV + w.hi * Gr::kSet, lane, vw);
    const uint16_t* from = reinterpret_cast<const uint16_t*>(w.group + Gr::k_scale(8 * w.hi + g, 0));
#pragma unroll
    for (int b = 0; b < NB / 2; ++b) ks[b] = from[b];
    vs = *reinterpret_cast<const uint16_t*>(w.group + Gr::v_scale(8 * w.hi + 2 * t, g * NB / 8));
  }
  const int64_t kat = w.b * p.k_sb + w.h * p.k_sh + (w.i0 + g) * p.k_sn + t * 8;
  const int64_t vat = w.b * p.v_sb + w.h * p.v_sh + (w.i0 + 2 * t) * p.v_sn + g * (4 * NB);
  // rows from counts[b] on are zeros, whatever the page holds behind the sequence
  const bool k_real = w.group && w.real(g);
  if (w.in(p, g)) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      unsigned h[4];
      fp4_unpack4(kw[b], h);
      const unsigned byte = b % 2 ? ks[b / 2] >> 8 : ks[b / 2] & 255, s = half_scales(byte, byte);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = k_real ? mul2(h[i], s) : 0;
      store_halves<VEC>(p.k, p.dtype, kat + 32 * b, h);
    }
  }
  const bool real0 = w.group && w.real(2 * t), real1 = w.group && w.real(2 * t + 1);
  // (the byte of a row that was never written could borrow from the other half)
  const unsigned s = half_scales(real0 ? vs & 255 : 112, real1 ? vs >> 8 : 112);
#pragma unroll
  for (int c = 0; c < NB / 2; ++c) {          // 8 channels of both rows
    unsigned r0[4], r1[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      unsigned h[4];
      fp4_unpack4(vw[2 * c + j], h);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = mul2(h[i], s);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        r0[2 * j + i] = real0 ? __byte_perm(h[2 * i], h[2 * i + 1], 0x5410) : 0;
        r1[2 * j + i] = real1 ? __byte_perm(h[2 * i], h[2 * i + 1], 0x7632) : 0;
      }
    }
    if (w.in(p, 2 * t)) store_halves<VEC>(p.v, p.dtype, vat + 8 * c, r0);
    if (w.in(p, 2 * t + 1)) store_halves<VEC>(p.v, p.dtype, vat + p.v_sn + 8 * c, r1);
  }
}

template <int NB>
int launch_rows(const RowsParams& p, bool append, bool vec, cudaStream_t s) {
  const int64_t per = kRowThreads / 32;
  const int64_t blocks = (static_cast<int64_t>(p.B) * p.Ht * p.octets + per - 1) / per;
  if (blocks > 0x7fffffffLL) return fail(IAK_ERR_UNSUPPORTED, "iak_fp4 rows: too many rows for one launch");
  const unsigned g = static_cast<unsigned>(blocks);
  if (append) {
    if (vec) fp4_append_kernel<NB, true><<<g, kRowThreads, 0, s>>>(p);
    else fp4_append_kernel<NB, false><<<g, kRowThreads, 0, s>>>(p);
  } else {
    if (vec) fp4_read_kernel<NB, true><<<g, kRowThreads, 0, s>>>(p);
    else fp4_read_kernel<NB, false><<<g, kRowThreads, 0, s>>>(p);
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
