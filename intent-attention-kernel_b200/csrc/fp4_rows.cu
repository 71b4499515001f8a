// FP4 page pool: quantise-on-write of new rows (iak_fp4_append) and reading rows back (iak_fp4_read).
//
// Both are copies: per row and channel they move 2 * (element size + 17/32) bytes, which bounds them for long
// prompts; a decode step's few rows are bound by the launch.  One thread owns 8 channels of the two rows 2i and
// 2i + 1, which share their bytes of V: it moves 16 bytes of each of the four dense rows, independent of one another.
// A warp has 4 such row pairs by 64 channels, so that it covers 128-byte runs of the dense rows (16-bit types) and
// 64-byte runs of the group.  A block's largest magnitude spans 4 neighbouring lanes.  A V byte whose other row is not
// part of the call keeps that row's half.
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

// where a thread works: its (b, h), row pair and 8 channels; tokens are 64-bit
struct Place {
  int b, h, l;            // l: which 8 channels
  int64_t i0;             // the pair's first row among the call's (negative when it starts before them)
  bool in0, in1;          // rows that the call covers (index in [0, N))
  bool real0, real1;      // rows below counts[b]
  uint8_t* group;         // the 16 rows' bytes, or null: no such page
  int row;                // of the group, even
};

template <int NB>
__device__ __forceinline__ bool find_place(const RowsParams& p, Place& w) {
  constexpr int LP = NB * 16;                // threads of 8 rows: 4 row pairs, D / 8 channel runs
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (kRowThreads / LP) + threadIdx.x / LP;
  const int64_t bh = at / p.octets;
  if (bh >= static_cast<int64_t>(p.B) * p.Ht) return false;   // whole groups of LP threads leave together
  w.l = (threadIdx.x % LP / 32) * 8 + (threadIdx.x & 7);
  w.b = static_cast<int>(bh / p.Ht);
  w.h = static_cast<int>(bh - static_cast<int64_t>(w.b) * p.Ht);
  const int64_t pos = p.positions ? p.positions[w.b] : 0;
  const int n = p.counts ? min(max(p.counts[w.b], 0), p.N) : p.N;
  const int64_t tok0 = (pos & ~int64_t(7)) + 8 * (at - bh * p.octets) + 2 * ((threadIdx.x >> 3) & 3);
  w.i0 = tok0 - pos;
  w.in0 = w.i0 >= 0 && w.i0 < p.N;
  w.in1 = w.i0 + 1 >= 0 && w.i0 + 1 < p.N;
  w.real0 = w.in0 && w.i0 < n;
  w.real1 = w.in1 && w.i0 + 1 < n;
  w.group = nullptr;
  w.row = static_cast<int>(tok0 & 15);       // page sizes are multiples of 16: so are pages' first tokens
  if (tok0 >= 0 && (w.real0 || w.real1)) {
    const int64_t slot = tok0 / p.pool.PS;
    if (slot < p.W) {
      const int id = p.pt[w.b * p.pt_sb + w.h * p.pt_sh + slot];
      if (id >= 0 && id < p.pool.num_pages)
        w.group = p.pool.data + ((static_cast<int64_t>(id) * p.pool.PS + (tok0 - slot * p.pool.PS)) >> 4) * Fp4Group<NB>::kBytes;
    }
  }
  return w.in0 || w.in1;                     // the 4 lanes of a block agree
}

// 8 values of a block of 4 lanes -> their codes (value i in bits 4i) and the block's scale byte
__device__ __forceinline__ unsigned quantize8(float (&x)[8], int& byte) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = x[i] != x[i] ? 0.f : x[i];
    amax = fmaxf(amax, fabsf(x[i]));
  }
  const unsigned group = 0xfu << (threadIdx.x & 28);      // the block's lanes: all of them are here
  amax = fmaxf(amax, __shfl_xor_sync(group, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(group, amax, 2));
  byte = fp4_scale_byte(amax);
  const float inv = fp4_inv_scale(byte);                  // a power of two: the product is exact
  unsigned w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= fp4_pack2(x[2 * i] * inv, x[2 * i + 1] * inv) << (8 * i);
  return w;
}

// bits 4i of a and b interleaved: byte i = a's code i (low half), b's code i (high half), i = 0..3
__device__ __forceinline__ unsigned zip_codes(unsigned a, unsigned b) {
  unsigned r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= (((a >> (4 * i)) & 15u) | (((b >> (4 * i)) & 15u) << 4)) << (8 * i);
  return r;
}

template <int NB, bool VEC>
__global__ void __launch_bounds__(kRowThreads) fp4_append_kernel(const RowsParams p) {
  Place w;
  if (!find_place<NB>(p, w)) return;
  if (!w.group) {
    if (p.dropped && w.l == 0) {
      const int n = (w.real0 ? 1 : 0) + (w.real1 ? 1 : 0);
      if (n) atomicAdd(p.dropped, n);
    }
    return;
  }
  const int blk = w.l >> 2, t = w.l & 3;      // the thread's block and its word of the block
  float k0[8] = {}, k1[8] = {}, v0[8] = {}, v1[8] = {};
  const int64_t kat = w.b * p.k_sb + w.h * p.k_sh + w.i0 * p.k_sn + w.l * 8;
  const int64_t vat = w.b * p.v_sb + w.h * p.v_sh + w.i0 * p.v_sn + w.l * 8;
  if (w.real0) {
    load8<VEC>(p.k, p.dtype, kat, k0);
    load8<VEC>(p.v, p.dtype, vat, v0);
  }
  if (w.real1) {
    load8<VEC>(p.k, p.dtype, kat + p.k_sn, k1);
    load8<VEC>(p.v, p.dtype, vat + p.v_sn, v1);
  }
  int kb0, kb1, vb0, vb1;
  const unsigned kw0 = quantize8(k0, kb0), kw1 = quantize8(k1, kb1);
  const unsigned vw0 = quantize8(v0, vb0), vw1 = quantize8(v1, vb1);
  using Gr = Fp4Group<NB>;
  if (w.real0) *reinterpret_cast<uint32_t*>(w.group + Gr::k_word(w.row, blk, t)) = kw0;
  if (w.real1) *reinterpret_cast<uint32_t*>(w.group + Gr::k_word(w.row + 1, blk, t)) = kw1;
  uint2* vrow = reinterpret_cast<uint2*>(w.group + Gr::v_bytes(w.row, w.l * 8));
  uint2 vz = make_uint2(zip_codes(vw0, vw1), zip_codes(vw0 >> 16, vw1 >> 16));
  if (!(w.real0 && w.real1)) {                // the other row's half stays as it is
    const uint2 old = *vrow;
    const unsigned mine = w.real0 ? 0x0f0f0f0fu : 0xf0f0f0f0u;
    vz.x = (vz.x & mine) | (old.x & ~mine);
    vz.y = (vz.y & mine) | (old.y & ~mine);
  }
  *vrow = vz;
  if (t == 0) {
    if (w.real0) {
      w.group[Gr::k_scale(w.row, blk)] = static_cast<uint8_t>(kb0);
      w.group[Gr::v_scale(w.row, blk)] = static_cast<uint8_t>(vb0);
    }
    if (w.real1) {
      w.group[Gr::k_scale(w.row + 1, blk)] = static_cast<uint8_t>(kb1);
      w.group[Gr::v_scale(w.row + 1, blk)] = static_cast<uint8_t>(vb1);
    }
  }
}

__device__ __forceinline__ void dequant_k(unsigned w, float s, float (&x)[8]) {
  unsigned h[4];
  fp4_unpack4(w, h);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    x[2 * i] = f.x * s;
    x[2 * i + 1] = f.y * s;
  }
}

__device__ __forceinline__ void dequant_v(uint2 w, float s0, float s1, float (&x0)[8], float (&x1)[8]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    unsigned h[4];
    fp4_unpack4(j ? w.y : w.x, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
      x0[4 * j + i] = f.x * s0;
      x1[4 * j + i] = f.y * s1;
    }
  }
}

template <int NB, bool VEC>
__global__ void __launch_bounds__(kRowThreads) fp4_read_kernel(const RowsParams p) {
  Place w;
  if (!find_place<NB>(p, w)) return;
  float k0[8] = {}, k1[8] = {}, v0[8] = {}, v1[8] = {};
  if (w.group) {
    using Gr = Fp4Group<NB>;
    const int blk = w.l >> 2, t = w.l & 3;
    const unsigned kw0 = *reinterpret_cast<const uint32_t*>(w.group + Gr::k_word(w.row, blk, t));
    const unsigned kw1 = *reinterpret_cast<const uint32_t*>(w.group + Gr::k_word(w.row + 1, blk, t));
    const uint2 vz = *reinterpret_cast<const uint2*>(w.group + Gr::v_bytes(w.row, w.l * 8));
    const uint16_t vs = *reinterpret_cast<const uint16_t*>(w.group + Gr::v_scale(w.row, blk));
    dequant_k(kw0, fp4_scale(w.group[Gr::k_scale(w.row, blk)]), k0);
    dequant_k(kw1, fp4_scale(w.group[Gr::k_scale(w.row + 1, blk)]), k1);
    dequant_v(vz, fp4_scale(vs & 255), fp4_scale(vs >> 8), v0, v1);
    // rows from counts[b] on are zeros, whatever the page holds behind the sequence
    if (!w.real0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) k0[i] = v0[i] = 0.f;
    }
    if (!w.real1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) k1[i] = v1[i] = 0.f;
    }
  }
  const int64_t kat = w.b * p.k_sb + w.h * p.k_sh + w.i0 * p.k_sn + w.l * 8;
  const int64_t vat = w.b * p.v_sb + w.h * p.v_sh + w.i0 * p.v_sn + w.l * 8;
  if (w.in0) {
    store8<VEC>(p.k, p.dtype, kat, k0);
    store8<VEC>(p.v, p.dtype, vat, v0);
  }
  if (w.in1) {
    store8<VEC>(p.k, p.dtype, kat + p.k_sn, k1);
    store8<VEC>(p.v, p.dtype, vat + p.v_sn, v1);
  }
}

template <int NB>
int launch_rows(const RowsParams& p, bool append, bool vec, cudaStream_t s) {
  const int64_t per = kRowThreads / (NB * 16);
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
  if (pool->page_size <= 0 || pool->page_size % 16)
    return fail(IAK_ERR_UNSUPPORTED, "%s: page_size %d is not a multiple of 16", what, pool->page_size);
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
