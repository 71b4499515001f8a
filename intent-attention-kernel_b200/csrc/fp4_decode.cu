// Attention of a sequence's last tokens over an FP4 page pool (iak_fp4_decode), plain and differential.
//
// Mathematics.  A table head's queries form NC = G * M * (1 or 2) softmax columns (differential: two per query, the
// first with q2 = 0 and the second with q1 = 0, so that both halves run as one product).  Per tile of 32 keys
//   S' = K Q',  P = exp2(c (S - m) + 7),  O' += V' P'
// with running maximum m and sum l per column, fp32, c the softmax scale: the difference is taken before the scale, so
// that scores of any size keep their distances (a maximum rounded after it lies whole units off from 2^24 on).  Keys are the rows of the first product and the contraction of
// the second, columns the narrow side (n = 8 per mma.m16n8k16), so that few queries waste little.
//   K: a lane's 32-bit word holds 8 channels of one row; the byte pairs become half pairs in one conversion each, and
//      a row's block scale 2^e multiplies the fp32 product of its 32 channels (4 lanes x 8), not its elements.
//   V: a byte holds one channel of two neighbouring keys, so that its half pair lies along the contraction; it is
//      multiplied by the two keys' scales (exact: the pool's values are halves).
//   P: rounded to halves (fp32 queries: the sum of two), from the accumulator's layout to the operand's by movmatrix.
//   m is raised only when c (S - m) passes 8 (P up to 2^15), which leaves the rescaling of O to few tiles.
// What bounds it: the cache's bytes, 4.25 bits an element, and close behind them the issue slots: of 233 per 16
// rows at D 128 and 8 columns a warp spends 64 on conversions, 32 on V's scales, 16 on K's and 16 on products.
// Work is cut into equal runs of steps over all (sequence, table head, column group) units, one for each resident warp,
// so that ragged batches, many short sequences and one long sequence fill the GPU alike.  A step is a tile; what a unit
// costs besides its tiles counts as three (256 sequences of up to 512 tokens: 31 us, with equal runs of tiles 44; 16 of up
// to 8001 with 4 queries and D 256: 43 against 48).  A unit cut over several runs
// leaves partial (m, l, O) that a second kernel adds in order of the runs (no atomics: results do not depend on timing).
// Warps share nothing: with units cut per block of 8 warps, their sums joined in shared memory, 256 sequences of up to
// 700 tokens took 87 us instead of 39.
// Each warp streams its tiles through a ring of 16-byte asynchronous copies: a group's codes and scales lie together in
// the order in which lanes read them, so that copies and reads are linear in the lane, free of bank conflicts, and five
// copies per 16 rows need one address.  (Bulk copies with an mbarrier measured the same at D 128 and slower at D 64, 70 us
// against 66 for 16 sequences of 32k; they would need bounded waits besides.)
// 32 sequences of up to 32k tokens, 32 query and 8 table heads, D 128, launched one after another: 135 us, 5.9 TB/s; 64 of
// 32k 366 us, 6.2 TB/s; one of 512k 102 us, 5.6 TB/s; 4096 of 256 tokens 245 us, 4.7 TB/s.
#include <algorithm>
#include <cfloat>
#include <mutex>

#include "fp4.cuh"
#include "tc_ptx.cuh"

namespace iak {
namespace {

constexpr int kTileKeys = 32;      // keys of a warp's tile: two groups of 16
constexpr int kMaxTokens = 1 << 30; // of a table row: token numbers stay 32-bit
constexpr int kDirectTiles = 8;    // units of at most so many tiles are never cut
constexpr int kOpen = 3;           // a unit's queries, first copies and output take a warp as long as so many tiles
constexpr float kHead = 7.f;       // the maximum's own P is 2^7, so that small P stay normal halves
constexpr float kLazy = 15.f;      // P may grow to 2^15 before the maximum is raised
// Of a column.  With the least, -FLT_MAX as the first maximum still is raised by every score; with the
// largest (products of scale and queries beyond fp32) equal scores keep their equal weights.
constexpr float kScaleMin = 1e-37f, kScaleMax = FLT_MAX;

struct DecP {
  Fp4Pool pool;
  int gpp;                           // groups of 16 rows per page, at most 2^10
  unsigned long long gpp_inv;        // 2^36 / gpp, rounded up
  const void* q; int q_dtype; int64_t q_sb, q_sh, q_sm;
  void* out; int out_dtype; int64_t o_sb, o_sh, o_sm;
  int B, Ht, G, M;
  const int32_t* pt; int64_t pt_sb, pt_sh; int W;
  const int32_t* lengths;
  float scale;                       // |sm_scale| * log2(e)
  float sign;                        // of sm_scale
  int diff; const float* lam; const float* norm_w; float eps, out_scale;
  int NC;                            // softmax columns of a table head
  int CG;                            // column groups of 8 * NT
  int HC;                            // units of a sequence: Ht * CG
  int cols;                          // columns of a unit's partials: min(8 * NT, NC)
  int q_vec, o_vec;                  // 16-byte accesses to q (out) are aligned
  int runs;                          // warps of the main kernel
  int direct;                        // a warp per unit, nothing to join
  int by_unit;                       // cuts are recorded per unit, not per border
  int min_steps;                     // of a run, at least
  float* ws;
};

// ------------------------------------------------------------------ schedule
__device__ __forceinline__ int seq_len(const DecP& p, int b) {
  return min(max(p.lengths[b], 0), p.W * p.pool.PS);
}
// tiles of one unit; an empty sequence has one, which writes its zeros
__device__ __forceinline__ int tiles_of(const DecP& p, int len) {
  return max(1, (len + kTileKeys - 1) / kTileKeys);
}
// A unit's steps: kOpen for what a warp does before and after its tiles, then the tiles.
__device__ __forceinline__ int steps_of(const DecP& p, int len) { return tiles_of(p, len) + kOpen; }

// Table entry of group g: g / gpp, exact for g < 2^26 and gpp <= 2^10, where g times the inverse's excess stays below 2^36.
__device__ __forceinline__ int slot_of(const DecP& p, int g) {
  return static_cast<int>((static_cast<unsigned>(g) * p.gpp_inv) >> 36);
}

// Inclusive sum over the lanes before and this one.
__device__ __forceinline__ int lanes_upto(int n) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(~0u, n, o);
    if (lane >= o) n += v;
  }
  return n;
}
// Where a run's tiles lie is found in the steps of all units.  A warp's lane holds the steps of one sequence (up to 32
// of them, chunk 0), or of four threads' sequences: a block's thread i adds up those from i * chunk on, in `sums`; upto
// counts with all lanes before.  (With sums of its own for each warp, the join's too, 4096 sequences of 256 tokens took
// 365 us instead of 248.)
constexpr int kScan = 128;
struct Lanes { int chunk; int4 n; int upto, len; };
__device__ __forceinline__ int four(const int4& n) { return n.x + n.y + n.z + n.w; }
__device__ __forceinline__ Lanes scan_batch(const DecP& p, int* sums) {
  Lanes s;
  s.len = 0;
  if (p.B <= 32) {
    s.chunk = 0;
    s.n = make_int4(0, 0, 0, 0);
    const int b = threadIdx.x & 31;
    if (b < p.B) {
      s.len = seq_len(p, b);
      s.n.x = steps_of(p, s.len) * p.HC;
    }
  } else {
    s.chunk = (p.B + kScan - 1) / kScan;
    int n = 0;
    const int first = threadIdx.x * s.chunk;
#pragma unroll 8
    for (int b = first; b < min(first + s.chunk, p.B); ++b) n += steps_of(p, seq_len(p, b));
    sums[threadIdx.x] = n * p.HC;
    __syncthreads();
    s.n = reinterpret_cast<const int4*>(sums)[threadIdx.x & 31];
  }
  s.upto = lanes_upto(four(s.n));
  return s;
}
// all steps of the call; the host keeps their number within 31 bits
__device__ __forceinline__ int total_steps(const Lanes& s) { return __shfl_sync(~0u, s.upto, 31); }
// the sequence that holds step t, its length, and t's offset among its steps
__device__ __forceinline__ void find_sequence(const DecP& p, const Lanes& s, int t, int& b, int& len, int& off) {
  const int lane = threadIdx.x & 31;
  const int l = __ffs(__ballot_sync(~0u, s.upto > t)) - 1;       // t < total: some lane has it
  int before = __shfl_sync(~0u, s.upto - four(s.n), l);
  if (s.chunk == 0) {
    b = l;
    len = __shfl_sync(~0u, s.len, l);
    off = t - before;
    return;
  }
  const int n0 = __shfl_sync(~0u, s.n.x, l), n1 = __shfl_sync(~0u, s.n.y, l), n2 = __shfl_sync(~0u, s.n.z, l);
  b = 4 * l;
  if (t >= before + n0) {
    before += n0;
    ++b;
    if (t >= before + n1) {
      before += n1;
      ++b;
      if (t >= before + n2) {
        before += n2;
        ++b;
      }
    }
  }
  b *= s.chunk;
  if (s.chunk == 1) {
    len = seq_len(p, b);
  } else {
    const int end = min(b + s.chunk, p.B);
    for (; b < end; b += 32) {
      const int own = b + lane < end ? seq_len(p, b + lane) : 0;
      const int n = b + lane < end ? steps_of(p, own) * p.HC : 0, upto = lanes_upto(n);
      const unsigned hit = __ballot_sync(~0u, before + upto > t);
      if (hit) {
        const int k = __ffs(hit) - 1;
        b += k;
        len = __shfl_sync(~0u, own, k);
        before += __shfl_sync(~0u, upto - n, k);
        break;
      }
      before += __shfl_sync(~0u, upto, 31);
    }
  }
  off = t - before;
}

// The steps in equal runs, one for each of `used` warps, the first `more` of them with each + 1.
struct Runs { int used, each, more; };
__device__ __forceinline__ Runs make_runs(const DecP& p, int total) {
  Runs r;
  r.used = static_cast<int>(min((static_cast<unsigned>(total) + p.min_steps - 1) / p.min_steps, static_cast<unsigned>(p.runs)));
  r.each = total / r.used;
  r.more = total - r.each * r.used;
  return r;
}
__device__ __forceinline__ int run_begin(const Runs& r, int i) { return i * r.each + min(i, r.more); }
__device__ __forceinline__ int run_of(const Runs& r, int t) {
  const int large = r.more * (r.each + 1);
  return t < large ? t / (r.each + 1) : r.more + (t - large) / r.each;
}

// A run leaves at most two parts of units: [0] of the unit that it begins in, [1] of the one that it ends in.  A part
// is D sums, the maximum, the sum of the weights and the scale for each column.
__device__ __forceinline__ float* part_at(const DecP& p, int run, int which, int col) {
  return p.ws + ((static_cast<int64_t>(run) * 2 + which) * p.cols + col) * (p.pool.D + 4);
}
// What the join kernel reads of a unit cut over several runs.  Where there are no more units than runs a record per
// unit, written by the run that has its first tile; else one per border between two runs, written by the run that the
// border begins (all of them have tiles then) and empty unless it is a unit's first cut.
struct Cut { int b, h, j0, first, which, last; };   // first, last: runs with a part; which: first's; last < 0: none
__device__ __forceinline__ Cut* cuts(const DecP& p) {
  return reinterpret_cast<Cut*>(p.ws + static_cast<int64_t>(p.runs) * 2 * p.cols * (p.pool.D + 4));
}

// ---------------------------------------------------------------------- PTX
__device__ __forceinline__ void mma16816(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                         unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same product on its own: d = A B
__device__ __forceinline__ void mma16816_new(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3,
                                             unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ unsigned transpose8x8(unsigned x) {
  unsigned r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ unsigned pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ unsigned mul_half2(unsigned a, unsigned b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const unsigned*>(&r);
}
// four scale bytes e + 127 -> 2^e: two conversions to bf16 pairs, whose bits are the upper halves of the floats
__device__ __forceinline__ void scales4(unsigned w, float* s) {
  unsigned lo, hi;
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.bf16x2.ue8m0x2 %0, a;\ncvt.rn.bf16x2.ue8m0x2 %1, b;\n}"
      : "=r"(lo), "=r"(hi) : "r"(w));
  s[0] = __uint_as_float(lo << 16);
  s[1] = __uint_as_float(lo & 0xffff0000u);
  s[2] = __uint_as_float(hi << 16);
  s[3] = __uint_as_float(hi & 0xffff0000u);
}
__device__ __forceinline__ unsigned lds32(unsigned a) {
  unsigned r;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ void copy16(unsigned dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// a volatile statement, as the reads of the copied bytes are: they keep their order
__device__ __forceinline__ void warp_sync() { asm volatile("bar.warp.sync 0xffffffff;" ::: "memory"); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Pairs of floats, one instruction for both: c (s - m) + 7 (the difference before the scale is what an fma alone would
// leave out, at no more instructions than it), and sums.
__device__ __forceinline__ void exponents(const float* s, const float* m, const float* c, float* e) {
  asm("{\n.reg .b64 s, m, c, h;\nmov.b64 s, {%2, %3};\nmov.b64 m, {%4, %5};\nmov.b64 c, {%6, %7};\nmov.b64 h, {%8, %8};\n"
      "sub.rn.f32x2 s, s, m;\nfma.rn.f32x2 s, s, c, h;\nmov.b64 {%0, %1}, s;\n}"
      : "=f"(e[0]), "=f"(e[1])
      : "f"(s[0]), "f"(s[1]), "f"(m[0]), "f"(m[1]), "f"(c[0]), "f"(c[1]), "f"(kHead));
}
__device__ __forceinline__ void add_pair(float* a, const float* b) {
  asm("{\n.reg .b64 a, b;\nmov.b64 a, {%0, %1};\nmov.b64 b, {%2, %3};\nadd.rn.f32x2 a, a, b;\nmov.b64 {%0, %1}, a;\n}"
      : "+f"(a[0]), "+f"(a[1]) : "f"(b[0]), "f"(b[1]));
}
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int NW>
__device__ __forceinline__ void lds_words(unsigned a, unsigned (&w)[NW]) {
  if constexpr (NW == 1) {
    w[0] = lds32(a);
  } else if constexpr (NW == 2) {
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
  } else {
    static_assert(NW == 4, "words per access");
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a));
  }
}

// ------------------------------------------------------------- shared layout
struct Cursor { int left, off, at, b, len; };   // steps left to the run; the next one, of sequence b and of all
struct Segment { int b, h, cg, len, n_tiles, c_begin, c_end, at; };   // at: the unit's first step, of all

// What a kernel for D = 32 NB, 8 NT columns a unit and (SPLIT) fp32 queries is made of.  Warps work alone; a block has
// four so that an SM's share can be cut finely.
template <int NB, int NT, bool SPLIT>
struct Shape {
  using Gr = Fp4Group<NB>;
  static constexpr int D = NB * 32, COLS = 8 * NT;
  static constexpr int kWarps = 4;
  static constexpr int kThreads = kWarps * 32;
  // Warps of an SM: 16 with 128 registers each while the accumulators are small, 12 with 168, 8 with 255.  A tile's two
  // groups of 16 keys go through the products together, for the independent work.  Measured when chosen:
  //   D 128, 8 columns, 32 sequences of up to 32k: 139 us with 12 warps, 141 with 16 and a stage less
  //   D 128, 16 columns, 8 sequences of 32k: 80 us with 8, 83 with 12; fp32 queries, 8 columns: 71 with 12, 75 with 8
  //   D 64, 32 columns, 16 sequences of 32k: 150 us with 8, 153 with 12, 196 with 16
  static constexpr int kSize = NB * NT * (SPLIT ? 2 : 1);
  // steps of a run, at least: wide heads' parts cost more to join
  static constexpr int kMinSteps = NB == 8 ? 4 : 1;
  static_assert(kMinSteps <= kOpen + 1, "with more units than runs every run has more than kOpen steps, so a tile");
  static constexpr int kPerSm = kSize <= 4 && NB == 2 ? 16 : (kSize <= (SPLIT ? 8 : 4) && NB < 8 ? 12 : 8);
  static constexpr int kBlocks = kPerSm / kWarps;
  static constexpr int kStages = NB == 8 ? 2 : 3;
  static constexpr int kStage = 2 * Gr::kBytes;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kQuery = NT * NB * 512 * (SPLIT ? 2 : 1);
  static constexpr int kWarpBytes = kRing + kQuery;        // a multiple of 128
  static constexpr int kOwnBytes = kWarpBytes + static_cast<int>(sizeof(Cursor)) + static_cast<int>(sizeof(Segment));
  static constexpr int kSmem = kWarps * kOwnBytes + kScan * static_cast<int>(sizeof(int));
  static_assert(kThreads == kScan && kWarps * kOwnBytes % 16 == 0, "the block's sums of the batch");
  static_assert(kWarpBytes % 128 == 0, "copies and reads are linear runs of 128 bytes");
  static_assert(kBlocks * (kSmem + 1024) <= 228 * 1024, "shared memory of an SM");
};

// 1 / sqrt(mean square + eps) of a row with sum of squares sq (a row of zeros stays zero with eps 0)
template <int NB>
__device__ __forceinline__ float norm_factor(const DecP& p, float sq) {
  const float ms = sq * (1.f / (NB * 32)) + p.eps;
  return ms > 0.f || ms != ms ? rsqrtf(ms) : 0.f;
}

// x: one row's D values, lane i holding channels i, i + 32, ..
template <int NB>
__device__ __forceinline__ void finish_row(const DecP& p, int b, int head, int m, float (&x)[NB]) {
  const int lane = threadIdx.x & 31;
  if (p.diff) {
    float mul = p.out_scale;
    if (p.norm_w) {
      float sq = 0.f;
#pragma unroll
      for (int i = 0; i < NB; ++i) sq = fmaf(x[i], x[i], sq);
#pragma unroll
      for (int o = 16; o; o >>= 1) sq += __shfl_xor_sync(~0u, sq, o);
      mul *= norm_factor<NB>(p, sq);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) x[i] *= p.norm_w ? mul * p.norm_w[i * 32 + lane] : mul;
  }
  const int64_t at = b * p.o_sb + head * p.o_sh + m * p.o_sm;
#pragma unroll
  for (int i = 0; i < NB; ++i) store_from_float(p.out, p.out_dtype, at + i * 32 + lane, x[i]);
}

__device__ __forceinline__ float safe_inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// Of two maps' outputs, each rounded before (__fmul_rn keeps the compiler from fusing them in): equal maps of weight 1
// leave exactly 0, not the rounding of one product, which a norm without eps would make a whole row of.
__device__ __forceinline__ float difference(float x1, float lam, float x2) { return fmaf(-lam, x2, x1); }

// x: N neighbouring values of an output row, from element `at` on
template <int N>
__device__ __forceinline__ void store_run(const DecP& p, int64_t at, const float (&x)[N]) {
  if (!p.o_vec) {
#pragma unroll
    for (int i = 0; i < N; ++i) store_from_float(p.out, p.out_dtype, at + i, x[i]);
  } else if (p.out_dtype == IAK_DT_F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 8) {
      unsigned u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (p.out_dtype == IAK_DT_F16) {
          u[k] = pack_half2(x[i + 2 * k], x[i + 2 * k + 1]);
        } else {
          const __nv_bfloat162 v = __floats2bfloat162_rn(x[i + 2 * k], x[i + 2 * k + 1]);
          u[k] = *reinterpret_cast<const unsigned*>(&v);
        }
      }
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at + i) = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
}

// ---------------------------------------------------------------- main kernel
template <int NB, int NT, bool SPLIT>
__global__ void __launch_bounds__(Shape<NB, NT, SPLIT>::kThreads, Shape<NB, NT, SPLIT>::kBlocks)
fp4_decode_kernel(const DecP p) {
  using L = Shape<NB, NT, SPLIT>;
  using Gr = typename L::Gr;
  constexpr int D = L::D, MT = D / 16, COLS = L::COLS, kWarps = L::kWarps;
  extern __shared__ __align__(128) char smem[];   // (no static shared memory: it would move the rings off their 128 bytes)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int run = blockIdx.x * kWarps + warp;
  char* const q_frag = smem + warp * L::kWarpBytes + L::kRing;      // [hi, lo][NT][NB][lane] 16 bytes
  Cursor& cursor = reinterpret_cast<Cursor*>(smem + kWarps * L::kWarpBytes)[warp];
  Segment& segment = reinterpret_cast<Segment*>(smem + kWarps * (L::kWarpBytes + sizeof(Cursor)))[warp];
  const unsigned ring = static_cast<unsigned>(__cvta_generic_to_shared(smem)) + warp * L::kWarpBytes;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ------------------------------------------------------------- segments
  // A segment is the run's share of one unit's tiles.  What only its ends need lies in shared memory.
  Runs runs = {};
  {
    Cursor cur = {};
    if (p.direct) {
      cur.b = run / p.HC;
      if (cur.b >= p.B) return;
      cur.len = seq_len(p, cur.b);
      cur.left = steps_of(p, cur.len);
      cur.off = (run - cur.b * p.HC) * cur.left;
    } else {
      const Lanes s = scan_batch(p, reinterpret_cast<int*>(smem + kWarps * L::kOwnBytes));
      runs = make_runs(p, total_steps(s));
      if (run >= runs.used) {
        if (lane == 0 && !p.by_unit) cuts(p)[run] = {0, 0, 0, 0, 0, -1};
        return;
      }
      cur.at = run_begin(runs, run);
      cur.left = run_begin(runs, run + 1) - cur.at;
      find_sequence(p, s, cur.at, cur.b, cur.len, cur.off);
    }
    if (lane == 0) cursor = cur;
    __syncwarp();
  }

  // ---------------------------------------------------------------- copies
  // Of every 16 tiles lane 2 i + u looks up group u of tile i: it reads the page id a batch ahead and holds the group's
  // number in the pool (0 for a page that does not exist: its rows are masked).
  int n_mine = 0;                                 // tiles of the segment that are copied
  int stage = 0;                                  // of the ring, next to be read
  int next_id = -1, src_group = 0;
  unsigned history = 0;                           // two bits per tile issued, the last in bits 0, 1: its groups' pages exist
  constexpr int kBatch = 16;
  unsigned batch_ok = 0;
  const uint8_t* const lane_data = p.pool.data + lane * 16;
  auto group_of = [&](int k) { return (segment.c_begin + k + (lane >> 1)) * 2 + (lane & 1); };
  auto load_id = [&](int k) {
    const int gr = group_of(k);
    return k + (lane >> 1) < n_mine && gr * 16 < segment.len
               ? __ldg(p.pt + segment.b * p.pt_sb + segment.h * p.pt_sh + slot_of(p, gr)) : -1;
  };
  auto issue = [&](int k, int to_stage) {
    history <<= 2;
    if (k < n_mine) {
      const int i = k % kBatch;
      if (i == 0) {
        const bool ok = next_id >= 0 && next_id < p.pool.num_pages;
        const int gr = group_of(k);
        src_group = ok ? next_id * p.gpp + gr - slot_of(p, gr) * p.gpp : 0;
        batch_ok = __ballot_sync(~0u, ok);
        next_id = load_id(k + kBatch);
      }
      history |= (batch_ok >> (2 * i)) & 3;
      const unsigned to = ring + to_stage * L::kStage + lane * 16;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint8_t* from = lane_data + static_cast<int64_t>(__shfl_sync(~0u, src_group, 2 * i + u)) * Gr::kBytes;
#pragma unroll
        for (int c = 0; c < Gr::kBytes / 512; ++c) copy16(to + u * Gr::kBytes + c * 512, from + c * 512);
        constexpr int rest = Gr::kBytes % 512 / 16;               // lanes of the last copy
        if (lane < rest) copy16(to + u * Gr::kBytes + Gr::kBytes / 512 * 512, from + Gr::kBytes / 512 * 512);
      }
    }
    copy_commit();
  };
  auto read_words = [&](unsigned at, unsigned (&w)[NB]) {
    constexpr int PW = Gr::kPW;
#pragma unroll
    for (int i = 0; i < NB / PW; ++i) {
      unsigned part[PW];
      lds_words<PW>(at + (i * 32 + lane) * (PW * 4), part);
#pragma unroll
      for (int j = 0; j < PW; ++j) w[i * PW + j] = part[j];
    }
  };
  // the segment's column `col`: its query row, and the tokens that it sees
  auto row_of = [&](int col) { return p.diff ? (segment.cg * COLS + col) >> 1 : segment.cg * COLS + col; };
  auto limit = [&](int col) {
    return p.M == 1 ? segment.len : segment.len - (p.M - 1 - row_of(col) % p.M);
  };

  bool begins_run = true;
  while (true) {
    {
      Cursor cur = cursor;
      if (cur.left <= 0 || cur.b >= p.B) break;
      Segment sg;
      sg.b = cur.b;
      sg.len = cur.len;
      sg.n_tiles = tiles_of(p, cur.len);
      const int steps = sg.n_tiles + kOpen, unit = cur.off / steps;   // of the sequence: table head, column group
      const int from = cur.off - unit * steps, n = min(steps - from, cur.left);
      sg.at = cur.at - from;
      sg.c_begin = max(from - kOpen, 0);
      sg.c_end = max(from + n - kOpen, 0);
      sg.h = p.CG == 1 ? unit : unit / p.CG;
      sg.cg = unit - sg.h * p.CG;
      cur.left -= n;
      cur.off += n;
      cur.at += n;
      if (cur.off == steps * p.HC) {
        cur.off = 0;
        ++cur.b;
        cur.len = cur.left > 0 && cur.b < p.B ? seq_len(p, cur.b) : 0;
      }
      __syncwarp();
      if (lane == 0) {
        segment = sg;
        cursor = cur;
      }
      __syncwarp();
      if (sg.c_begin == sg.c_end) continue;                       // the run ends before the unit's first tile
      // (an empty pool has no group that could stand in for the missing ones: its tiles are left out)
      n_mine = p.pool.num_pages > 0 ? sg.c_end - sg.c_begin : 0;
    }
    next_id = load_id(0);

    // ------------------------------------------------------------- queries
    // Lane 4 g + t: channels 32 b + 8 t .. of column 8 nt + g, as halves after a power of two that puts the row's largest
    // in [1, 2).  A differential column has one half of the channels, the other is 0.
    float sc[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int j = segment.cg * COLS + nt * 8 + g, row = row_of(nt * 8 + g);
      const int gi = p.M == 1 ? row : row / p.M, m = row - gi * p.M;
      const int64_t at = segment.b * p.q_sb + (segment.h * p.G + gi) * p.q_sh + m * p.q_sm + t * 8;
      constexpr int WORDS = SPLIT ? 8 : 4;
      unsigned raw[NB][WORDS];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int e = 0; e < WORDS; ++e) raw[b][e] = 0;
        if (j >= p.NC || (p.diff && (2 * b >= NB) != (j & 1))) continue;
        const int64_t el = at + 32 * b;
        if (p.q_vec) {
#pragma unroll
          for (int e = 0; e < WORDS; e += 4) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(static_cast<const char*>(p.q) + el * (SPLIT ? 4 : 2) + e * 4));
            raw[b][e] = w.x; raw[b][e + 1] = w.y; raw[b][e + 2] = w.z; raw[b][e + 3] = w.w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < WORDS; ++e) {
            if (SPLIT) raw[b][e] = __float_as_uint(static_cast<const float*>(p.q)[el + e]);
            else raw[b][e] = static_cast<const uint16_t*>(p.q)[el + 2 * e] |
                             static_cast<unsigned>(static_cast<const uint16_t*>(p.q)[el + 2 * e + 1]) << 16;
          }
        }
      }
      // two neighbouring values
      auto pair = [&](int b, int e) {
        if constexpr (SPLIT) return make_float2(__uint_as_float(raw[b][2 * e]), __uint_as_float(raw[b][2 * e + 1]));
        else return p.q_dtype == IAK_DT_F16 ? __half22float2(*reinterpret_cast<const __half2*>(&raw[b][e]))
                                            : make_float2(__uint_as_float(raw[b][e] << 16), __uint_as_float(raw[b][e] & 0xffff0000u));
      };
      float amax = 0.f;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 v = pair(b, e);
          amax = fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y)));
        }
      }
      amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
      // exponent of amax, held to normal numbers on both sides
      const int ex = min(max(static_cast<int>(__float_as_uint(amax) >> 23), 2), 252);
      const float down = __uint_as_float((254 - ex) << 23) * p.sign;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        unsigned hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 v = pair(b, e);
          const float y0 = v.x * down, y1 = v.y * down;
          hi[e] = pack_half2(y0, y1);
          if (SPLIT) {
            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi[e]));
            lo[e] = pack_half2(y0 - back.x, y1 - back.y);
          }
        }
        uint4* dst = reinterpret_cast<uint4*>(q_frag) + (nt * NB + b) * 32 + lane;
        *dst = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (SPLIT) dst[NT * NB * 32] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      // of the lane's own columns 8 nt + 2 t and the next
      const float mine = fminf(fmaxf(p.scale * __uint_as_float(ex << 23), kScaleMin), kScaleMax);
      sc[nt][0] = __shfl_sync(~0u, mine, 8 * t);
      sc[nt][1] = __shfl_sync(~0u, mine, 8 * t + 4);
    }
    {
      int to = stage;
#pragma unroll 1
      for (int i = 0; i < L::kStages - 1; ++i) {
        issue(i, to);
        to = to + 1 == L::kStages ? 0 : to + 1;
      }
    }

    float o[NT][MT][4];
    float m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m_run[nt][0] = m_run[nt][1] = -FLT_MAX;
      l_run[nt][0] = l_run[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
    }
    const int full_end = segment.len - (p.M - 1);         // every query sees the tokens before it
    int key0 = segment.c_begin * kTileKeys;
    for (int k = 0; k < n_mine; ++k, key0 += kTileKeys) {
      // the stage read in the last round is free: every lane is past its reads
      warp_sync();
      issue(k + L::kStages - 1, stage == 0 ? L::kStages - 1 : stage - 1);
      copy_wait<L::kStages - 1>();
      warp_sync();
      const unsigned at = ring + stage * L::kStage;
      stage = stage + 1 == L::kStages ? 0 : stage + 1;
      const unsigned ok_here = (history >> (2 * (L::kStages - 1))) & 3;
      const bool full = ok_here == 3 && key0 + kTileKeys <= full_end;

      // ---------------------------------------------------------- S' = K Q'
      float s[2][NT][4];
      {
        unsigned kw[2][2][NB];
        float ks[2][2 * NB];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          read_words(at + u * Gr::kBytes, kw[u][0]);
          read_words(at + u * Gr::kBytes + Gr::kSet, kw[u][1]);
          unsigned ksw[NB / 2];
          lds_words<NB / 2>(at + u * Gr::kBytes + Gr::kKs + g * 2 * NB, ksw);
#pragma unroll
          for (int i = 0; i < NB / 2; ++i) scales4(ksw[i], &ks[u][4 * i]);
        }
#pragma unroll
        for (int bk = 0; bk < NB; ++bk) {
          uint4 q_hi[NT], q_lo[NT];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            q_hi[nt] = reinterpret_cast<const uint4*>(q_frag)[(nt * NB + bk) * 32 + lane];
            if (SPLIT) q_lo[nt] = reinterpret_cast<const uint4*>(q_frag)[(NT * NB + nt * NB + bk) * 32 + lane];
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            unsigned r0[4], r1[4];
            fp4_unpack4(kw[u][0][bk], r0);
            fp4_unpack4(kw[u][1][bk], r1);
            const float s0 = ks[u][bk], s1 = ks[u][NB + bk];   // of rows g and g + 8
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float acc[4];
              mma16816_new(acc, r0[0], r1[0], r0[1], r1[1], q_hi[nt].x, q_hi[nt].y);
              mma16816(acc, r0[2], r1[2], r0[3], r1[3], q_hi[nt].z, q_hi[nt].w);
              if (SPLIT) {
                mma16816(acc, r0[0], r1[0], r0[1], r1[1], q_lo[nt].x, q_lo[nt].y);
                mma16816(acc, r0[2], r1[2], r0[3], r1[3], q_lo[nt].z, q_lo[nt].w);
              }
              if (bk == 0) {
                s[u][nt][0] = acc[0] * s0; s[u][nt][1] = acc[1] * s0;
                s[u][nt][2] = acc[2] * s1; s[u][nt][3] = acc[3] * s1;
              } else {
                s[u][nt][0] = fmaf(acc[0], s0, s[u][nt][0]); s[u][nt][1] = fmaf(acc[1], s0, s[u][nt][1]);
                s[u][nt][2] = fmaf(acc[2], s1, s[u][nt][2]); s[u][nt][3] = fmaf(acc[3], s1, s[u][nt][3]);
              }
            }
          }
        }
      }
      if (!full) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bool ok = (ok_here >> u) & 1;
          const int key = key0 + u * 16 + g;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool seen = ok && key + (i >> 1) * 8 < limit(nt * 8 + 2 * t + (i & 1));
              if (!seen) s[u][nt][i] = -INFINITY;
            }
          }
        }
      }

      // ---------------------------------------------------------- softmax
      float mx[NT][2];
      bool raise = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[nt][e] = fmaxf(s[0][nt][e], s[0][nt][e + 2]);
          mx[nt][e] = fmaxf(mx[nt][e], fmaxf(s[1][nt][e], s[1][nt][e + 2]));
        }
        float top[2];
        exponents(mx[nt], m_run[nt], sc[nt], top);
        raise = raise || top[0] > kLazy || top[1] > kLazy;
      }
      if (__any_sync(~0u, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float v = mx[nt][e];
            v = fmaxf(v, __shfl_xor_sync(~0u, v, 4));
            v = fmaxf(v, __shfl_xor_sync(~0u, v, 8));
            v = fmaxf(v, __shfl_xor_sync(~0u, v, 16));
            const float m_new = fmaxf(m_run[nt][e], v);
            f[e] = tc::ex2((m_run[nt][e] - m_new) * sc[nt][e]);
            m_run[nt][e] = m_new;
            l_run[nt][e] *= f[e];
          }
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            o[nt][i][0] *= f[0]; o[nt][i][1] *= f[1];
            o[nt][i][2] *= f[0]; o[nt][i][3] *= f[1];
          }
        }
      }
      unsigned pf[2][NT][2], pl[2][NT][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            exponents(&s[u][nt][i], m_run[nt], sc[nt], &x[i]);
            x[i] = tc::ex2(x[i]);
            x[i + 1] = tc::ex2(x[i + 1]);
            add_pair(l_run[nt], &x[i]);
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const unsigned hi = pack_half2(x[2 * r], x[2 * r + 1]);
            pf[u][nt][r] = transpose8x8(hi);
            if (SPLIT) {
              const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi));
              pl[u][nt][r] = transpose8x8(pack_half2(x[2 * r] - back.x, x[2 * r + 1] - back.y));
            }
          }
        }
      }

      // ---------------------------------------------------------- O' += V' P'
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        unsigned vw[2][NB];
        read_words(at + u * Gr::kBytes + Gr::kV, vw[0]);
        read_words(at + u * Gr::kBytes + Gr::kV + Gr::kSet, vw[1]);
        // keys 2t, 2t + 1, 2t + 8, 2t + 9 of the lane's channels' block
        unsigned vs = lds32(at + u * Gr::kBytes + Gr::kVs + (g * NB / 8) * 16 + t * 4);
        if (!full) {          // rows behind the sequence or without a page hold anything: scale 0 keeps NaN away
          const int key = key0 + u * 16 + 2 * t;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!((ok_here >> u) & 1) || key + (i & 1) + 8 * (i >> 1) >= full_end + p.M - 1) vs = (vs & ~(255u << (8 * i))) | (112u << (8 * i));
          }
        }
        const unsigned tops = fp4_half_tops(vs), v01 = fp4_scale_pair<0, 1>(tops), v23 = fp4_scale_pair<2, 3>(tops);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          unsigned r0[4], r1[4];
          fp4_unpack4(vw[0][j], r0);
          fp4_unpack4(vw[1][j], r1);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            r0[i] = mul_half2(r0[i], v01);
            r1[i] = mul_half2(r1[i], v23);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816(o[nt][2 * j], r0[0], r0[1], r1[0], r1[1], pf[u][nt][0], pf[u][nt][1]);
            mma16816(o[nt][2 * j + 1], r0[2], r0[3], r1[2], r1[3], pf[u][nt][0], pf[u][nt][1]);
            if (SPLIT) {
              mma16816(o[nt][2 * j], r0[0], r0[1], r1[0], r1[1], pl[u][nt][0], pl[u][nt][1]);
              mma16816(o[nt][2 * j + 1], r0[2], r0[3], r1[2], r1[3], pl[u][nt][0], pl[u][nt][1]);
            }
          }
        }
      }
    }

    // ------------------------------------------------------------- the segment's end
    float l_all[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = l_run[nt][e];
        v += __shfl_xor_sync(~0u, v, 4);
        v += __shfl_xor_sync(~0u, v, 8);
        v += __shfl_xor_sync(~0u, v, 16);
        l_all[nt][e] = v;
      }
    }
    const int which = begins_run ? 0 : 1;
    const bool whole = segment.c_begin == 0 && segment.c_end == segment.n_tiles;
    if (!p.direct && lane == 0) {
      const int begin = segment.at + kOpen, end = begin + segment.n_tiles - 1;   // the steps of the first and last tile
      Cut d = {segment.b, segment.h, segment.cg * COLS, run, which, -1};
      if (p.by_unit) {
        if (!whole) d.last = run_of(runs, end);
        if (segment.c_begin == 0) cuts(p)[segment.b * p.HC + segment.h * p.CG + segment.cg] = d;
      } else if (begins_run) {
        d.first = run - 1;
        if (segment.c_begin > 0 && run_begin(runs, run - 1) <= begin) {
          d.which = run_begin(runs, run - 1) >= segment.at ? 0 : 1;
          d.last = run_of(runs, end);
        }
        cuts(p)[run] = d;
      }
    }
    // a lane has channels 4 NB g .. of columns 8 nt + 2 t and the next: with differential attention, of a row's two maps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = nt * 8 + 2 * t, j = segment.cg * COLS + col;
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (j + e >= p.NC) continue;
          float* part = part_at(p, run, which, col + e);
#pragma unroll
          for (int i = 0; i < MT; i += 2)
            *reinterpret_cast<float4*>(part + g * (4 * NB) + 2 * i) =
                make_float4(o[nt][i][e], o[nt][i][e + 2], o[nt][i + 1][e], o[nt][i + 1][e + 2]);
          if (g == 0) *reinterpret_cast<float4*>(part + D) = make_float4(m_run[nt][e], l_all[nt][e], sc[nt][e], 0.f);
        }
        continue;
      }
      if (p.diff) {
        const int row = j >> 1, gi = row / p.M;
        const bool real = j < p.NC;
        const float w0 = safe_inverse(l_all[nt][0]), w1 = safe_inverse(l_all[nt][1]);
        const float lam = real ? p.lam[segment.h * p.G + gi] : 0.f;
        float x[4 * NB], mul = p.out_scale;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          x[2 * i] = difference(__fmul_rn(o[nt][i][0], w0), lam, __fmul_rn(o[nt][i][1], w1));
          x[2 * i + 1] = difference(__fmul_rn(o[nt][i][2], w0), lam, __fmul_rn(o[nt][i][3], w1));
        }
        if (p.norm_w) {
          float sq = 0.f;
#pragma unroll
          for (int i = 0; i < 4 * NB; ++i) sq = fmaf(x[i], x[i], sq);
          sq += __shfl_xor_sync(~0u, sq, 4);
          sq += __shfl_xor_sync(~0u, sq, 8);
          sq += __shfl_xor_sync(~0u, sq, 16);
          mul *= norm_factor<NB>(p, sq);
        }
#pragma unroll
        for (int i = 0; i < 4 * NB; ++i) x[i] *= p.norm_w ? mul * p.norm_w[g * (4 * NB) + i] : mul;
        if (real)
          store_run(p, segment.b * p.o_sb + (segment.h * p.G + gi) * p.o_sh + (row - gi * p.M) * p.o_sm + g * (4 * NB), x);
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (j + e >= p.NC) continue;
          const int row = j + e, gi = p.M == 1 ? row : row / p.M;
          const float w = safe_inverse(l_all[nt][e]);
          float x[4 * NB];
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            x[2 * i] = o[nt][i][e] * w;
            x[2 * i + 1] = o[nt][i][e + 2] * w;
          }
          store_run(p, segment.b * p.o_sb + (segment.h * p.G + gi) * p.o_sh + (row - gi * p.M) * p.o_sm + g * (4 * NB), x);
        }
      }
    }
    begins_run = false;
    __syncwarp();                                 // before the next segment's record and queries
  }
}

// ---------------------------------------------------------------- join kernel
// For every (record of a cut, output row) the unit's parts are added in order of the runs that left them, by a team of
// warps: a block each, but for TEAM 1, where a block has 16.
__host__ __device__ constexpr int join_warps(int team) { return team == 1 ? 16 : team; }

__host__ __device__ inline int join_rows(const DecP& p) { return p.cols / (p.diff ? 2 : 1); }

template <int NB, int TEAM>
__global__ void __launch_bounds__(join_warps(TEAM) * 32) fp4_join_kernel(const DecP p, int records) {
  constexpr int D = NB * 32;
  __shared__ float part_sum[TEAM][D + 2];
  const int per = p.diff ? 2 : 1, rows = join_rows(p);
  const int lane = threadIdx.x & 31, warp = TEAM == 1 ? 0 : threadIdx.x >> 5;
  const int item = TEAM == 1 ? blockIdx.x * join_warps(1) + (threadIdx.x >> 5) : blockIdx.x;
  const int record = item / rows + (p.by_unit ? 0 : 1), r = item % rows;
  // every warp waits, so that this kernel never ends before the main one
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (item / rows >= records) return;
  const Cut d = cuts(p)[record];
  const int n = d.last - d.first + 1, j0 = d.j0 + r * per;
  if (d.last < 0 || j0 >= p.NC) return;
  float x[NB];
  for (int half = 0; half < per; ++half) {
    const int col = r * per + half;
    // a warp takes every TEAM-th part, four at a time, so that their loads run together
    float top = -FLT_MAX, l = 0.f, sc = 0.f, acc[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) acc[i] = 0.f;
    constexpr int kAt = NB <= 4 ? 4 : 2;
    for (int c = warp; c < n; c += kAt * TEAM) {
      float m[kAt], pl[kAt], v[kAt][NB];
#pragma unroll
      for (int k = 0; k < kAt; ++k) {
        const int part = min(c + k * TEAM, n - 1);
        const float* at = part_at(p, d.first + part, part == 0 ? d.which : 0, col);
        const float4 ends = *reinterpret_cast<const float4*>(at + D);
        m[k] = ends.x;
        pl[k] = ends.y;
        sc = ends.z;                               // the same in every part
#pragma unroll
        for (int i = 0; i < NB; ++i) v[k][i] = at[i * 32 + lane];
      }
      float next = top;
#pragma unroll
      for (int k = 0; k < kAt; ++k) next = fmaxf(next, m[k]);
      const float old = tc::ex2((top - next) * sc);
      l *= old;
#pragma unroll
      for (int i = 0; i < NB; ++i) acc[i] *= old;
#pragma unroll
      for (int k = 0; k < kAt; ++k) {
        if (c + k * TEAM < n) {                    // (the last part stands in for missing ones)
          const float f = tc::ex2((m[k] - next) * sc);
          l = fmaf(pl[k], f, l);
#pragma unroll
          for (int i = 0; i < NB; ++i) acc[i] = fmaf(v[k][i], f, acc[i]);
        }
      }
      top = next;
    }
    if constexpr (TEAM > 1) {
#pragma unroll
      for (int i = 0; i < NB; ++i) part_sum[warp][i * 32 + lane] = acc[i];
      if (lane == 0) { part_sum[warp][D] = top; part_sum[warp][D + 1] = l; }
      __syncthreads();
      if (warp == 0) {
        top = -FLT_MAX;
        l = 0.f;
#pragma unroll
        for (int w = 0; w < TEAM; ++w) top = fmaxf(top, part_sum[w][D]);
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i] = 0.f;
#pragma unroll
        for (int w = 0; w < TEAM; ++w) {
          const float f = tc::ex2((part_sum[w][D] - top) * sc);
          l = fmaf(part_sum[w][D + 1], f, l);
#pragma unroll
          for (int i = 0; i < NB; ++i) acc[i] = fmaf(part_sum[w][i * 32 + lane], f, acc[i]);
        }
      }
    }
    if (warp == 0) {
      const int row = p.diff ? (j0 >> 1) : j0;
      const float inv = safe_inverse(l);
      const float lam = half ? p.lam[d.h * p.G + row / p.M] : 0.f;
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const float part = __fmul_rn(acc[i], inv);
        x[i] = half ? difference(x[i], lam, part) : part;
      }
      if (half == per - 1) finish_row<NB>(p, d.b, d.h * p.G + row / p.M, row % p.M, x);
    }
    if (TEAM > 1) __syncthreads();
  }
}

// -------------------------------------------------------------------- launch
struct Plan { int grid; size_t ws; };

template <int NB, int NT, bool SPLIT>
int resident_blocks(int* blocks) {
  static std::mutex mu;
  static int cache[64] = {0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return check_cuda(e, "cudaGetDevice");
  std::lock_guard<std::mutex> lock(mu);
  if (dev < 0 || dev >= 64 || cache[dev] == 0) {
    auto kern = fp4_decode_kernel<NB, NT, SPLIT>;
    const int smem = Shape<NB, NT, SPLIT>::kSmem;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return check_cuda(e, "fp4_decode shared memory");
    int per_sm = 0;
    e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, Shape<NB, NT, SPLIT>::kThreads, smem);
    if (e != cudaSuccess) return check_cuda(e, "fp4_decode occupancy");
    if (per_sm < 1) return fail(IAK_ERR_UNSUPPORTED, "fp4_decode does not fit on an SM");
    if (dev < 0 || dev >= 64) { *blocks = per_sm * device_sm_count(); return IAK_OK; }
    cache[dev] = per_sm * device_sm_count();
  }
  *blocks = cache[dev];
  return IAK_OK;
}

template <int NB, int NT, bool SPLIT>
int make_plan(DecP& p, Plan* plan) {
  using L = Shape<NB, NT, SPLIT>;
  p.CG = (p.NC + L::COLS - 1) / L::COLS;
  p.cols = std::min(p.NC, L::COLS);
  const int64_t hc = static_cast<int64_t>(p.Ht) * p.CG, units = hc * p.B;
  if (units * L::COLS > 0x7fffffffLL) return fail(IAK_ERR_UNSUPPORTED, "iak_fp4_decode: too many rows for one launch");
  p.HC = static_cast<int>(hc);
  p.min_steps = L::kMinSteps;
  const int64_t most = (static_cast<int64_t>(p.W) * p.pool.PS + kTileKeys - 1) / kTileKeys;
  if ((most + kOpen) * units > 0x7fffffffLL - 64)
    return fail(IAK_ERR_UNSUPPORTED, "iak_fp4_decode: tables of more than 2^31 tiles of %d tokens", kTileKeys);
  // units that a warp covers about as fast as two would with their parts joined
  p.direct = most <= kDirectTiles;
  int blocks = 0;
  if (int st = resident_blocks<NB, NT, SPLIT>(&blocks)) return st;
  if (p.direct) {
    plan->grid = static_cast<int>((units + L::kWarps - 1) / L::kWarps);
    p.runs = plan->grid * L::kWarps;
    p.by_unit = 1;
    plan->ws = 0;
    return IAK_OK;
  }
  const int64_t useful = (most * units + L::kMinSteps - 1) / L::kMinSteps;
  plan->grid = static_cast<int>(std::min<int64_t>(blocks, (useful + L::kWarps - 1) / L::kWarps));
  p.runs = plan->grid * L::kWarps;
  p.by_unit = units <= p.runs;
  plan->ws = static_cast<size_t>(p.runs) * (2 * p.cols * (L::D + 4) * sizeof(float) + sizeof(Cut));
  return IAK_OK;
}

template <int NB, int TEAM>
int launch_join(const DecP& p, int records, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  const int64_t items = static_cast<int64_t>(records) * join_rows(p);
  cfg.gridDim = dim3(static_cast<unsigned>(TEAM == 1 ? (items + join_warps(1) - 1) / join_warps(1) : items));
  cfg.blockDim = dim3(join_warps(TEAM) * 32);
  cfg.stream = s;
  // starts while the main kernel's last blocks run; it waits for them before it reads a part
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, fp4_join_kernel<NB, TEAM>, p, records), "fp4_join launch");
}

template <int NB, int NT, bool SPLIT>
int run_shape(DecP& p, bool launch, void* ws, size_t ws_bytes, size_t* need, cudaStream_t s) {
  using L = Shape<NB, NT, SPLIT>;
  Plan plan;
  if (int st = make_plan<NB, NT, SPLIT>(p, &plan)) return st;
  if (need) *need = plan.ws;
  if (!launch) return IAK_OK;
  if (plan.ws > ws_bytes || (plan.ws && !ws))
    return fail(IAK_ERR_WORKSPACE, "iak_fp4_decode needs %zu workspace bytes, got %zu", plan.ws, ws_bytes);
  if (reinterpret_cast<uintptr_t>(ws) % 16) return fail(IAK_ERR_INVALID_ARG, "iak_fp4_decode: workspace not 16-byte aligned");
  p.ws = static_cast<float*>(ws);
  fp4_decode_kernel<NB, NT, SPLIT><<<plan.grid, L::kThreads, L::kSmem, s>>>(p);
  if (int st = check_cuda(cudaGetLastError(), "fp4_decode launch")) return st;
  if (p.direct) return IAK_OK;
  const int units = p.B * p.HC;
  const int records = p.by_unit ? units : p.runs - 1;
  // warps per row: as many as share the parts well, while all rows' teams run at once
  // (8 sequences of 32k, 27 parts a unit, 256 rows: 56 us in all with 16, 63 with 1; 16 of D 64, 18 parts, 2048 rows:
  // 103 with 16, 92 with 1)
  const int parts = p.runs / units;
  const int64_t rows = static_cast<int64_t>(records) * join_rows(p);
  if (parts >= 12 && rows <= 512) return launch_join<NB, 16>(p, records, s);
  return parts >= 4 && rows <= 4096 ? launch_join<NB, 4>(p, records, s) : launch_join<NB, 1>(p, records, s);
}

// Columns per block: as many n = 8 tiles as the columns need, up to what the accumulators leave registers for; more
// columns read the cache again.
template <int NB, bool SPLIT>
int run_cols(DecP& p, bool launch, void* ws, size_t ws_bytes, size_t* need, cudaStream_t s) {
  if constexpr (NB < 8 && !SPLIT) {
    if (p.NC > 16) return run_shape<NB, 4, SPLIT>(p, launch, ws, ws_bytes, need, s);
  }
  if constexpr (NB < 8 || !SPLIT) {
    if (p.NC > 8) return run_shape<NB, 2, SPLIT>(p, launch, ws, ws_bytes, need, s);
  }
  return run_shape<NB, 1, SPLIT>(p, launch, ws, ws_bytes, need, s);
}

template <int NB>
int run_types(DecP& p, bool launch, void* ws, size_t ws_bytes, size_t* need, cudaStream_t s) {
  // fp32 queries: q and P as the sum of two halves
  if (p.q_dtype == IAK_DT_F32) return run_cols<NB, true>(p, launch, ws, ws_bytes, need, s);
  return run_cols<NB, false>(p, launch, ws, ws_bytes, need, s);
}

int decode_call(const iak_fp4_pool* pool, const iak_fp4_decode_args* a, bool launch, void* ws, size_t ws_bytes,
                size_t* need, void* stream) {
  const char* what = "iak_fp4_decode";
  if (need) *need = 0;
  if (!pool || !a) return fail(IAK_ERR_INVALID_ARG, "%s: null arguments", what);
  if (int st = check_fp4_pool(pool, what)) return st;
  if (a->batch < 0 || a->num_q_heads < 0 || a->num_table_heads < 0 || a->num_queries < 0 || a->table_width < 0)
    return fail(IAK_ERR_INVALID_ARG, "%s: negative size", what);
  if (a->q_dtype < IAK_DT_F32 || a->q_dtype > IAK_DT_BF16 || a->out_dtype < IAK_DT_F32 || a->out_dtype > IAK_DT_BF16)
    return fail(IAK_ERR_INVALID_ARG, "%s: bad dtype", what);
  if (a->num_queries > IAK_FP4_MAX_QUERIES)
    return fail(IAK_ERR_UNSUPPORTED, "%s: %d queries, at most %d", what, a->num_queries, IAK_FP4_MAX_QUERIES);
  if (a->differential && !(a->eps >= 0.f && a->eps - a->eps == 0.f && a->out_scale - a->out_scale == 0.f))
    return fail(IAK_ERR_INVALID_ARG, "%s: eps must be finite and not negative, out_scale finite", what);
  if (a->batch == 0 || a->num_q_heads == 0 || a->num_queries == 0) return IAK_OK;
  if (a->num_table_heads == 0 || a->num_q_heads % a->num_table_heads)
    return fail(IAK_ERR_INVALID_ARG, "%s: query heads (%d) must be a multiple of table heads (%d)", what,
                a->num_q_heads, a->num_table_heads);
  if (!(a->sm_scale - a->sm_scale == 0.f)) return fail(IAK_ERR_INVALID_ARG, "%s: sm_scale is not finite", what);
  if (launch) {
    if (!a->q || !a->out || !a->lengths || (a->table_width > 0 && !a->page_table))
      return fail(IAK_ERR_INVALID_ARG, "%s: null q, out, lengths or page_table", what);
    if (a->differential && !a->lam) return fail(IAK_ERR_INVALID_ARG, "%s: differential attention needs lam", what);
  }
  DecP p = {};
  p.pool = {static_cast<uint8_t*>(pool->data), pool->num_pages, pool->page_size, pool->head_dim};
  p.gpp = pool->page_size / 16;
  p.gpp_inv = ((1ull << 36) + p.gpp - 1) / p.gpp;
  if (pool->num_pages * p.gpp > 0x7fffffffLL) return fail(IAK_ERR_UNSUPPORTED, "%s: more than 2^31 groups of rows", what);
  p.q = a->q; p.q_dtype = a->q_dtype; p.q_sb = a->q_stride_b; p.q_sh = a->q_stride_h; p.q_sm = a->q_stride_m;
  p.out = a->out; p.out_dtype = a->out_dtype;
  p.o_sb = a->out_stride_b; p.o_sh = a->out_stride_h; p.o_sm = a->out_stride_m;
  p.B = a->batch; p.Ht = a->num_table_heads; p.G = a->num_q_heads / p.Ht; p.M = a->num_queries;
  p.pt = a->page_table; p.pt_sb = a->pt_stride_b; p.pt_sh = a->pt_stride_h;
  p.W = pool->num_pages > 0 ? a->table_width : 0;      // an empty pool holds no token
  p.lengths = a->lengths;
  p.scale = (a->sm_scale < 0.f ? -a->sm_scale : a->sm_scale) * 1.44269504088896340736f;
  p.sign = a->sm_scale < 0.f ? -1.f : 1.f;
  p.diff = a->differential ? 1 : 0;
  p.lam = a->lam; p.norm_w = a->norm_weight; p.eps = a->eps; p.out_scale = a->out_scale;
  const int64_t nc = static_cast<int64_t>(p.G) * p.M * (1 + p.diff);
  if (nc > (1 << 20)) return fail(IAK_ERR_UNSUPPORTED, "%s: too many query heads", what);
  p.NC = static_cast<int>(nc);
  auto aligned = [](const void* base, int dtype, int64_t a, int64_t b, int64_t c) {
    const int64_t per16 = dtype == IAK_DT_F32 ? 4 : 8;
    return reinterpret_cast<uintptr_t>(base) % 16 == 0 && a % per16 == 0 && b % per16 == 0 && c % per16 == 0 ? 1 : 0;
  };
  p.q_vec = aligned(p.q, p.q_dtype, p.q_sb, p.q_sh, p.q_sm);
  p.o_vec = aligned(p.out, p.out_dtype, p.o_sb, p.o_sh, p.o_sm);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (static_cast<int64_t>(p.W) * p.pool.PS > kMaxTokens)
    return fail(IAK_ERR_UNSUPPORTED, "%s: tables of more than %d tokens", what, kMaxTokens);
  if (pool->head_dim == 64) return run_types<2>(p, launch, ws, ws_bytes, need, s);
  if (pool->head_dim == 128) return run_types<4>(p, launch, ws, ws_bytes, need, s);
  return run_types<8>(p, launch, ws, ws_bytes, need, s);
}

}  // namespace

}  // namespace iak

extern "C" int iak_fp4_decode_workspace_size(const iak_fp4_pool* pool, const iak_fp4_decode_args* args, size_t* bytes) {
  if (!bytes) return iak::fail(IAK_ERR_INVALID_ARG, "iak_fp4_decode: null arguments");
  return iak::decode_call(pool, args, false, nullptr, 0, bytes, nullptr);
}

extern "C" int iak_fp4_decode(const iak_fp4_pool* pool, const iak_fp4_decode_args* args, void* workspace,
                              size_t workspace_bytes, void* stream) {
  return iak::decode_call(pool, args, true, workspace, workspace_bytes, nullptr, stream);
}
