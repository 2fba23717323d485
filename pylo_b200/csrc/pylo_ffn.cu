// The gated feed-forward block on the tensor cores, forward and backward.
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T
//   dh = dy Wd;  dg = dh P with P = u act'(g), du = dh Q with Q = act(g)
//   dx = dg Wg + du Wu;  dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// Four launches of one product kernel, C = sum_k A(m, k) B(n, k) over 16-bit operands with fp32 sums, whose epilogues differ:
//   gate    both projections of a tile of h at once: half of a tile's columns are rows of Wg, the other half the same rows of Wu, so g and u
//           meet in one thread's registers, which makes h, P and Q of them; g and u themselves reach no memory
//   plain   y = h Wd^T
//   back    dh = dy Wd, which reaches no memory either: dg and du of P and Q
//   plain   dx (a contraction of two parts), dWg, dWu, dWd side by side in one launch
// No operand is transposed: 16-bit operands may be read with the contraction index as rows ("MN-major"), as dx and the weights' gradients
// need them.
//
// What is kept for the backward pass: h in 16 bits, which the forward pass needs in memory anyway, P and Q with 24 (16 significant bits, an fp32
// value's upper three bytes, rounded): 8 bytes per element of h, what g, u, act(g) and h take in 16 bits.
// With P and Q in 16 bits, dg and du would be rounded twice on their way into dx, dWg and dWu: an error of 1.7 instead of 1.4 times that of the
// result's own rounding.
//
// A CTA has ten or eighteen warps: one lane issues the copies (TMA, 128-byte swizzle), one the products, the others run the epilogue.  Every wait is bounded;
// one that runs out ends the CTA's work in order and sets a bit of the caller's status word.
#include <cuda.h>
#include <cuda_bf16.h>
#include <math_constants.h>

#include "pylo_common.cuh"
#include "pylo_launch.cuh"

#define FF_BM 128               // rows of a CTA's tile
#define FF_BK 64                // terms per stage
#define FF_BOX 8192             // bytes of a box: 64 x 64 elements
#define FF_SPIN_LIMIT (1 << 22)
#define FF_SPINS 64             // more for each stage of a whole tile that is waited for: a stage takes less time than so many looks at a barrier
#define FF_GROUP 4              // products of a launch
#define FF_BAND 8               // rows of tiles that are taken together, so that what is in flight shares operands in the L2 cache
enum { FF_PLAIN = 0, FF_GATE = 1, FF_BACK = 2 };
// Warps of the epilogue, and columns that each takes at a time.  8192 rows x 1024 x 4096: gate 101 us with 8 warps and 105 with 16 (one more wait for the
// tile's sums per warp); back, whose warps wait for P and Q, 110 and 94.
__host__ __device__ constexpr int ff_epi_warps(int epi) { return epi == FF_BACK ? 16 : 8; }
__host__ __device__ constexpr int ff_columns(int epi) { return epi == FF_PLAIN ? 32 : 16; }
__host__ __device__ constexpr int ff_threads(int epi) { return (ff_epi_warps(epi) + 2) * 32; }

// ------------------------------------------------------------------------------------------------
// tensor cores and barriers
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t ff_cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t ff_cluster_size() { uint32_t n; asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n)); return n; }
__device__ __forceinline__ void cluster_sync() {   // all threads of the cluster's CTAs; orders accesses to all memory
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of another CTA's copy of a shared variable
__device__ __forceinline__ uint32_t nf_at_rank(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ bool ff_elect() {
  uint32_t pred;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(pred));
  return pred != 0;
}
__device__ __forceinline__ void ff_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ bool ff_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_addr(bar)), "r"(parity) : "memory");
  return ok;
}
// false if the wait ran out, here or in another warp of the CTA; stages: how many are worked on meanwhile (2^24 at most)
__device__ __forceinline__ bool ff_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int stages = 0) {
  for (int it = 0; it < FF_SPIN_LIMIT + FF_SPINS * stages; ++it) {
    if (ff_try(bar, parity)) return true;
    if ((it & 63) == 63 && *abort) return false;
  }
  *abort = 1;
  return false;
}
// The accumulator has been read (and nothing else is passed on with it: a release would wait for the warp's stores).  A pair's: at the first CTA's barrier
template <bool PAIR>
__device__ __forceinline__ void ff_arrive(uint64_t* bar) {
  if constexpr (PAIR) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(nf_at_rank(bar, 0)) : "memory");
  else asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ void ff_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void ff_copy(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  if constexpr (PAIR)   // the barrier may be the other CTA's
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void ff_commit(uint64_t* bar) {
  if constexpr (PAIR)   // arrives at the barriers of both CTAs
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)), "h"((uint16_t)3) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void ff_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// A kernel that is launched while its predecessor runs must not take tensor memory that the latter has yet to ask for, nor let a successor take what it
// has yet to ask for itself: each would wait for the other.  So, other than pdl_begin(): wait, allocate, and only then let the next kernel be set up.
template <bool PAIR>
__device__ __forceinline__ void ff_take_tmem(uint32_t* at, int columns, int warp) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(at)), "r"(columns) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(at)), "r"(columns) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
}
// Descriptor of a 128-byte-swizzled operand of 64 x 64 boxes.  K-major: rows of 64 k, groups of eight rows 1024 bytes apart, boxes one behind
// the other.  MN-major: rows are k and hold 64 mn, groups of eight k 1024 bytes apart, boxes of 64 mn FF_BOX apart.
__device__ __forceinline__ uint64_t ff_desc(uint32_t saddr, int mn) {
  return (uint64_t)((saddr >> 4) & 0x3fff) | ((uint64_t)(mn ? FF_BOX >> 4 : 1) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// fp32 sums of products of two operands of one 16-bit type (bf16 or fp16)
__device__ __forceinline__ uint32_t ff_idesc(uint32_t m, uint32_t n, int a_mn, int b_mn, bool bf16) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ void ff_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ff_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 32 columns of a warp's 32 rows, a row per lane
__device__ __forceinline__ void ff_ld(uint32_t taddr, float (&f)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
#pragma unroll
  for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(r[j]);
}
// 16 of them
__device__ __forceinline__ void ff_ld(uint32_t taddr, float (&f)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr) : "memory");
#pragma unroll
  for (int j = 0; j < 16; ++j) f[j] = __uint_as_float(r[j]);
}

// ------------------------------------------------------------------------------------------------
// 16-bit elements, two in a word
// ------------------------------------------------------------------------------------------------
template <bool BF>
__device__ __forceinline__ uint32_t ff_pack(float a, float b) {
  if constexpr (BF) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
// an fp32 value rounded to its upper three bytes (NaN stays NaN, what rounds beyond the largest becomes infinite)
__device__ __forceinline__ uint32_t ff_round24(float v) {
  const uint32_t b = __float_as_uint(v);
  return v != v ? b | 0x400000u : b + 0x7f + ((b >> 8) & 1);
}

// ------------------------------------------------------------------------------------------------
// the product kernel
// ------------------------------------------------------------------------------------------------
// What is kept: h [rows][ld], and of P and Q the upper 16 bits and the 8 below, in the order in which the epilogues' lanes have them: blocks of 32 rows and 16
// columns (3 KB), row by row of blocks, of which each lane writes and reads its row in pieces of 16 bytes, side by side with its neighbours' (P's upper bits
// 2, Q's 2, P's lower ones, Q's).  Few rows: planes [rows][2 ld], 16 columns of P, the same 16 of Q, the next 16 of P.
#define FF_KEPT_PIECES 6
struct ff_kept {
  uint16_t* h;
  uint4* blocks;
  uint16_t* hi;
  uint8_t* lo;
};
__device__ __forceinline__ long long ff_place(long long row, long long ld, int col) { return row * 2 * ld + (col >> 4) * 32 + (col & 15); }   // of P; Q is 16 behind
__device__ __forceinline__ uint4* ff_block(const ff_kept& kept, int row, long long ld, int col) {   // this lane's first piece
  return kept.blocks + ((row >> 5) * (ld >> 4) + (col >> 4)) * (32 * FF_KEPT_PIECES) + (threadIdx.x & 31);
}
struct ff_product {
  CUtensorMap A[2], B[2];   // the two parts of the contraction; GATE: B is Wg, Wu
  CUtensorMap Cm;           // of C, where mapped
  void* C;                  // PLAIN: [M][ldc]
  long long ldc;
  int M, N, K;              // of each part; GATE, BACK: N = hidden
  int parts;                // of the contraction: 1 or 2
  int a_mn, b_mn;           // the operand's rows are the contraction index
  int mapped;               // C's rows begin on 16-byte boundaries: it is written by copies from shared memory
  int tiles_m, tiles_n, tile0;   // tile0: tiles of the products before this one
};
struct ff_args {
  ff_product p[FF_GROUP];
  CUtensorMap planes[2];    // what the epilogue writes by copies from shared memory, 32 rows of 16 columns at a time: GATE: h; BACK: dg, du (of many rows)
  ff_kept kept;             // GATE: P and Q written, of few rows h too; BACK: read
  uint16_t *dg, *du;        // BACK of few rows: written
  long long ld;             // of kept, dg, du
  int n, tiles, activation, keep;
  int *status, *host_status;
};

template <int EPI>
struct FfSmem {
  static constexpr int STAGES = 6, WARPS = ff_epi_warps(EPI), OUT = EPI == FF_PLAIN ? 4096 : EPI == FF_BACK ? 2048 : 1024;
  // per stage: A (128 x 64), B (128 x 64; of a pair one half of the tile's 256)
  unsigned char st[STAGES][4 * FF_BOX];
  // per epilogue warp: results on their way
  unsigned char out[WARPS][OUT];
  uint64_t full[STAGES], empty[STAGES], ready[2], free[2], sums;
  uint32_t tmem;
  volatile int abort;
};

// A warp's block of 32 rows x 64 bytes (32 x 16 bit) or 32 x 32 bytes (16 x 16 bit) between rows per lane and rows of four (two) lanes: 16-byte
// pieces, spread over the banks.
__device__ __forceinline__ uint4* ff_at64(unsigned char* s, int row, int piece) { return reinterpret_cast<uint4*>(s + row * 64 + 16 * (piece ^ ((row >> 1) & 3))); }
__device__ __forceinline__ uint4* ff_at32(unsigned char* s, int row, int piece) { return reinterpret_cast<uint4*>(s + row * 32 + 16 * (piece ^ ((row >> 2) & 1))); }

__device__ __forceinline__ void ff_put64(unsigned char* s, const uint32_t (&w)[16]);
// 32 x 32 elements of 16 bits from a row per lane to memory where rows begin anywhere (else they leave by copies), a row at a time; rows and columns beyond
// the matrix are left out
__device__ __forceinline__ void ff_store16(unsigned char* s, const uint32_t (&w)[16], uint16_t* dst, long long ld, int rows, int cols) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  ff_put64(s, w);
  __syncwarp();
  if (lane < cols) {
#pragma unroll 8
    for (int r = 0; r < min(32, rows); ++r)
      dst[r * ld + lane] = reinterpret_cast<const uint16_t*>(ff_at64(s, r, lane >> 3))[lane & 7];
  }
}
// A lane's row of 32 elements of 16 bits into such a block
__device__ __forceinline__ void ff_put64(unsigned char* s, const uint32_t (&w)[16]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int q = 0; q < 4; ++q) *ff_at64(s, lane, q) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
}
// of 16
__device__ __forceinline__ void ff_put32(unsigned char* s, const uint32_t (&w)[8]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int q = 0; q < 2; ++q) *ff_at32(s, lane, q) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
}
// 16 values of P (which = 0) or Q to their pieces of a block, and back
__device__ __forceinline__ void ff_put24(uint4* to, int which, const float (&v)[16]) {
  uint32_t h[8], l[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = ff_round24(v[4 * j + i]);
    h[2 * j] = __byte_perm(b[0], b[1], 0x7632);
    h[2 * j + 1] = __byte_perm(b[2], b[3], 0x7632);
    l[j] = __byte_perm(__byte_perm(b[0], b[1], 0x0051), __byte_perm(b[2], b[3], 0x0051), 0x5410);
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) __stcs(to + 32 * (2 * which + q), make_uint4(h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]));
  __stcs(to + 32 * (4 + which), make_uint4(l[0], l[1], l[2], l[3]));
}
__device__ __forceinline__ void ff_take24(const uint4 (&from)[FF_KEPT_PIECES], int which, float (&v)[16]) {
  const uint4 h0 = from[2 * which], h1 = from[2 * which + 1], l0 = from[4 + which];
  const uint32_t h[8] = {h0.x, h0.y, h0.z, h0.w, h1.x, h1.y, h1.z, h1.w}, l[4] = {l0.x, l0.y, l0.z, l0.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {   // an fp32 value's upper half, and the byte below
    v[4 * j] = __uint_as_float((h[2 * j] << 16) | ((l[j] << 8) & 0xff00u));
    v[4 * j + 1] = __uint_as_float((h[2 * j] & 0xffff0000u) | (l[j] & 0xff00u));
    v[4 * j + 2] = __uint_as_float((h[2 * j + 1] << 16) | ((l[j] >> 8) & 0xff00u));
    v[4 * j + 3] = __uint_as_float((h[2 * j + 1] & 0xffff0000u) | ((l[j] >> 16) & 0xff00u));
  }
}
// One of the epilogue's blocks to memory; what of it lies behind the matrix is not written
__device__ __forceinline__ void ff_send(const CUtensorMap* map, const unsigned char* from, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(smem_addr(from)), "r"(x), "r"(y) : "memory");
}

// act(g) and its slope
__device__ __forceinline__ void ff_act(int activation, float g, float& a, float& slope) {
  if (activation == PYLO_ACT_SILU) {
    const float s = __fdividef(1.0f, 1.0f + __expf(-g));
    a = g * s;
    slope = fmaf(a, 1.0f - s, s);
  } else if (activation == PYLO_ACT_GELU) {
    const float phi = 0.5f + 0.5f * erff(g * 0.70710678118654752f);
    a = g * phi;
    slope = fmaf(g * 0.3989422804014327f, __expf(-0.5f * g * g), phi);
  } else if (activation == PYLO_ACT_GELU_TANH) {
    const float k = 0.7978845608028654f, t = tanhf(k * fmaf(0.044715f * g * g, g, g));
    a = 0.5f * g * (1.0f + t);
    const float b = fminf(fmaxf(g, -100.0f), 100.0f);   // beyond, 1 - t^2 is 0, and a square might be infinite
    slope = 0.5f * (1.0f + t) + 0.5f * b * (1.0f - t * t) * k * fmaf(3.0f * 0.044715f * b, b, 1.0f);
  } else {
    a = g > 0.f ? g : g != g ? g : 0.f;
    slope = g > 0.f ? 1.0f : 0.f;
  }
}

// PAIR: two CTAs on two SMs share a tile of 256 x 256 (each has its own 128 rows of A and one half of B's columns, and the tensor cores of both
// read both halves); persistent, with two accumulators, so that one tile's epilogue runs beside the next one's products.
// Otherwise the CTAs of a cluster (1, 2, 4 or 8) share one tile of 128 x 128, each with its part of the contraction; the first adds their sums up
// through distributed shared memory, in rank order.
//
// 8192 rows x 4096 x 14336 bf16 on a B200, passes in loops of their own: forward 2051 us (1.41 PFLOP/s), backward 4356 (1.33); one behind the other 6.6 to 7.0 ms, all at the
// power limit.  8192 x 1024 x 4096: 173, 335 and 547 to 581.
template <bool PAIR, int EPI, bool BF>
__global__ void __launch_bounds__(ff_threads(EPI), 1) k_ffn_product(const __grid_constant__ ff_args a) {
  extern __shared__ unsigned char ff_dyn[];
  using Smem = FfSmem<EPI>;
  constexpr int STAGES = Smem::STAGES, WARPS = Smem::WARPS, COLS = ff_columns(EPI);
  constexpr int BN = PAIR ? 256 : 128, TILE_M = PAIR ? 256 : 128, OUT_N = EPI == FF_GATE ? BN / 2 : BN;
  constexpr uint32_t STAGE = 4 * FF_BOX;
  Smem& sm = *reinterpret_cast<Smem*>(ff_dyn + ((1024 - (smem_addr(ff_dyn) & 1023)) & 1023));   // at the same place in all CTAs of a cluster
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int rank = (int)ff_cluster_rank(), ctas = (int)ff_cluster_size();
  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) { ff_init(&sm.full[s], 1); ff_init(&sm.empty[s], 1); }
    for (int s = 0; s < 2; ++s) { ff_init(&sm.ready[s], 1); ff_init(&sm.free[s], (PAIR ? 2 : 1) * WARPS); }
    ff_init(&sm.sums, ctas > 1 ? (ctas - 1) * WARPS : 1);
    sm.abort = 0;
  }
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  ff_take_tmem<PAIR>(&sm.tmem, 512, warp);
  ff_fence_before();
  __syncthreads();
  cluster_sync();   // the other CTAs' barriers exist
  ff_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
  const int step = (int)gridDim.x / ctas, first = (int)blockIdx.x / ctas;
  // the product a tile belongs to and its place there: bands of FF_BAND rows of tiles, column by column
  auto locate = [&](int tile, int& tm, int& tn) -> const ff_product& {
    int k = 0;
    while (k + 1 < a.n && tile >= a.p[k + 1].tile0) ++k;
    const ff_product& p = a.p[k];
    const int r = tile - p.tile0, band = r / (FF_BAND * p.tiles_n), at = r - band * FF_BAND * p.tiles_n, high = min(FF_BAND, p.tiles_m - band * FF_BAND);
    tn = at / high;
    tm = band * FF_BAND + at - tn * high;
    return p;
  };
  // this CTA's share of the contraction, in stages
  auto share = [&](const ff_product& p, int& kb0, int& kb1) {
    const int per_part = (p.K + FF_BK - 1) / FF_BK, n = per_part * p.parts, per = PAIR ? n : (n + ctas - 1) / ctas;
    kb0 = PAIR ? 0 : min(rank * per, n);
    kb1 = PAIR ? n : min(kb0 + per, n);
    return per_part;
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- copies
    if (ff_elect()) {
      asm volatile("fence.proxy.async;" ::: "memory");   // what earlier kernels stored is read through the async proxy
      uint32_t n = 0;
      bool dead = false;
      for (int tile = first; tile < a.tiles && !dead && !sm.abort; tile += step) {
        int tm, tn, kb0, kb1;
        const ff_product& p = locate(tile, tm, tn);
        const int per_part = share(p, kb0, kb1);
        for (int kb = kb0; kb < kb1; ++kb, ++n) {
          const uint32_t s = n % STAGES, use = n / STAGES;
          if (use > 0 && !ff_wait(&sm.empty[s], (use - 1) & 1, &sm.abort)) { dead = true; break; }
          // boxes that reach beyond the matrix are filled with zeros and count in full; of a pair the first CTA's barrier takes the bytes of both
          if (!PAIR || rank == 0) ff_expect(&sm.full[s], (PAIR ? 2 : 1) * STAGE);
          const uint32_t bar = PAIR ? nf_at_rank(&sm.full[s], 0) : smem_addr(&sm.full[s]);
          const int part = kb >= per_part, k = (kb - part * per_part) * FF_BK;
          uint32_t dst = smem_addr(sm.st[s]);
#pragma unroll
          for (int u = 0; u < 2; ++u, dst += FF_BOX) {
            const int mn = tm * TILE_M + (PAIR ? rank * FF_BM : 0) + 64 * u;
            ff_copy<PAIR>(dst, &p.A[part], bar, p.a_mn ? mn : k, p.a_mn ? k : mn);
          }
#pragma unroll
          for (int u = 0; u < 2; ++u, dst += FF_BOX) {
            int mn = tn * OUT_N + (PAIR ? rank * 128 : 0) + 64 * u, which = part;
            if constexpr (EPI == FF_GATE) {   // the first half of a tile's columns are Wg's, the second Wu's
              which = PAIR ? rank : u;
              mn = tn * OUT_N + (PAIR ? 64 * u : 0);
            }
            ff_copy<PAIR>(dst, &p.B[which], bar, p.b_mn ? mn : k, p.b_mn ? k : mn);
          }
        }
      }
      // the CTA must not end while a copy into its shared memory is in flight: normally the issuing lane has waited for every stage; after an
      // abort wait (bounded) for the stages filled last
      if ((!PAIR || rank == 0) && (dead || sm.abort))
        for (uint32_t f = n > STAGES ? n - STAGES : 0; f < n; ++f)
          for (int it = 0; it < FF_SPIN_LIMIT; ++it)
            if (ff_try(&sm.full[f % STAGES], (f / STAGES) & 1)) break;
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products (of a pair the first CTA issues them)
    if ((!PAIR || rank == 0) && ff_elect()) {
      uint32_t n = 0, c = 0;
      bool dead = false;
      for (int tile = first; tile < a.tiles && !dead && !sm.abort; tile += step, ++c) {
        int tm, tn, kb0, kb1;
        const ff_product& p = locate(tile, tm, tn);
        share(p, kb0, kb1);
        const uint32_t idesc = ff_idesc(TILE_M, BN, p.a_mn, p.b_mn, BF), acc = tmem + (c & 1) * 256;
        const uint64_t a_step = (p.a_mn ? 2048 : 32) >> 4, b_step = (p.b_mn ? 2048 : 32) >> 4;   // 16 terms further
        if (c >= 2) {   // the tile before the last has left its accumulator
          if (!ff_wait(&sm.free[c & 1], ((c >> 1) - 1) & 1, &sm.abort)) break;
          ff_fence_after();
        }
        for (int kb = kb0; kb < kb1; ++kb, ++n) {
          const uint32_t s = n % STAGES;
          if (!ff_wait(&sm.full[s], (n / STAGES) & 1, &sm.abort)) { dead = true; break; }
          ff_fence_after();
          const uint64_t da = ff_desc(smem_addr(sm.st[s]), p.a_mn), db = ff_desc(smem_addr(sm.st[s]) + 2 * FF_BOX, p.b_mn);
#pragma unroll
          for (int ks = 0; ks < FF_BK / 16; ++ks) ff_mma<PAIR>(acc, da + ks * a_step, db + ks * b_step, idesc, kb > kb0 || ks > 0);
          ff_commit<PAIR>(&sm.empty[s]);
        }
        if (!dead) ff_commit<PAIR>(&sm.ready[c & 1]);
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- epilogue: a warp's 32 rows, a half or a quarter of the tile's columns, COLS at a time
    constexpr int PARTS = WARPS / 4, BLOCKS = OUT_N / COLS / PARTS;   // BLOCKS of COLS columns for this warp
    const int quarter = warp & 3, part = (warp - 2) >> 2, e = warp - 2;
    const uint32_t t_lane = tmem + ((uint32_t)(quarter * 32) << 16);
    unsigned char* const stage = sm.out[e];
    uint32_t c = 0;
    // BACK: the block of P and Q that is on its way
    struct { int tile, q; } ahead = {first, -1};
    uint4 coming[EPI == FF_BACK ? FF_KEPT_PIECES : 1] = {};
    auto ask = [&] {   // for the one behind it that has rows and columns
      ++ahead.q;
      for (; ahead.tile < a.tiles; ahead.tile += step, ahead.q = 0) {
        int tm, tn;
        const ff_product& p = locate(ahead.tile, tm, tn);
        const int m = tm * TILE_M + (PAIR ? rank * FF_BM : 0) + quarter * 32, n = tn * OUT_N + COLS * (part * BLOCKS + ahead.q);
        if (ahead.q >= BLOCKS || m >= p.M || n >= p.N) continue;
        const uint4* const from = ff_block(a.kept, m, a.ld, n);
#pragma unroll
        for (int i = 0; i < (EPI == FF_BACK ? FF_KEPT_PIECES : 1); ++i) coming[i] = __ldcs(from + 32 * i);
        break;
      }
    };
    if (EPI == FF_BACK && (PAIR || rank == 0)) ask();
    for (int tile = first; tile < a.tiles && !sm.abort; tile += step, ++c) {
      int tm, tn, kb0, kb1;
      const ff_product& p = locate(tile, tm, tn);
      share(p, kb0, kb1);
      const int m0 = tm * TILE_M + (PAIR ? rank * FF_BM : 0) + quarter * 32, rows = p.M - m0;
      if (!ff_wait(&sm.ready[c & 1], (c >> 1) & 1, &sm.abort, kb1 - kb0)) break;
      ff_fence_after();
      const uint32_t acc = t_lane + (c & 1) * 256;
      bool leave = false;
      if constexpr (!PAIR) {
        // this CTA's sums, where another one has the tile: the stages are free, all products being done
        if (rank > 0) {
          constexpr int MINE = BN / COLS / PARTS;
          for (int q = 0; q < MINE; ++q) {
            const int block = part * MINE + q;
            float v[COLS];
            ff_ld(acc + COLS * block, v);
            const bool none = kb0 == kb1;   // no share: nothing has been written there
            float4* const box = reinterpret_cast<float4*>(sm.st) + (block * 4 + quarter) * 8 * COLS + lane;
#pragma unroll
            for (int j = 0; j < COLS / 4; ++j) box[32 * j] = none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          }
          __syncwarp();
          if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(nf_at_rank(&sm.sums, 0)) : "memory");
          leave = true;
        } else if (ctas > 1) {
          if (!ff_wait(&sm.sums, 0, &sm.abort, kb1 - kb0)) break;
          asm volatile("fence.acq_rel.cluster;" ::: "memory");
        }
      }
      // COLS columns of the tile's sums
      auto tile_sums = [&](int block, float (&v)[COLS]) {
        ff_ld(acc + COLS * block, v);
        if constexpr (!PAIR) {
          for (int r = 1; r < ctas; ++r) {
            const uint32_t src = nf_at_rank(reinterpret_cast<float4*>(sm.st) + (block * 4 + quarter) * 8 * COLS + lane, r);
#pragma unroll
            for (int j = 0; j < COLS / 4; ++j) {
              float4 o;
              asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(o.x), "=f"(o.y), "=f"(o.z), "=f"(o.w) : "r"(src + 512 * j) : "memory");
              v[4 * j] += o.x; v[4 * j + 1] += o.y; v[4 * j + 2] += o.z; v[4 * j + 3] += o.w;
            }
          }
        }
      };
      int left = BLOCKS;                   // of them to be read; behind the last, the accumulator is free
      auto read = [&] {
        if (--left > 0) return;
        ff_fence_before();
        __syncwarp();
        if (lane == 0) ff_arrive<PAIR>(&sm.free[c & 1]);
      };
      if (!leave && rows > 0) {
#pragma unroll 1
        for (int q = 0; q < BLOCKS; ++q) {
          const int block = part * BLOCKS + q, n0 = tn * OUT_N + COLS * block, cols = p.N - n0;
          if (cols <= 0) break;
          if constexpr (EPI == FF_PLAIN) {
            float v[32];
            tile_sums(block, v);
            read();
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = ff_pack<BF>(v[2 * j], v[2 * j + 1]);
            if (!p.mapped) ff_store16(stage, w, (uint16_t*)p.C + (long long)m0 * p.ldc + n0, p.ldc, rows, cols);
            else {
              // 64 columns to a copy, rows of 128 bytes in its swizzle
              if (!(q & 1)) {
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // the copy before has read the stage
                __syncwarp();
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint4*>(stage + lane * 128 + 16 * ((4 * (q & 1) + i) ^ (lane & 7))) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
              if ((q & 1) || cols <= 32) {   // (what lies behind the matrix is not written, whatever the stage holds there)
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                  ff_send(&p.Cm, stage, n0 - 32 * (q & 1), m0);
                  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
              }
            }
          } else if constexpr (EPI == FF_GATE) {
            float g[COLS], u[COLS], q_[COLS];
            tile_sums(block, g);
            tile_sums(block + OUT_N / COLS, u);
            read();
            uint32_t w[COLS / 2];
#pragma unroll
            for (int j = 0; j < COLS / 2; ++j) {
              float slope[2], h[2];
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                ff_act(a.activation, g[2 * j + i], q_[2 * j + i], slope[i]);
                h[i] = q_[2 * j + i] * u[2 * j + i];
                u[2 * j + i] *= slope[i];
              }
              w[j] = ff_pack<BF>(h[0], h[1]);
            }
            // h: out by copies from shared memory, rows of 32 bytes in their swizzle
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // the block before has left
            __syncwarp();
            ff_put32(stage, w);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              ff_send(&a.planes[0], stage, n0, m0);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
            if (a.keep) {
              uint4* const to = ff_block(a.kept, m0, a.ld, n0);
              ff_put24(to, 0, u);
              ff_put24(to, 1, q_);
            }
          } else {
            float v[COLS], f[COLS];
            tile_sums(block, v);
            read();
            uint32_t w[2][COLS / 2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              ff_take24(coming, k, f);
#pragma unroll
              for (int j = 0; j < COLS / 2; ++j) w[k][j] = ff_pack<BF>(v[2 * j] * f[2 * j], v[2 * j + 1] * f[2 * j + 1]);
            }
            ask();
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // the block before has left
            __syncwarp();
            ff_put32(stage, w[0]);
            ff_put32(stage + 1024, w[1]);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              ff_send(&a.planes[0], stage, n0, m0);
              ff_send(&a.planes[1], stage + 1024, n0, m0);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          }
        }
      }
      if (left > 0) {   // nothing of the tile, or not all of it, lies in the matrix
        left = 1;
        read();
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  ff_fence_before();
  __syncthreads();
  cluster_sync();   // no CTA leaves while another may reach into its shared memory
  if (tid == 0 && sm.abort) {
    if (a.status) atomicOr(a.status, 16);
    if (a.host_status) *reinterpret_cast<volatile int*>(a.host_status) = 16;
  }
  if (warp == 1) {
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ------------------------------------------------------------------------------------------------
// Few rows (32 at most): the weights' bytes are the cost, so as many of them as possible are on their way.  The weights are operand A, 128 rows of them to
// a tile, the rows of x operand B, ROWS = 16 or 32 of them: a stage is 16 KB of weights and 2 or 4 KB of the rest (the tiles above hold 16 KB of each,
// nearly all of the latter zeros), and two CTAs share an SM.  A tile's sums lie feature by feature in the lanes, row by row in the columns, so that a
// warp's lanes write neighbours.  The CTAs of a cluster share a tile as above.  Gate: a tile has 64 rows of Wg and the same 64 of Wu; the warps
// of the latter hand their sums to those of the former.
//
// Up to FF_FINE rows, h, dg and du are 16 bits and 16 more of what their rounding left, FF_FINE rows below: of so few values the roundings' average may be far
// from what it is expected to be, and as more rows of operand B, beside the same weights, they cost next to nothing.  The result adds both rows' sums up; the
// weights' gradients take them as two parts of their contractions.
// ------------------------------------------------------------------------------------------------
#define FF_FEW 32
#define FF_FINE 16
#define FF_FEW_THREADS 192
template <int ROWS>
struct FfFewSmem {
  static constexpr int STAGES = ROWS == 16 ? 6 : 5, B_BYTES = ROWS * 128, STAGE = 2 * FF_BOX + B_BYTES;
  unsigned char st[STAGES][STAGE];
  uint64_t full[STAGES], empty[STAGES], ready, sums;
  uint32_t tmem;
  volatile int abort;
};
__device__ __forceinline__ float ff_load24(const uint16_t* hi, const uint8_t* lo, long long i) {
  return __uint_as_float((uint32_t)hi[i] << 16 | (uint32_t)lo[i] << 8);
}
__device__ __forceinline__ void ff_keep24(uint16_t* hi, uint8_t* lo, long long i, float v) {
  const uint32_t b = ff_round24(v);
  hi[i] = (uint16_t)(b >> 16);
  lo[i] = (uint8_t)(b >> 8);
}
template <bool BF>
__device__ __forceinline__ uint16_t ff_one(float v) { return (uint16_t)ff_pack<BF>(v, 0.f); }
// A value that becomes an operand: rounded, and FF_FINE rows below what that left of it
template <bool BF>
__device__ __forceinline__ void ff_two(uint16_t* to, long long ld, bool fine, float v) {
  const uint16_t high = ff_one<BF>(v);
  *to = high;
  if (fine) {
    float f;
    if constexpr (BF) f = __uint_as_float((uint32_t)high << 16);
    else f = __half2float(__ushort_as_half(high));
    to[FF_FINE * ld] = fabsf(f) < CUDART_INF_F ? ff_one<BF>(v - f) : 0;
  }
}

template <int EPI, bool BF, int ROWS>
__global__ void __launch_bounds__(FF_FEW_THREADS, 2) k_ffn_few(const __grid_constant__ ff_args a) {
  extern __shared__ unsigned char ff_dyn[];
  using Smem = FfFewSmem<ROWS>;
  constexpr int STAGES = Smem::STAGES, COLUMNS = 32, OUT_M = EPI == FF_GATE ? 64 : 128;
  Smem& sm = *reinterpret_cast<Smem*>(ff_dyn + ((1024 - (smem_addr(ff_dyn) & 1023)) & 1023));   // at the same place in all CTAs of a cluster
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int rank = (int)ff_cluster_rank(), ctas = (int)ff_cluster_size();
  const ff_product& p = a.p[0];
  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) { ff_init(&sm.full[s], 1); ff_init(&sm.empty[s], 1); }
    ff_init(&sm.ready, 1);
    ff_init(&sm.sums, ctas > 1 ? (ctas - 1) * 4 : 1);
    sm.abort = 0;
  }
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  ff_take_tmem<false>(&sm.tmem, COLUMNS, warp);
  ff_fence_before();
  __syncthreads();
  cluster_sync();   // the other CTAs' barriers exist
  ff_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
  const int tile = (int)blockIdx.x / ctas, per_part = (p.K + FF_BK - 1) / FF_BK, n_kb = per_part * p.parts, per = (n_kb + ctas - 1) / ctas;
  const int kb0 = min(rank * per, n_kb), kb1 = min(kb0 + per, n_kb);
  if (warp == 0) {
    // ---------------------------------------------------------------- copies
    if (ff_elect()) {
      asm volatile("fence.proxy.async;" ::: "memory");   // what earlier kernels stored is read through the async proxy
      uint32_t n = 0;
      bool dead = false;
      for (int kb = kb0; kb < kb1; ++kb, ++n) {
        const uint32_t s = n % STAGES, use = n / STAGES;
        if (use > 0 && !ff_wait(&sm.empty[s], (use - 1) & 1, &sm.abort)) { dead = true; break; }
        ff_expect(&sm.full[s], Smem::STAGE);   // boxes that reach beyond the matrix are filled with zeros and count in full
        const uint32_t bar = smem_addr(&sm.full[s]);
        const int part = kb >= per_part, k = (kb - part * per_part) * FF_BK;
        uint32_t dst = smem_addr(sm.st[s]);
#pragma unroll
        for (int u = 0; u < 2; ++u, dst += FF_BOX) {
          const int mn = EPI == FF_GATE ? tile * 64 : tile * 128 + 64 * u, which = EPI == FF_GATE ? u : part;
          ff_copy<false>(dst, &p.A[which], bar, p.a_mn ? mn : k, p.a_mn ? k : mn);
        }
        ff_copy<false>(dst, &p.B[part], bar, k, 0);
      }
      // the CTA must not end while a copy into its shared memory is in flight
      if (dead || sm.abort)
        for (uint32_t f = n > STAGES ? n - STAGES : 0; f < n; ++f)
          for (int it = 0; it < FF_SPIN_LIMIT; ++it)
            if (ff_try(&sm.full[f % STAGES], (f / STAGES) & 1)) break;
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products
    if (ff_elect()) {
      uint32_t n = 0;
      bool dead = false;
      const uint32_t idesc = ff_idesc(128, ROWS, p.a_mn, 0, BF);
      const uint64_t a_step = (p.a_mn ? 2048 : 32) >> 4;   // 16 terms further
      for (int kb = kb0; kb < kb1; ++kb, ++n) {
        const uint32_t s = n % STAGES;
        if (!ff_wait(&sm.full[s], (n / STAGES) & 1, &sm.abort)) { dead = true; break; }
        ff_fence_after();
        const uint64_t da = ff_desc(smem_addr(sm.st[s]), p.a_mn), db = ff_desc(smem_addr(sm.st[s]) + 2 * FF_BOX, 0);
#pragma unroll
        for (int ks = 0; ks < FF_BK / 16; ++ks) ff_mma<false>(tmem, da + ks * a_step, db + ks * 2, idesc, kb > kb0 || ks > 0);
        ff_commit<false>(&sm.empty[s]);
      }
      if (!dead) ff_commit<false>(&sm.ready);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- a thread per feature
    const int quarter = warp & 3, at = quarter * 32 + lane;   // of the tile's 128
    bool good = ff_wait(&sm.ready, 0, &sm.abort, kb1 - kb0);
    ff_fence_after();
    float v[ROWS];
    if (good) {
#pragma unroll
      for (int j = 0; j < ROWS; j += 16) {
        uint32_t r[16];
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
              "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(tmem + ((uint32_t)(quarter * 32) << 16) + j) : "memory");
#pragma unroll
        for (int i = 0; i < 16; ++i) v[j + i] = kb1 > kb0 ? __uint_as_float(r[i]) : 0.f;   // (no share of the contraction: nothing has been written there)
      }
    }
    float* const box = reinterpret_cast<float*>(sm.st);   // the stages are free: all products are done
    if (rank > 0) {
      if (good) {
#pragma unroll
        for (int n = 0; n < ROWS; ++n) box[n * 128 + at] = v[n];
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(nf_at_rank(&sm.sums, 0)) : "memory");
      }
    } else {
      if (good && ctas > 1) {
        good = ff_wait(&sm.sums, 0, &sm.abort, kb1 - kb0);
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
        if (good)
          for (int r = 1; r < ctas; ++r) {   // in rank order
            const uint32_t src = nf_at_rank(box + at, r);
#pragma unroll
            for (int n = 0; n < ROWS; ++n) {
              float o;
              asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o) : "r"(src + 512 * n) : "memory");
              v[n] += o;
            }
          }
      }
      good = __all_sync(0xffffffffu, good);
      const int f = tile * OUT_M + (EPI == FF_GATE ? at & 63 : at);   // the feature
      if constexpr (EPI == FF_GATE) {
        if (at >= 64) {
#pragma unroll
          for (int n = 0; n < ROWS; ++n) box[n * 64 + at - 64] = v[n];
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");   // the four warps of the epilogue
        if (good && at < 64 && f < p.M) {
#pragma unroll
          for (int n0 = 0; n0 < ROWS; n0 += 8) {   // eight rows at a time
            if (n0 >= p.N) break;
#pragma unroll
            for (int n = n0; n < n0 + 8; ++n)
              if (n < p.N) {
                const float u = box[n * 64 + at];
                float q, slope;
                ff_act(a.activation, v[n], q, slope);
                ff_two<BF>(a.kept.h + n * a.ld + f, a.ld, ROWS == FF_FINE, q * u);
                if (a.keep) {
                  const long long i = ff_place(n, a.ld, f);
                  ff_keep24(a.kept.hi, a.kept.lo, i, u * slope);
                  ff_keep24(a.kept.hi, a.kept.lo, i + 16, q);
                }
              }
          }
        }
      } else if (good && f < p.M) {
        if (EPI == FF_PLAIN && p.N <= FF_FINE) {
#pragma unroll
          for (int n = 0; n < ROWS - FF_FINE; ++n) v[n] += v[n + FF_FINE];
        }
#pragma unroll
        for (int n0 = 0; n0 < ROWS; n0 += 8) {
          if (n0 >= p.N) break;
          if constexpr (EPI == FF_PLAIN) {
#pragma unroll
            for (int n = n0; n < n0 + 8; ++n)
              if (n < p.N) ((uint16_t*)p.C)[n * p.ldc + f] = ff_one<BF>(v[n]);
          } else {
            float pf[8], qf[8];   // on their way together
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const long long i = ff_place(min(n0 + j, p.N - 1), a.ld, f);
              pf[j] = ff_load24(a.kept.hi, a.kept.lo, i);
              qf[j] = ff_load24(a.kept.hi, a.kept.lo, i + 16);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (n0 + j < p.N) {
                const long long i = (n0 + j) * a.ld + f;
                ff_two<BF>(a.dg + i, a.ld, ROWS == FF_FINE, v[n0 + j] * pf[j]);
                ff_two<BF>(a.du + i, a.ld, ROWS == FF_FINE, v[n0 + j] * qf[j]);
              }
          }
        }
      }
    }
  }
  ff_fence_before();
  __syncthreads();
  cluster_sync();   // no CTA leaves while another may reach into its shared memory
  if (tid == 0 && sm.abort) {
    if (a.status) atomicOr(a.status, 16);
    if (a.host_status) *reinterpret_cast<volatile int*>(a.host_status) = 16;
  }
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLUMNS) : "memory");
}

// ------------------------------------------------------------------------------------------------
// Operands whose rows do not begin on 16-byte boundaries, copied so that they do: 16 bytes of the copy to a thread, all matrices in one launch
// ------------------------------------------------------------------------------------------------
#define FF_PADS 4
struct ff_pads {
  pylo_pad p[FF_PADS];
  long long first[FF_PADS + 1];   // pieces of 8 elements of the matrices before
  int n;
};
__global__ void __launch_bounds__(NT) k_ffn_pad(const ff_pads a) {
  pdl_begin();
  for (long long i = (long long)blockIdx.x * NT + threadIdx.x; i < a.first[a.n]; i += (long long)gridDim.x * NT) {
    int k = 0;
    while (k + 1 < a.n && i >= a.first[k + 1]) ++k;
    const pylo_pad& p = a.p[k];
    const long long at = i - a.first[k];
    const uint32_t per = (uint32_t)(p.ld / 8);
    const long long row = at < (1ll << 32) ? (uint32_t)at / per : at / per, c = (at - row * per) * 8;
    const uint16_t* const src = (const uint16_t*)p.src + row * p.row_stride + c * p.col_stride;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < p.cols) w[j >> 1] |= (uint32_t)src[j * p.col_stride] << (16 * (j & 1));
    *reinterpret_cast<uint4*>((uint16_t*)p.dst + row * p.ld + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
typedef CUresult (*FfEncode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static FfEncode ff_encode() {
  static FfEncode fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
    return (FfEncode)p;
  }();
  return fn;
}
// [rows][cols] of 16-bit elements, boxes of so many rows of 64; what a box reaches beyond the matrix reads as zero
static int ff_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld, int type, int box_rows = 64) {
  FfEncode fn = ff_encode();
  if (!fn) return -5;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, unit[2] = {1, 1};
  return fn(map, type == PYLO_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base), dims, strides, box, unit,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -5;
}

// Encoding a tensor map wants the device's context to be the thread's current one, which a thread that has only asked for the device (autograd's, at its
// first backward pass) need not have.
static int ff_begin() {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaSetDevice(dev);
  return (int)e;
}
static int64_t ff_ld(int hidden) { return ((int64_t)hidden + 15) / 16 * 16; }   // of h and what is made like it
static int64_t ff_plane(int64_t rows, int hidden, int bytes) { return (rows * ff_ld(hidden) * bytes + 255) / 256 * 256; }
static int64_t ff_rows(int64_t rows) { return rows <= FF_FINE ? FF_FINE + rows : rows; }   // of h, dg, du
static int64_t ff_kept_bytes(int64_t rows, int hidden) { return ff_plane(rows <= FF_FEW ? rows : (rows + 31) / 32 * 32, hidden, 6) + 256; }   // of P and Q: planes or blocks
static ff_kept ff_planes(void* base, int64_t rows, int hidden) {
  char* const p = (char*)base + ff_plane(ff_rows(rows), hidden, 2);
  return {(uint16_t*)base, (uint4*)p, (uint16_t*)p, (uint8_t*)(p + ff_plane(rows, hidden, 4))};
}

// Which form a product takes.  Pairs where their tiles, with those of the products beside it whose contractions are equally long, fill the GPU more than half
// (74 run at once): rows x 1024 by 1024 x 4096, both projections, 512 rows (64 tiles) 17 us and 22 in tiles of 128 x 128, 256 rows (32) 16 and 13.
static int ff_length(const ff_product& p) { return p.K * p.parts; }
static bool ff_pairs(const ff_args& all, const ff_product& q, int epi) {
  int64_t tiles = 0;
  for (int k = 0; k < all.n; ++k) {
    const ff_product& p = all.p[k];
    if (ff_length(p) == ff_length(q)) tiles += (int64_t)((p.M + 255) / 256) * ((p.N + (epi == FF_GATE ? 127 : 255)) / (epi == FF_GATE ? 128 : 256));
  }
  return tiles >= 48;
}
template <bool PAIR, int EPI, bool BF>
static int ff_go(ff_args& a, cudaStream_t s) {
  constexpr int TILE_M = PAIR ? 256 : 128, TILE_N = (PAIR ? 256 : 128) / (EPI == FF_GATE ? 2 : 1);
  int64_t tiles = 0;
  int longest = 1;
  for (int k = 0; k < a.n; ++k) {
    ff_product& p = a.p[k];
    p.tiles_m = (p.M + TILE_M - 1) / TILE_M;
    p.tiles_n = (p.N + TILE_N - 1) / TILE_N;
    p.tile0 = (int)tiles;
    tiles += (int64_t)p.tiles_m * p.tiles_n;
    const int blocks = (p.K + FF_BK - 1) / FF_BK * p.parts;
    if (blocks > longest) longest = blocks;
  }
  if (tiles > (1 << 27)) return -1;
  a.tiles = (int)tiles;
  if (!tiles) return 0;
  static bool configured[PYLO_MAX_DEVICES] = {};
  constexpr int SMEM = (int)sizeof(FfSmem<EPI>) + 1024;
  if (int rc = allow_dynamic_smem(k_ffn_product<PAIR, EPI, BF>, SMEM, configured)) return rc;
  int cluster = 2, grid;
  if constexpr (PAIR) {
    const int pairs = sm_count() / 2;
    grid = 2 * (int)(tiles < pairs ? tiles : pairs);
  } else {
    // how many CTAs share a tile, by the time that is to be expected: 0.15 us a stage, and what a tile costs besides
    float best = 0.f;
    for (int c = 1; c <= 8; c *= 2) {
      const int64_t at_once = active_clusters<k_ffn_product<PAIR, EPI, BF>>(ff_threads(EPI), c, SMEM), waves = (tiles + at_once - 1) / at_once;
      const float t = (float)waves * (0.15f * (float)((longest + c - 1) / c) + (c > 1 ? 4.0f + 0.3f * (float)c : 3.0f));
      if (c == 1 || t < best) { best = t; cluster = c; }
    }
    grid = (int)tiles * cluster;
  }
  launch_clusters(k_ffn_product<PAIR, EPI, BF>, grid, ff_threads(EPI), cluster, SMEM, s, a);
  return launch_status();
}
// The products of a that take pairs in one launch, the others in one for those whose contractions are equally long
template <int EPI>
static int ff_run(const ff_args& all, int type, cudaStream_t s) {
  ff_args a = all;
  a.n = 0;
  for (int k = 0; k < all.n; ++k)
    if (ff_pairs(all, all.p[k], EPI)) a.p[a.n++] = all.p[k];
  if (a.n)
    if (int rc = type == PYLO_BF16 ? ff_go<true, EPI, true>(a, s) : ff_go<true, EPI, false>(a, s)) return rc;
  bool done[FF_GROUP] = {};
  for (int k = 0; k < all.n; ++k) {
    if (done[k] || ff_pairs(all, all.p[k], EPI)) continue;
    a.n = 0;
    for (int j = k; j < all.n; ++j)
      if (ff_length(all.p[j]) == ff_length(all.p[k])) {
        a.p[a.n++] = all.p[j];
        done[j] = true;
      }
    if (int rc = type == PYLO_BF16 ? ff_go<false, EPI, true>(a, s) : ff_go<false, EPI, false>(a, s)) return rc;
  }
  return 0;
}
// Few rows: a.p[0] as it is for many, C[rows][features]; the operands change places
template <int EPI, bool BF, int ROWS>
static int ff_go_few(ff_args& a, cudaStream_t s) {
  constexpr int SMEM = (int)sizeof(FfFewSmem<ROWS>) + 1024;
  const int tiles = (a.p[0].M + (EPI == FF_GATE ? 63 : 127)) / (EPI == FF_GATE ? 64 : 128), blocks = (a.p[0].K + FF_BK - 1) / FF_BK * a.p[0].parts;
  static bool configured[PYLO_MAX_DEVICES] = {};
  if (int rc = allow_dynamic_smem(k_ffn_few<EPI, BF, ROWS>, SMEM, configured)) return rc;
  // the CTAs that share a tile: as many as run at once, each with two stages at least
  int cluster = 1;
  while (cluster < 8 && blocks >= cluster * 2 * 2 && tiles <= active_clusters<k_ffn_few<EPI, BF, ROWS>>(FF_FEW_THREADS, cluster * 2, SMEM)) cluster *= 2;
  launch_clusters(k_ffn_few<EPI, BF, ROWS>, tiles * cluster, FF_FEW_THREADS, cluster, SMEM, s, a);
  return launch_status();
}
template <int EPI>
static int ff_run_few(ff_args& a, int rows, int type, cudaStream_t s) {
  const bool bf = type == PYLO_BF16;
  if constexpr (EPI != FF_PLAIN)
    if (rows <= FF_FINE) return bf ? ff_go_few<EPI, true, 16>(a, s) : ff_go_few<EPI, false, 16>(a, s);
  return bf ? ff_go_few<EPI, true, 32>(a, s) : ff_go_few<EPI, false, 32>(a, s);
}
static int ff_few_rows(int64_t rows) { return rows > FF_FEW ? 0 : rows <= FF_FINE ? FF_FINE : FF_FEW; }   // of a tile; 0: not few
static bool ff_operand(const void* p, int64_t ld, int64_t cols) { return p && ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && ld >= cols; }
static bool ff_good(const pylo_ffn* f) {
  return f && f->rows >= 0 && f->rows <= (1 << 30) && f->width > 0 && f->hidden > 0 && f->out > 0 && f->width <= (1 << 24) && f->hidden <= (1 << 24) &&
         f->out <= (1 << 24) && (f->type == PYLO_BF16 || f->type == PYLO_FP16) && f->activation >= PYLO_ACT_SILU && f->activation <= PYLO_ACT_RELU &&
         (((uintptr_t)f->y | (uintptr_t)f->dx | (uintptr_t)f->dw_gate | (uintptr_t)f->dw_up | (uintptr_t)f->dw_down) & 1) == 0 &&
         (((uintptr_t)f->status | (uintptr_t)f->host_status) & 3) == 0;
}
// Maps of [rows][hidden] that an epilogue writes: boxes of 32 rows and 16 columns
static int ff_map_planes(ff_args& a, int64_t rows, int64_t hidden, void* first, void* second) {
  FfEncode fn = ff_encode();
  if (!fn) return -5;
  const cuuint64_t dims[2] = {(cuuint64_t)hidden, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)a.ld * 2};
  const cuuint32_t box[2] = {16, 32}, unit[2] = {1, 1};
  for (int i = 0; i < (second ? 2 : 1); ++i)
    if (fn(&a.planes[i], CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, i ? second : first, dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_32B,
           CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) return -5;
  return 0;
}
// C's map, where its rows allow for one: boxes of 32 rows of 64
static int ff_map_c(ff_product& p, int type) {
  p.mapped = ((uintptr_t)p.C & 15) == 0 && p.ldc % 8 == 0;
  return p.mapped ? ff_map(&p.Cm, p.C, p.M, p.N, p.ldc, type, 32) : 0;
}
static ff_product ff_of(void* C, int64_t ldc, int64_t M, int64_t N, int64_t K, int parts, int a_mn, int b_mn) {
  ff_product p = {};
  p.C = C; p.ldc = ldc; p.M = (int)M; p.N = (int)N; p.K = (int)K; p.parts = parts; p.a_mn = a_mn; p.b_mn = b_mn;
  return p;
}

extern "C" {

int64_t pylo_b200_gated_ffn_kept(int64_t rows, int hidden, int keep) {
  if (rows <= 0 || hidden <= 0) return 0;
  return ff_plane(ff_rows(rows), hidden, 2) + (keep ? ff_kept_bytes(rows, hidden) : 0);
}
int64_t pylo_b200_gated_ffn_workspace(int64_t rows, int hidden) { return rows <= 0 || hidden <= 0 ? 0 : 2 * ff_plane(ff_rows(rows), hidden, 2); }

int pylo_b200_gated_ffn(const pylo_ffn* f, void* stream) {
  CHECK_ARG(ff_good(f));
  if (f->rows == 0) return 0;
  CHECK_ARG(ff_operand(f->x, f->ld_x, f->width) && ff_operand(f->w_gate, f->ld_gate, f->width) && ff_operand(f->w_up, f->ld_up, f->width) &&
            ff_operand(f->w_down, f->ld_down, f->hidden) && f->y && f->kept && ((uintptr_t)f->kept & 255) == 0);
  if (int rc = ff_begin()) return rc;
  const ff_kept kept = ff_planes(f->kept, f->rows, f->hidden);
  const int64_t ld = ff_ld(f->hidden);
  ff_args a = {};
  a.kept = kept; a.ld = ld; a.n = 1; a.activation = f->activation; a.keep = f->keep; a.status = f->status; a.host_status = f->host_status;
  cudaStream_t s = (cudaStream_t)stream;
  if (const int few = ff_few_rows(f->rows)) {
    const bool fine = few == FF_FINE;
    a.p[0] = ff_of(nullptr, 0, f->hidden, f->rows, f->width, 1, 0, 0);
    if (int rc = ff_map(&a.p[0].A[0], f->w_gate, f->hidden, f->width, f->ld_gate, f->type)) return rc;
    if (int rc = ff_map(&a.p[0].A[1], f->w_up, f->hidden, f->width, f->ld_up, f->type)) return rc;
    if (int rc = ff_map(&a.p[0].B[0], f->x, f->rows, f->width, f->ld_x, f->type, few)) return rc;
    if (int rc = ff_run_few<FF_GATE>(a, (int)f->rows, f->type, s)) return rc;
    a.p[0] = ff_of(f->y, f->out, f->out, f->rows, f->hidden, 1, 0, 0);
    if (int rc = ff_map(&a.p[0].A[0], f->w_down, f->out, f->hidden, f->ld_down, f->type)) return rc;
    if (int rc = ff_map(&a.p[0].B[0], kept.h, fine ? FF_FINE + f->rows : f->rows, f->hidden, ld, f->type, FF_FEW)) return rc;
    return ff_run_few<FF_PLAIN>(a, (int)f->rows, f->type, s);
  }
  a.p[0] = ff_of(nullptr, 0, f->rows, f->hidden, f->width, 1, 0, 0);
  if (int rc = ff_map(&a.p[0].A[0], f->x, f->rows, f->width, f->ld_x, f->type)) return rc;
  if (int rc = ff_map(&a.p[0].B[0], f->w_gate, f->hidden, f->width, f->ld_gate, f->type)) return rc;
  if (int rc = ff_map(&a.p[0].B[1], f->w_up, f->hidden, f->width, f->ld_up, f->type)) return rc;
  if (int rc = ff_map_planes(a, f->rows, f->hidden, kept.h, nullptr)) return rc;
  if (int rc = ff_run<FF_GATE>(a, f->type, s)) return rc;
  a.p[0] = ff_of(f->y, f->out, f->rows, f->out, f->hidden, 1, 0, 0);
  if (int rc = ff_map(&a.p[0].A[0], kept.h, f->rows, f->hidden, ld, f->type)) return rc;
  if (int rc = ff_map(&a.p[0].B[0], f->w_down, f->out, f->hidden, f->ld_down, f->type)) return rc;
  if (int rc = ff_map_c(a.p[0], f->type)) return rc;
  return ff_run<FF_PLAIN>(a, f->type, s);
}

int pylo_b200_gated_ffn_backward(const pylo_ffn* f, void* stream) {
  CHECK_ARG(ff_good(f) && f->rows > 0);
  const bool inner = f->dx || f->dw_gate || f->dw_up;
  CHECK_ARG(ff_operand(f->dy, f->ld_dy, f->out) && f->kept && ((uintptr_t)f->kept & 255) == 0);
  CHECK_ARG(!inner || (ff_operand(f->w_down, f->ld_down, f->hidden) && f->work && ((uintptr_t)f->work & 255) == 0));
  CHECK_ARG(!f->dx || (ff_operand(f->w_gate, f->ld_gate, f->width) && ff_operand(f->w_up, f->ld_up, f->width)));
  CHECK_ARG(!(f->dw_gate || f->dw_up) || ff_operand(f->x, f->ld_x, f->width));
  if (int rc = ff_begin()) return rc;
  const ff_kept kept = ff_planes(f->kept, f->rows, f->hidden);
  const int64_t ld = ff_ld(f->hidden);
  ff_args a = {};
  a.kept = kept; a.ld = ld; a.activation = f->activation; a.status = f->status; a.host_status = f->host_status;
  a.dg = (uint16_t*)f->work;
  a.du = (uint16_t*)((char*)f->work + ff_plane(ff_rows(f->rows), f->hidden, 2));
  cudaStream_t s = (cudaStream_t)stream;
  const int few = ff_few_rows(f->rows);
  const bool fine = few == FF_FINE;
  if (inner) {   // dh (m: rows, n: hidden, k: out), Wd's rows being the contraction index
    a.n = 1;
    if (few) {
      a.p[0] = ff_of(nullptr, 0, f->hidden, f->rows, f->out, 1, 1, 0);
      if (int rc = ff_map(&a.p[0].A[0], f->w_down, f->out, f->hidden, f->ld_down, f->type)) return rc;
      if (int rc = ff_map(&a.p[0].B[0], f->dy, f->rows, f->out, f->ld_dy, f->type, few)) return rc;
      if (int rc = ff_run_few<FF_BACK>(a, (int)f->rows, f->type, s)) return rc;
    } else {
      a.p[0] = ff_of(nullptr, 0, f->rows, f->hidden, f->out, 1, 0, 1);
      if (int rc = ff_map(&a.p[0].A[0], f->dy, f->rows, f->out, f->ld_dy, f->type)) return rc;
      if (int rc = ff_map(&a.p[0].B[0], f->w_down, f->out, f->hidden, f->ld_down, f->type)) return rc;
      if (int rc = ff_map_planes(a, f->rows, f->hidden, a.dg, a.du)) return rc;
      if (int rc = ff_run<FF_BACK>(a, f->type, s)) return rc;
    }
  }
  if (f->dx && few) {
    a.p[0] = ff_of(f->dx, f->width, f->width, f->rows, f->hidden, 2, 1, 0);
    if (int rc = ff_map(&a.p[0].A[0], f->w_gate, f->hidden, f->width, f->ld_gate, f->type)) return rc;
    if (int rc = ff_map(&a.p[0].A[1], f->w_up, f->hidden, f->width, f->ld_up, f->type)) return rc;
    for (int k = 0; k < 2; ++k)
      if (int rc = ff_map(&a.p[0].B[k], k ? a.du : a.dg, fine ? FF_FINE + f->rows : f->rows, f->hidden, ld, f->type, FF_FEW)) return rc;
    if (int rc = ff_run_few<FF_PLAIN>(a, (int)f->rows, f->type, s)) return rc;
  }
  a.n = 0;
  if (f->dx && !few) {
    ff_product& p = a.p[a.n++] = ff_of(f->dx, f->width, f->rows, f->width, f->hidden, 2, 0, 1);
    if (int rc = ff_map(&p.A[0], a.dg, f->rows, f->hidden, ld, f->type)) return rc;
    if (int rc = ff_map(&p.A[1], a.du, f->rows, f->hidden, ld, f->type)) return rc;
    if (int rc = ff_map(&p.B[0], f->w_gate, f->hidden, f->width, f->ld_gate, f->type)) return rc;
    if (int rc = ff_map(&p.B[1], f->w_up, f->hidden, f->width, f->ld_up, f->type)) return rc;
  }
  for (int k = 0; k < 2; ++k)
    if (void* const out = k ? f->dw_up : f->dw_gate) {
      ff_product& p = a.p[a.n++] = ff_of(out, f->width, f->hidden, f->width, f->rows, 1 + fine, 1, 1);
      for (int i = 0; i <= (int)fine; ++i) {
        if (int rc = ff_map(&p.A[i], (k ? a.du : a.dg) + i * FF_FINE * ld, f->rows, f->hidden, ld, f->type)) return rc;
        if (int rc = ff_map(&p.B[i], f->x, f->rows, f->width, f->ld_x, f->type)) return rc;
      }
    }
  if (f->dw_down) {
    ff_product& p = a.p[a.n++] = ff_of(f->dw_down, f->hidden, f->out, f->hidden, f->rows, 1 + fine, 1, 1);
    for (int i = 0; i <= (int)fine; ++i) {
      if (int rc = ff_map(&p.A[i], f->dy, f->rows, f->out, f->ld_dy, f->type)) return rc;
      if (int rc = ff_map(&p.B[i], kept.h + i * FF_FINE * ld, f->rows, f->hidden, ld, f->type)) return rc;
    }
  }
  for (int k = 0; k < a.n; ++k)
    if (int rc = ff_map_c(a.p[k], f->type)) return rc;
  return a.n ? ff_run<FF_PLAIN>(a, f->type, s) : 0;
}

int pylo_b200_sizeof_layers(int what) {
  return what == 0 ? (int)sizeof(pylo_norm) : what == 1 ? (int)sizeof(pylo_distill) : what == 2 ? (int)sizeof(pylo_ffn) : what == 3 ? (int)sizeof(pylo_pad) : -1;
}

int pylo_b200_pad_rows(const pylo_pad* items, int n, void* stream) {
  CHECK_ARG(items && n >= 0 && n <= FF_PADS);
  ff_pads a = {};
  a.n = n;
  for (int k = 0; k < n; ++k) {
    const pylo_pad& p = items[k];
    CHECK_ARG(p.rows >= 0 && p.rows <= (1 << 30) && p.cols >= 0 && p.ld >= p.cols && p.ld <= (1 << 25) && p.ld % 8 == 0 && (p.rows == 0 || (p.src && p.dst)) &&
              ((uintptr_t)p.dst & 15) == 0 && ((uintptr_t)p.src & 1) == 0);
    a.p[k] = p;
    a.first[k + 1] = a.first[k] + p.rows * (p.ld / 8);
  }
  const long long ctas = (a.first[n] + NT - 1) / NT, most = (long long)sm_count() * 16;
  if (ctas) launch(k_ffn_pad, (int)(ctas < most ? ctas : most), NT, 0, (cudaStream_t)stream, a);
  return launch_status();
}

}  // extern "C"
