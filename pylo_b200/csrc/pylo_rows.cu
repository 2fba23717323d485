// Operators on the rows of a matrix that a model's training step needs beside its optimizer: layer norm with its gradients, and the
// loss of a distillation from a teacher's largest logits with its gradient.
//
// Both read and write whole rows once and compute a few operations per element: the memory's bandwidth bounds them, and a small call
// the latency of its launches.  A row belongs to a warp where it is short, else to a CTA; the CTAs are as many as run at once and go
// from row to row.  Everything is computed in fp32 from the elements' own type and rounded once, where it is stored.
#include <cuda_bf16.h>
#include <limits.h>

#include "pylo_common.cuh"
#include "pylo_launch.cuh"

// ------------------------------------------------------------------------------------------------
// elements of a row
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ float rw_float(float v) { return v; }
__device__ __forceinline__ float rw_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float rw_float(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T rw_to(float v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}
template <class T>
constexpr int RW_VEC = 16 / (int)sizeof(T);   // elements of 16 bytes

// N neighbouring elements: 16 bytes, or one element
template <class T, int N>
struct RwPiece {
  static_assert(N * sizeof(T) == 16, "16 bytes or one element");
  uint32_t w[4];   // two 16-bit elements in each, or one of 32
  __device__ __forceinline__ void load(const T* p) {   // read once: not kept in the L1 cache
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
  }
  __device__ __forceinline__ void from_shared(uint32_t p) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(p) : "memory");
  }
  __device__ __forceinline__ void store(T* p) const { __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3])); }
  __device__ __forceinline__ float at(int j) const {
    if constexpr (std::is_same_v<T, float>) return __uint_as_float(w[j]);
    else if constexpr (std::is_same_v<T, __half>) {
      const __half2 h = *reinterpret_cast<const __half2*>(&w[j >> 1]);
      return j & 1 ? __high2float(h) : __low2float(h);
    } else return __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
  }
  __device__ __forceinline__ T one(int j) const {
    if constexpr (std::is_same_v<T, float>) return __uint_as_float(w[j]);
    else {
      const uint16_t h = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
      return *reinterpret_cast<const T*>(&h);
    }
  }
  __device__ __forceinline__ uint64_t two(int j) const {   // elements j, j + 1
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(at(j)), "f"(at(j + 1)));
    return r;
  }
  template <class F>
  __device__ __forceinline__ void make(F&& f) {   // element j from f(j), rounded
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, float>) w[i] = __float_as_uint(f(i));
      else if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(f(2 * i), f(2 * i + 1));
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f(2 * i), f(2 * i + 1));
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
};
template <class T>
struct RwPiece<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }   // (__ldg of 16-bit types is assembly that the compiler may move out of a branch, to where p is not valid)
  __device__ __forceinline__ void store(T* p) const { *p = v; }
  __device__ __forceinline__ float at(int) const { return rw_float(v); }
  template <class F>
  __device__ __forceinline__ void make(F&& f) { v = rw_to<T>(f(0)); }
};

// the largest of a piece's elements that are numbers
template <class T, int N>
__device__ __forceinline__ float rw_most(const RwPiece<T, N>& v) {
  if constexpr (std::is_same_v<T, float>) return fmaxf(fmaxf(v.at(0), v.at(1)), fmaxf(v.at(2), v.at(3)));
  else {   // two at a time
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const T2* const q = reinterpret_cast<const T2*>(v.w);
    const T2 most = __hmax2(__hmax2(q[0], q[1]), __hmax2(q[2], q[3]));
    return fmaxf(rw_float(most.x), rw_float(most.y));
  }
}

__device__ __forceinline__ void rw_cluster_sync() {   // all threads of the cluster's CTAs; orders accesses to all memory
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of another CTA's copy of a shared variable
__device__ __forceinline__ uint32_t rw_at_rank(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
  return a;
}
// two fp32 values, and operations on two at once
__device__ __forceinline__ uint64_t rw_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void rw_unpair(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ float rw_both(uint64_t r) {   // their sum
  float a, b;
  rw_unpair(r, a, b);
  return a + b;
}
__device__ __forceinline__ uint64_t rw_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t rw_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t rw_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float rw_warp_sum(float v) {   // in every lane, in an order of its own
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float rw_warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
// all copies of this thread but the last n groups have arrived
__device__ __forceinline__ void rw_arrived(int n) {
  switch (n) {
#define RW_CASE(N) case N: asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); break;
    RW_CASE(1) RW_CASE(2) RW_CASE(3) RW_CASE(4) RW_CASE(5) RW_CASE(6) RW_CASE(7) RW_CASE(8) RW_CASE(9) RW_CASE(10) RW_CASE(11)
    RW_CASE(12) RW_CASE(13) RW_CASE(14) RW_CASE(15) RW_CASE(16) RW_CASE(17) RW_CASE(18) RW_CASE(19) RW_CASE(20) RW_CASE(21) RW_CASE(22) RW_CASE(23)
#undef RW_CASE
    default: asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
}
__device__ __forceinline__ void rw_copy(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void rw_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// ------------------------------------------------------------------------------------------------
// Layer norm.  m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), xh = (x - m) r:
//   y = xh w + b;   dx = r (q - mean q - xh mean(q xh)) with q = dy w;   dw = sum over rows dy xh, db = sum over rows dy
//
// A row is read once and stays in registers, 16 or 32 elements of each thread, so that the variance is that of the differences from the mean (a
// sum of squares less the mean's would lose what rows far off centre have).  A row is a warp's, a CTA's, or that of a cluster of two
// CTAs; the next one is on its way while one is worked on.  The weights stay in registers from row to row, the sums of their
// gradients too; those leave as one partial sum per CTA, and a second kernel adds them up in a fixed order.
//
// 32768 x 4096 on a B200: bf16 forward 101 us (5.3 TB/s), backward with the columns' sums 175 (4.6 TB/s), whose bound is as much the issue slots as the memory; fp16 93 and
// 183, fp32 177 (6.1 TB/s) and 286.  A row's elements one at a time, 12289 x 1001 fp16: 22 and 32.
// ------------------------------------------------------------------------------------------------
#define LN_WARP_THREADS 128   // of a CTA whose warps have a row each
#define LN_WARPS (LN_WARP_THREADS / 32)
#define LN_MOST 16384         // elements of a row
// CTAs of so many threads on an SM, with E elements per thread: 64 to 168 registers.  At 128, 32 elements of a warp's row spill (forward 24 to 40 bytes of stack, backward 72, fp16
// weights 176), 16 of a larger CTA's that come one at a time up to 56.
__host__ __device__ constexpr int ln_ctas(int threads, int e, bool backward, bool ring) {
  return threads > 128 ? 512 / threads : e <= 8 ? backward ? 6 : 8 : backward && !ring ? 3 : 4;
}
#define LN_DEPTH 3   // rows of a thread's ring: one that is worked on, two on their way
struct LnArgs {
  const void *x, *dy, *weight, *bias;
  void *y;               // or dx, or NULL
  float *mean, *rstd;    // written forward (or NULL), read backward
  float* part;           // [CTAs that begin rows][2][width]: sums for dw, db; or NULL
  long long rows, x_stride, dy_stride;
  int width;
  float eps;
};

// a vector's elements that are a thread's, NV pieces of VN, `gap` elements from one to the next
template <class W, int VN, int NV>
struct LnVector {
  static constexpr int WN = VN == 1 ? 1 : RW_VEC<W>, PER = VN / WN;
  RwPiece<W, WN> p[NV * PER];
  __device__ __forceinline__ void load(const W* v, int first, int gap, int width) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        if (first + i * gap < width) p[i * PER + k].load(v + first + i * gap + k * WN);
        else p[i * PER + k].make([](int) { return 0.f; });
      }
  }
  __device__ __forceinline__ uint64_t two(int k) const {   // elements 2k, 2k + 1 of the thread's
    if constexpr (VN == 1) return rw_pair(p[2 * k].at(0), p[2 * k + 1].at(0));
    else return p[2 * k / WN].two(2 * k % WN);
  }
};
template <class T, int VN, int NV>
__device__ __forceinline__ uint64_t ln_two(const RwPiece<T, VN> (&v)[NV], int k) {
  if constexpr (VN == 1) return rw_pair(v[2 * k].at(0), v[2 * k + 1].at(0));
  else return v[2 * k / VN].two(2 * k % VN);
}

// Two sums over the threads of a row, in every one of them, in an order of its own.  buf: what the warps leave for one another; two take turns.
template <bool BLOCK>
__device__ __forceinline__ float2 ln_sums(float a, float b, float2* buf, uint32_t rank, uint32_t share) {
  a = rw_warp_sum(a);
  b = rw_warp_sum(b);
  if constexpr (BLOCK) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (share == 1) {
      if (lane == 0) buf[warp] = make_float2(a, b);
      __syncthreads();
    } else {
      if (lane < (int)share)
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(rw_at_rank(&buf[rank * warps + warp], lane)), "f"(a), "f"(b) : "memory");
      rw_cluster_sync();
    }
    const float2 q = lane < (int)share * warps ? buf[lane] : make_float2(0.f, 0.f);
    a = rw_warp_sum(q.x);
    b = rw_warp_sum(q.y);
  }
  return make_float2(a, b);
}

// Which rows and which elements of them are a thread's
template <bool BLOCK, int VN, int NV>
struct LnPlace {
  uint32_t rank = 0, share = 1;
  int first, gap;          // elements first + i gap + j of a row
  long long row, step;
  __device__ __forceinline__ LnPlace() {
    if constexpr (BLOCK) {
      asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
      asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(share));
      gap = blockDim.x * VN;
      first = rank * gap * NV + threadIdx.x * VN;
      row = blockIdx.x / share;
      step = gridDim.x / share;
    } else {
      gap = 32 * VN;
      first = (threadIdx.x & 31) * VN;
      row = (long long)blockIdx.x * LN_WARPS + (threadIdx.x >> 5);
      step = (long long)gridDim.x * LN_WARPS;
    }
  }
  __device__ __forceinline__ bool in(int e, int width) const { return first + e / VN * gap < width; }   // whether the thread's element e is one of the row's
  template <class T, class F>
  __device__ __forceinline__ void store(T* out, int width, F&& f) const {   // elements 2k, 2k + 1 from f(k)
    float keep = 0.f;   // the second of two, where pieces have one element
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float x[VN];
      if constexpr (VN == 1) {
        if (i & 1) x[0] = keep;
        else rw_unpair(f(i / 2), x[0], keep);
      } else
        for (int j = 0; j < VN; j += 2) rw_unpair(f((i * VN + j) / 2), x[j], x[j + 1]);
      if (first + i * gap < width) {
        RwPiece<T, VN> o;
        o.make([&](int j) { return x[j]; });
        o.store(out + first + i * gap);
      }
    }
  }
};

template <class T, class W, int VN, int E, int MOST>
__global__ void __launch_bounds__(MOST ? MOST : LN_WARP_THREADS, ln_ctas(MOST, E, false, false)) k_layer_norm(const LnArgs a) {
  constexpr bool BLOCK = MOST > 0;   // a row is a CTA's, of so many threads at most
  constexpr int NV = E / VN;
  __shared__ float2 s_buf[2][32];   // a part of the sums per lane
  const LnPlace<BLOCK, VN, NV> at;
  const int width = a.width;
  if (at.share > 1) rw_cluster_sync();   // the others are running
  pdl_begin();
  const float inv = 1.0f / (float)width;
  const T* const x = (const T*)a.x;
  LnVector<W, VN, NV> weight, bias;
  if (a.weight) weight.load((const W*)a.weight, at.first, at.gap, width);
  if (a.bias) bias.load((const W*)a.bias, at.first, at.gap, width);
  RwPiece<T, VN> v[NV];
  auto fetch = [&](long long r) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (at.first + i * at.gap < width && r < a.rows) v[i].load(x + r * a.x_stride + at.first + i * at.gap);
      else v[i].make([](int) { return 0.f; });
  };
  fetch(at.row);
  for (long long row = at.row; row < a.rows; row += at.step) {
    // elements two by two: of a piece, or (VN = 1) of two pieces
    uint64_t f[E / 2], sum = rw_pair(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < E / 2; ++k) sum = rw_add2(sum, f[k] = ln_two<T, VN, NV>(v, k));
    fetch(row + at.step);
    const float mean = ln_sums<BLOCK>(rw_both(sum), 0.f, s_buf[0], at.rank, at.share).x * inv;
    const uint64_t off = rw_pair(-mean, -mean);
    uint64_t sq = rw_pair(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
      if (VN > 1 && !at.in(2 * k, width)) continue;
      f[k] = rw_add2(f[k], off);
      uint64_t d = f[k];
      if constexpr (VN == 1) {   // what lies behind the row does not differ from the mean
        float lo, hi;
        rw_unpair(d, lo, hi);
        d = rw_pair(at.in(2 * k, width) ? lo : 0.f, at.in(2 * k + 1, width) ? hi : 0.f);
      }
      sq = rw_fma2(d, d, sq);
    }
    const float rstd = 1.0f / sqrtf(fmaf(ln_sums<BLOCK>(rw_both(sq), 0.f, s_buf[1], at.rank, at.share).x, inv, a.eps));
    if (at.first == 0 && a.mean) { a.mean[row] = mean; a.rstd[row] = rstd; }
    const uint64_t by = rw_pair(rstd, rstd);
    at.store((T*)a.y + row * width, width, [&](int k) {
      uint64_t q = rw_mul2(f[k], by);
      if (a.weight) q = rw_mul2(q, weight.two(k));
      return a.bias ? rw_add2(q, bias.two(k)) : q;
    });
  }
}

template <class T, class W, int VN, int E, int MOST>
__global__ void __launch_bounds__(MOST ? MOST : LN_WARP_THREADS, ln_ctas(MOST, E, true, VN > 1)) k_layer_norm_backward(const LnArgs a) {
  constexpr bool BLOCK = MOST > 0, RING = VN > 1;   // rows by asynchronous copies through the thread's own part of shared memory, or through registers
  constexpr int NV = E / VN;
  __shared__ float2 s_buf[2][32];   // a part of the sums per lane
  __shared__ float s_cols[BLOCK ? 1 : 2 * 32 * E];
  extern __shared__ __align__(16) unsigned char ln_raw[];
  const LnPlace<BLOCK, VN, NV> at;
  const int width = a.width;
  if (at.share > 1) rw_cluster_sync();   // the others are running
  pdl_begin();
  const float inv = 1.0f / (float)width;
  LnVector<W, VN, NV> weight;
  if (a.weight) weight.load((const W*)a.weight, at.first, at.gap, width);
  uint64_t dw2[E / 2], db2[E / 2];
#pragma unroll
  for (int k = 0; k < E / 2; ++k) dw2[k] = db2[k] = rw_pair(0.f, 0.f);
  // What lies behind a row has a gradient of zero.
  const uint32_t piece = blockDim.x * 16, ring = smem_addr(ln_raw) + 16 * threadIdx.x;
  constexpr int KEPT = RING ? 1 : NV;
  RwPiece<T, VN> nx[KEPT], nd[KEPT], vx[KEPT], vd[KEPT];
  if constexpr (RING) {
    for (int i = 0; i < LN_DEPTH * 2 * NV; ++i) asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(ring + i * piece), "r"(0) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) { nx[i].make([](int) { return 0.f; }); nd[i].make([](int) { return 0.f; }); }
  }
  uint32_t in = 0, out = 0;   // the ring's places, as offsets
  auto fetch = [&](long long r) {
    if (r < a.rows) {
      const T* const x = (const T*)a.x + r * a.x_stride + at.first;
      const T* const dy = (const T*)a.dy + r * a.dy_stride + at.first;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (at.first + i * at.gap < width) {
          if constexpr (RING) {
            rw_copy(ring + in + 2 * i * piece, x + i * at.gap);
            rw_copy(ring + in + (2 * i + 1) * piece, dy + i * at.gap);
          } else {
            nx[i].load(x + i * at.gap);
            nd[i].load(dy + i * at.gap);
          }
        }
    }
    if constexpr (RING) {
      rw_commit();
      in = in == (LN_DEPTH - 1) * 2 * NV * piece ? 0 : in + 2 * NV * piece;
    }
  };
  // elements 2k, 2k + 1 of x and dy of the row that is worked on, asked for in order
  RwPiece<T, RING ? VN : RW_VEC<T>> px, pd;
  auto taken = [&](int k, uint64_t& x, uint64_t& d) {
    if constexpr (RING) {
      if (2 * k % VN == 0) {
        px.from_shared(ring + out + 2 * (2 * k / VN) * piece);
        pd.from_shared(ring + out + (2 * (2 * k / VN) + 1) * piece);
      }
      x = px.two(2 * k % VN);
      d = pd.two(2 * k % VN);
    } else {
      x = ln_two<T, VN, KEPT>(vx, k);
      d = ln_two<T, VN, KEPT>(vd, k);
    }
  };
  float next_mean = 0.f, next_rstd = 0.f;
  auto stats = [&](long long r) {
    if (r < a.rows) { next_mean = a.mean[r]; next_rstd = a.rstd[r]; }
  };
  stats(at.row);
  if constexpr (RING) {
#pragma unroll
    for (int d = 0; d < LN_DEPTH - 1; ++d) fetch(at.row + d * at.step);
  } else fetch(at.row);
  int flip = 0;
#pragma unroll 1
  for (long long row = at.row; row < a.rows; row += at.step, flip ^= 1) {
    // xh = (x - mean) rstd, as the forward pass has it: x rstd - mean rstd in one operation would add a rounding of mean rstd, which may be beyond fp32
    const uint64_t r2 = rw_pair(next_rstd, next_rstd), off = rw_pair(-next_mean, -next_mean);
    const float rstd = next_rstd;
    if constexpr (RING) {
      fetch(row + (LN_DEPTH - 1) * at.step);
      rw_arrived(LN_DEPTH - 1);
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) { vx[i] = nx[i]; vd[i] = nd[i]; }
      fetch(row + at.step);
    }
    stats(row + at.step);
    uint64_t t1 = rw_pair(0.f, 0.f), t2 = t1;
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
      uint64_t x, d;
      taken(k, x, d);
      const uint64_t from = rw_add2(x, off), xh = rw_mul2(from, r2), q = a.weight ? rw_mul2(d, weight.two(k)) : d;
      dw2[k] = rw_fma2(d, xh, dw2[k]);
      db2[k] = rw_add2(d, db2[k]);
      t1 = rw_add2(t1, q);
      t2 = rw_fma2(q, from, t2);   // (not of xh: what lies behind the row is 0 times a difference, and xh may be infinite there)
    }
    if (a.y) {
      const float2 sums = ln_sums<BLOCK>(rw_both(t1), rw_both(t2), s_buf[flip], at.rank, at.share);
      // rstd (q - s1 - (x - mean) s2); of a row whose variance is beyond fp32 xh is 0, whatever the differences add up to
      const float by = rstd != 0.f ? -sums.y * rstd * inv * rstd : 0.f;
      const uint64_t s1 = rw_pair(-sums.x * inv * rstd, -sums.x * inv * rstd), s2 = rw_pair(by, by);
      at.store((T*)a.y + row * width, width, [&](int k) {
        uint64_t x, d;
        taken(k, x, d);
        const uint64_t q = a.weight ? rw_mul2(d, weight.two(k)) : d;
        return rw_fma2(rw_fma2(rw_add2(x, off), s2, q), r2, s1);
      });
    }
    if constexpr (RING) out = out == (LN_DEPTH - 1) * 2 * NV * piece ? 0 : out + 2 * NV * piece;
  }
  if constexpr (RING) asm volatile("cp.async.wait_all;" ::: "memory");
  float dw[E], db[E];
#pragma unroll
  for (int k = 0; k < E / 2; ++k) {
    rw_unpair(dw2[k], dw[2 * k], dw[2 * k + 1]);
    rw_unpair(db2[k], db[2 * k], db[2 * k + 1]);
  }
  if (a.part) {
    float* const part = a.part + (long long)(BLOCK ? blockIdx.x / at.share : blockIdx.x) * 2 * width;
    if constexpr (BLOCK) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VN; ++j) {
          const int c = at.first + i * at.gap + j;
          if (c < width) { part[c] = dw[i * VN + j]; part[width + c] = db[i * VN + j]; }
        }
    } else {
      // the warps' sums, one warp after the other
      for (int w = 0; w < LN_WARPS; ++w) {
        if ((int)(threadIdx.x >> 5) == w)
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VN; ++j) {
              const int c = at.first + i * at.gap + j;
              s_cols[c] = w ? s_cols[c] + dw[i * VN + j] : dw[i * VN + j];
              s_cols[32 * E + c] = w ? s_cols[32 * E + c] + db[i * VN + j] : db[i * VN + j];
            }
        __syncthreads();
      }
      for (int c = threadIdx.x; c < width; c += LN_WARP_THREADS) { part[c] = s_cols[c]; part[width + c] = s_cols[32 * E + c]; }
    }
  }
}

// The partial sums of 32 columns by a CTA: sixteen rows of threads, each adding up every sixteenth partial, then those.
#define LN_COLUMN_GROUPS 16
template <class W>
__global__ void __launch_bounds__(32 * LN_COLUMN_GROUPS) k_layer_norm_columns(const float* __restrict__ part, int n, int width, W* dweight, W* dbias) {
  pdl_begin();
  __shared__ float s[LN_COLUMN_GROUPS][33];
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  W* const out = blockIdx.y ? dbias : dweight;
  if (out == nullptr) return;
  const float* p = part + (blockIdx.y ? width : 0) + c;
  float sum = 0.f;
  if (c < width)
#pragma unroll 8
    for (int i = g; i < n; i += LN_COLUMN_GROUPS) sum += p[(long long)i * 2 * width];
  s[g][lane] = sum;
  __syncthreads();
  if (g == 0 && c < width) {
#pragma unroll
    for (int i = 1; i < LN_COLUMN_GROUPS; ++i) sum += s[i][lane];
    out[c] = rw_to<W>(sum);
  }
}

// A call's form: elements of a thread, the most threads of a CTA that the kernel is made for (0: a warp per row), its threads, CTAs that share a row,
// groups of CTAs that begin with different rows
struct LnForm { int elems, most, threads, share, groups; };
static LnForm ln_form(long long rows, int width, bool wide, bool backward, bool ring) {   // wide: 16-bit elements by 16 bytes
  const int many = wide ? 32 : 16, few = wide ? 8 : 4;
  LnForm f = {many, 0, LN_WARP_THREADS, 1, 0};
  long long n = (rows + LN_WARPS - 1) / LN_WARPS;
  if (width <= 32 * few) f.elems = few;
  else if (wide && width <= 512) f.elems = 16;
  else if (width > 32 * many) {
    n = rows;
    f.threads = (width + 32 * many - 1) / (32 * many) * 32;
    while (f.threads > 512) f.threads = (f.threads / 2 + 31) / 32 * 32, f.share *= 2;
    f.most = f.threads <= 128 ? 128 : f.threads <= 256 ? 256 : 512;
  }
  long long at_once = (long long)sm_count() * ln_ctas(f.most, f.elems, backward, ring) / f.share;
  if (f.most && f.threads < 128) at_once = at_once * 128 / f.threads;
  f.groups = (int)(n < at_once ? n : at_once);
  return f;
}
template <class T, class W, int VN>
static int ln_launch(const LnArgs& a, bool backward, cudaStream_t s) {
  constexpr bool WIDE = sizeof(T) == 2 && VN > 1;
  constexpr int MANY = WIDE ? 32 : 16, FEW = WIDE ? 8 : 4;
  const LnForm f = ln_form(a.rows, a.width, WIDE, backward, VN > 1);
#define LN_GO(E, MOST)                                                                                                                   \
  if (!backward) launch_clusters(k_layer_norm<T, W, VN, E, MOST>, f.groups * f.share, f.threads, MOST ? f.share : 0, 0, s, a);           \
  else {                                                                                                                                 \
    const int smem = VN > 1 ? LN_DEPTH * 2 * (E / VN) * 16 * f.threads : 0;                                                              \
    static bool configured[PYLO_MAX_DEVICES] = {};                                                                                       \
    if (int rc = VN > 1 ? allow_dynamic_smem(k_layer_norm_backward<T, W, VN, E, MOST>, LN_DEPTH * 2 * (E / VN) * 16 * (MOST ? MOST : LN_WARP_THREADS), configured) : 0) return rc; \
    if (VN > 1 && f.groups > sm_count()) t_plain_next = true;   /* as many CTAs as an SM is to hold need more than a predecessor leaves of it */ \
    launch_clusters(k_layer_norm_backward<T, W, VN, E, MOST>, f.groups * f.share, f.threads, MOST ? f.share : 0, smem, s, a);            \
  }                                                                                                                                      \
  return 0;
  if (f.most == 128) { LN_GO(MANY, 128) }
  if (f.most == 256) { LN_GO(MANY, 256) }
  if (f.most == 512) { LN_GO(MANY, 512) }
  if (f.elems == FEW) { LN_GO(FEW, 0) }
  if constexpr (WIDE)
    if (f.elems == 16) { LN_GO(16, 0) }
  LN_GO(MANY, 0)
#undef LN_GO
}
// 16 bytes at a time where every row begins on their boundary (how far the next one would be from a single row says nothing)
static bool ln_aligned(const pylo_norm* n, bool backward) {
  const int vec = n->type == PYLO_FP32 ? 4 : 8;
  uintptr_t p = (uintptr_t)n->x | (uintptr_t)n->weight | (backward ? (uintptr_t)n->dy | (uintptr_t)n->dx : (uintptr_t)n->y | (uintptr_t)n->bias);
  return p % 16 == 0 && (n->width | (n->rows > 1 ? n->x_stride | (backward ? n->dy_stride : 0) : 0)) % vec == 0;
}
template <class T, class W>
static int ln_run(const LnArgs& a, bool aligned, bool backward, cudaStream_t s) {
  return aligned ? ln_launch<T, W, RW_VEC<T>>(a, backward, s) : ln_launch<T, W, 1>(a, backward, s);
}
static int ln_any(const LnArgs& a, int type, int weight_type, bool aligned, bool backward, cudaStream_t s) {
  int rc = -1;
  if (type == PYLO_FP32 && weight_type == PYLO_FP32) rc = ln_run<float, float>(a, aligned, backward, s);
  else if (type == PYLO_BF16 && weight_type == PYLO_BF16) rc = ln_run<__nv_bfloat16, __nv_bfloat16>(a, aligned, backward, s);
  else if (type == PYLO_FP16 && weight_type == PYLO_FP16) rc = ln_run<__half, __half>(a, aligned, backward, s);
  else if (type == PYLO_BF16 && weight_type == PYLO_FP32) rc = ln_run<__nv_bfloat16, float>(a, aligned, backward, s);
  else if (type == PYLO_FP16 && weight_type == PYLO_FP32) rc = ln_run<__half, float>(a, aligned, backward, s);
  return rc ? rc : launch_status();
}
static size_t rw_bytes(int type) { return type == PYLO_FP32 ? 4 : 2; }
// no element lies at another address: pointers that may be NULL
template <class... P>
static bool rw_on(size_t bytes, P... p) { return (((uintptr_t)p | ...) & (bytes - 1)) == 0; }
static bool rw_type(int type) { return type == PYLO_FP32 || type == PYLO_BF16 || type == PYLO_FP16; }

// ------------------------------------------------------------------------------------------------
// Distillation from a teacher's K largest logits t at the ids i, of a student's logits s over V classes, at temperature T:
//   p = softmax(t / T) over the K entries,  q = softmax(s / T) over the V classes
//   loss of a row = T^2 sum_k p_k (log p_k - log q_{i_k});   its gradient: T (q_j - sum of the p_k with i_k = j)
// An id outside of [0, V) is padding, whatever the teacher's logit beside it is; a row whose entries are all padding or -inf has no
// teacher and the weight zero.  Rows of weight zero are not read, whatever they hold: their loss and gradient are zero.
//
// One pass over a row with a running maximum and sum per thread; powers of two of differences from the maximum, scaled by log2(e) / T (not of scaled logits
// less the scaled maximum in one operation: of masks of -1e30, or far off centre, what that rounds off is a power of its own), of the teacher's logits as of the
// student's.  The gradient reads the row again (in the call that makes both, out of the SMs' shared memory, where a long row stays between the passes, or
// a short one through the caches).  The K columns with a teacher's entry are written a second time, behind a barrier, with what their entries add up to.
// Exponentials are ex2.approx: 2 ulp each, beside exponents that are rounded to 2^-24 of their size anyway.
// ------------------------------------------------------------------------------------------------
#define DT_MOST_K 1024
#define DT_WARP_VOCAB 1024     // classes up to which a row is a warp's
#define DT_WARP_THREADS 128
#define DT_MOST_CTAS 8         // of an SM, in whatever form
#define DT_LOG2E 1.4426950408889634
#define DT_LN2 0.6931471805599453f
#define DT_LOWEST (-3.402823466e38f)   // a maximum of nothing
enum { DT_LOSS = 1, DT_GRAD = 2 };

struct DtArgs {
  const void *logits, *teacher, *ids;
  const float* weights;     // [rows] or NULL
  float* row_loss;          // [rows]: weight * loss, or NULL
  float2* stat;             // [rows]: maximum, 1 / sum of powers; written with the loss, read for a gradient alone; or NULL
  double2* part;            // [CTAs or clusters]: sums of weight * loss, of weights
  void* grad;               // [rows][vocab]
  const float* upstream;    // of the loss: a scalar, or (per_row) [rows]; NULL: 1
  const float* inv;         // scalar: 1 / sum of the weights; NULL: 1, or
  const double* weight_sums;// [n_sums]: its parts
  // of long rows, what their teachers come to (k_distill_teachers)
  float4* teachers;         // [rows]: weight (0 where no entry counts), sum of p (log2 p - scaled difference of logit and r), sum of p, r
  int2* columns;            // [rows][top]: a class that an entry gives (the first of several; else -1), the bits of its probability; or NULL
  long long rows, stride;
  int vocab, top, teacher_type, wide_ids, n_sums, per_row;
  float c, temperature, scale;   // log2(e) / T, T, another factor of the gradient
};

__device__ __forceinline__ float dt_any(const void* p, int type, long long i) {
  return type == PYLO_FP32 ? ((const float*)p)[i] : type == PYLO_BF16 ? rw_float(((const __nv_bfloat16*)p)[i]) : rw_float(((const __half*)p)[i]);
}
// a teacher's entry: its id, or -1
__device__ __forceinline__ int dt_id(const DtArgs& a, long long i) {
  const long long id = a.wide_ids ? ((const long long*)a.ids)[i] : ((const int*)a.ids)[i];
  return id >= 0 && id < a.vocab ? (int)id : -1;
}

// 2^x; what is below 2^-126 is 0
__device__ __forceinline__ float dt_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// What the gradient of every row is multiplied by
__device__ __forceinline__ float dt_factor(const DtArgs& a) {
  float factor = a.scale * a.temperature;
  if (a.weight_sums) {   // in the same order in every CTA
    double w = 0.0;
    for (int i = 0; i < a.n_sums; ++i) w += a.weight_sums[i];
    factor = w != 0.0 ? (float)(factor / w) : 0.f;
  } else if (a.inv) factor *= *a.inv;
  if (a.upstream && !a.per_row) factor *= *a.upstream;
  return factor;
}
// A teacher's entry: its class, the probability and its logarithm to base 2, and what its column takes: of several entries of one class the first
// takes what all of them add up to, in their order.  id: ~class for those that leave the column alone; padding is DT_PADDING with p = 0.
#define DT_PADDING INT_MIN
struct DtEntry { int id; float p, lp, column; };
static __host__ __device__ __forceinline__ int dt_slots(int top) {   // of the table of classes: a power of two, half full at most
  int n = 64;
  while (n < 2 * top) n *= 2;
  return n;
}
// A warp's next 128 entries of a row, as they are in memory: asked for together, and ahead of their use
struct DtPeek { int id[4]; float t[4]; };
__device__ __forceinline__ DtPeek dt_peek(const DtArgs& a, long long row, int first) {
  DtPeek p;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = first + 32 * i + (threadIdx.x & 31);
    p.id[i] = -1;
    p.t[i] = 0.f;
    if (k < a.top && row < a.rows) {
      p.id[i] = dt_id(a, row * a.top + k);
      p.t[i] = dt_any(a.teacher, a.teacher_type, row * a.top + k);
    }
  }
  return p;
}
// A row's K entries, by a warp; slots: dt_slots(K) words.  False if there are none
__device__ __forceinline__ bool dt_teacher(const DtArgs& a, long long row, DtPeek peek, DtEntry* e, int* slots) {
  const int lane = threadIdx.x & 31, K = a.top, n = dt_slots(K);
  float most = -CUDART_INF_F, sum = 0.f;
  bool any = false;
  for (int i = lane; i < n; i += 32) slots[i] = -1;
  __syncwarp();
  bool twice = false;   // a class that has an entry already
  for (int first = 0; first < K; first += 128) {
    if (first) peek = dt_peek(a, row, first);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = first + 32 * i + lane, id = peek.id[i];
      if (k >= K) break;
      const float logit = id >= 0 ? peek.t[i] : -CUDART_INF_F;
      e[k].id = id >= 0 ? id : DT_PADDING;
      e[k].lp = logit;
      most = fmaxf(most, logit);
      any |= !(logit == -CUDART_INF_F);
      if (id >= 0)
        for (unsigned at = (unsigned)id * 2654435761u;; ++at) {   // ends: half of the slots stay free
          const int found = atomicCAS(&slots[(at ^ at >> 16) & (n - 1)], -1, id);
          twice |= found == id;
          if (found == -1 || found == id) break;
        }
    }
  }
  if (!__any_sync(0xffffffffu, any)) return false;
  twice = __any_sync(0xffffffffu, twice);
  most = rw_warp_max(most);
  for (int k = lane; k < K; k += 32) sum += dt_exp2((e[k].lp - most) * a.c);   // (the difference first, as of the student's)
  const float log_sum = log2f(rw_warp_sum(sum));
  for (int k = lane; k < K; k += 32) {
    const float lp = fmaf(e[k].lp - most, a.c, -log_sum), p = e[k].id == DT_PADDING ? 0.f : dt_exp2(lp);   // (beside a teacher's NaN or infinity lp is NaN)
    e[k].lp = lp;
    e[k].p = p;
    e[k].column = p;
  }
  __syncwarp();
  if (twice) {
    for (int k = lane; k < K; k += 32) {
      const int id = e[k].id;
      float all = 0.f;
      for (int j = 0; j < K; ++j)
        if (e[j].id == id || e[j].id == ~id) {   // (the other lanes are at work on them)
          if (j < k && id >= 0) { e[k].id = ~id; break; }
          all += e[j].p;
        }
      e[k].column = all;
    }
    __syncwarp();
  }
  return true;
}
// The loss of a row to base 2, without the student's sum: sum of p (log p - s) with logits relative to the largest of them, by a warp.  Relative to that,
// as to the row's maximum (which long rows do not know yet), the terms in s have one sign, so that no large ones cancel: not of logits far off centre, nor
// where the student masks a class that the teacher gives next to nothing.
struct DtCross { float cross, sum, near; };   // sum: of p; near: the largest logit of an entry that counts
template <class T>
__device__ __forceinline__ DtCross dt_cross(const DtArgs& a, const T* s, const DtEntry* e) {
  DtCross r = {0.f, 0.f, DT_LOWEST};
  auto raise = [&](float to) {
    if (to > r.near && r.sum != 0.f) r.cross = fmaf(r.sum * (to - r.near), a.c, r.cross);
    r.near = to;
  };
  for (int first = threadIdx.x & 31; first < a.top; first += 128) {
    DtEntry q[4];
    float v[4];
    bool counts[4];   // padding has no class to read, whatever its p
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      q[i] = {DT_PADDING, 0.f, 0.f, 0.f};
      v[i] = 0.f;
      if (first + 32 * i < a.top) q[i] = e[first + 32 * i];
      counts[i] = q[i].id != DT_PADDING && !(q[i].p == 0.f);
      if (counts[i]) v[i] = rw_float(s[q[i].id < 0 ? ~q[i].id : q[i].id]);   // all four on their way together
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (counts[i]) {
        raise(fmaxf(r.near, v[i]));
        r.cross = fmaf(q[i].p, fmaf(v[i] - r.near, -a.c, q[i].lp), r.cross);
        r.sum += q[i].p;
      }
  }
  raise(rw_warp_max(r.near));
  r.cross = rw_warp_sum(r.cross);
  r.sum = rw_warp_sum(r.sum);
  return r;
}
// The column of a teacher's entry, once more
template <class T>
__device__ __forceinline__ void dt_column(T* grad, int id, float p, float logit, float f, float total, float m, float c) {
  grad[id] = rw_to<T>(f * (total * dt_exp2((logit - m) * c) - p));
}

// Where a row's 16-byte pieces lie, and the element before or behind them that is thread t's
template <class T>
struct DtRow {
  const T* s;
  int head, pieces, edge;   // edge: -1 for none
  __device__ __forceinline__ DtRow(const T* s_, int V, int t) : s(s_) {
    constexpr int VN = RW_VEC<T>;
    head = min(V, (int)((16 - ((uintptr_t)s & 15)) & 15) / (int)sizeof(T));
    pieces = (V - head) / VN;
    const int tail = head + pieces * VN;
    edge = t < head ? t : tail + t - head < V ? tail + t - head : -1;
    static_assert(2 * (VN - 1) <= 32, "a thread per element outside of the pieces");
  }
};

// Short rows: a warp each.
template <class T, int DO>
__global__ void __launch_bounds__(DT_WARP_THREADS) k_distill_short(const DtArgs a) {
  pdl_begin();
  extern __shared__ __align__(16) unsigned char dt_raw[];
  __shared__ double s_sums[2][DT_WARP_THREADS / 32];
  constexpr int VN = RW_VEC<T>, GROUPS = DT_WARP_THREADS / 32;
  const int t = threadIdx.x & 31, group = threadIdx.x >> 5, V = a.vocab;
  DtEntry* const e = (DtEntry*)dt_raw + group * a.top;
  int* const slots = (int*)((DtEntry*)dt_raw + GROUPS * a.top) + group * dt_slots(a.top);
  const float factor = DO & DT_GRAD ? dt_factor(a) : 0.f;
  double loss_sum = 0.0, weight_sum = 0.0;
  for (long long row = (long long)blockIdx.x * GROUPS + group; row < a.rows; row += (long long)gridDim.x * GROUPS) {
    const float weight = a.weights ? a.weights[row] : 1.0f;
    const bool any = weight != 0.f && dt_teacher(a, row, dt_peek(a, row, 0), e, slots);
    T* const grad = DO & DT_GRAD ? (T*)a.grad + row * V : nullptr;
    if (!any) {
      if constexpr (DO & DT_LOSS) {
        if (t == 0 && a.row_loss) a.row_loss[row] = 0.f;
        if (t == 0 && a.stat) a.stat[row] = make_float2(0.f, 0.f);
      }
      if constexpr (DO & DT_GRAD)
        for (int j = t; j < V; j += 32) grad[j] = rw_to<T>(0.f);
      continue;
    }
    const DtRow<T> r((const T*)a.logits + row * a.stride, V, t);
    const T* const body = r.s + r.head;
    float m = DT_LOWEST, total = 0.f;   // maximum; sum of powers relative to it
    if constexpr (DO & DT_LOSS) {
      auto add = [&](const float (&v)[VN]) {
        float most = v[0];
#pragma unroll
        for (int j = 1; j < VN; ++j) most = fmaxf(most, v[j]);
        const float up = fmaxf(m, most);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < VN; ++j) sum += dt_exp2((v[j] - up) * a.c);
        total = fmaf(total, dt_exp2((m - up) * a.c), sum);
        m = up;
      };
      float f[VN];
      for (int i = t; i < r.pieces; i += 32) {
        RwPiece<T, VN> v;
        v.load(body + (long long)i * VN);
#pragma unroll
        for (int j = 0; j < VN; ++j) f[j] = v.at(j);
        add(f);
      }
      if (r.edge >= 0) {
        f[0] = rw_float(r.s[r.edge]);
#pragma unroll
        for (int j = 1; j < VN; ++j) f[j] = -CUDART_INF_F;
        add(f);
      }
      const float all = rw_warp_max(m);
      total = rw_warp_sum(total * dt_exp2((m - all) * a.c));
      m = all;
      const DtCross of = dt_cross(a, r.s, e);
      if (t == 0) {
        const float loss = weight * a.temperature * a.temperature * DT_LN2 * fmaf(of.sum, (m - of.near) * a.c, of.cross + log2f(total));
        if (a.row_loss) a.row_loss[row] = loss;
        if (a.stat) a.stat[row] = make_float2(m, 1.0f / total);
        loss_sum += loss;
        weight_sum += weight;
      }
      total = 1.0f / total;
    } else {
      const float2 st = a.stat[row];
      m = st.x;
      total = st.y;
    }
    if constexpr (DO & DT_GRAD) {
      const float f = factor * weight * (a.upstream && a.per_row ? a.upstream[row] : 1.0f), g = f * total;
      for (int i = t; i < V; i += 32) grad[i] = rw_to<T>(g * dt_exp2((rw_float(r.s[i]) - m) * a.c));
      __syncwarp();   // behind it, the columns of the teacher's entries are written again
      for (int k = t; k < a.top; k += 32)
        if (e[k].id >= 0) dt_column(grad, e[k].id, e[k].column, rw_float(r.s[e[k].id]), f, total, m, a.c);
    }
    __syncwarp();   // the next row's teacher takes the place of this one's
  }
  if constexpr (DO & DT_LOSS) {
    if (t == 0) { s_sums[0][group] = loss_sum; s_sums[1][group] = weight_sum; }
    __syncthreads();
    if (threadIdx.x == 0) {
      double2 sums = make_double2(0.0, 0.0);
      for (int g = 0; g < GROUPS; ++g) { sums.x += s_sums[0][g]; sums.y += s_sums[1][g]; }
      a.part[blockIdx.x] = sums;
    }
  }
}

// What the teachers of long rows come to, a warp for each row, before the rows themselves: in the kernel that streams through the logits a warp that did
// this beside the stream was what the stream waited for (4096 x 128256 bf16 with 128 entries, loss and gradient: 733 us, 494 without it).
template <class T>
__global__ void __launch_bounds__(DT_WARP_THREADS) k_distill_teachers(const DtArgs a, double* weight_sums) {
  pdl_begin();
  extern __shared__ __align__(16) unsigned char dt_raw[];
  __shared__ double s_sums[DT_WARP_THREADS / 32];
  constexpr int GROUPS = DT_WARP_THREADS / 32;
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
  DtEntry* const e = (DtEntry*)dt_raw + group * a.top;
  int* const slots = (int*)((DtEntry*)dt_raw + GROUPS * a.top) + group * dt_slots(a.top);
  double weight_sum = 0.0;
  const long long first = (long long)blockIdx.x * GROUPS + group, step = (long long)gridDim.x * GROUPS;
  DtPeek peek = dt_peek(a, first, 0);
  for (long long row = first; row < a.rows; row += step) {
    const float weight = a.weights ? a.weights[row] : 1.0f;
    const DtPeek mine = peek;
    peek = dt_peek(a, row + step, 0);
    const bool any = weight != 0.f && dt_teacher(a, row, mine, e, slots);
    if (any) {
      const DtCross of = dt_cross(a, (const T*)a.logits + row * a.stride, e);
      if (a.columns)
        for (int k = lane; k < a.top; k += 32) a.columns[row * a.top + k] = make_int2(e[k].id < 0 ? -1 : e[k].id, __float_as_int(e[k].column));
      if (lane == 0) a.teachers[row] = make_float4(weight, of.cross, of.sum, of.near);
      weight_sum += weight;
    } else if (lane == 0) a.teachers[row] = make_float4(0.f, 0.f, 0.f, 0.f);
    __syncwarp();
  }
  if (lane == 0) s_sums[group] = weight_sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int g = 1; g < GROUPS; ++g) weight_sum += s_sums[g];
    weight_sums[blockIdx.x] = weight_sum;
  }
}

// Long rows: a CTA each, or a cluster's, each CTA with its part of the row.  Each thread has a ring of pieces of 16 bytes of its own in shared memory,
// which it fills by asynchronous copies and alone reads, so that what is on its way takes neither registers nor barriers, and the next row's first pieces
// come behind this row's last.  In the call that makes loss and gradient a row's pieces stay in the ring between the two passes (dt_form sees to it that
// they fit).  What the warps leave for one another lies in two buffers that take turns.
//
// A cluster shares a row where there are too few rows for all CTAs, and where a row would not fit the ring.
//
// 8192 x 50257 bf16 on a B200: this kernel's loss 163 us (5.1 TB/s; issue slots 70 %, exponentials 68 %), gradient alone 303 (5.4 TB/s).  Calls, teachers and totals among
// them: fp16 171 and 312; 4096 x 50257 fp32 149 and 291, both in one 389 (4.2 TB/s).
#define DL_MOST_SHARE 8
#define DL_KEPT 16   // pieces of a row that stay in the ring of 24
__host__ __device__ constexpr int dl_ring(int what) { return what == (DT_LOSS | DT_GRAD) ? 24 : 16; }
__host__ __device__ constexpr int dl_ctas(int stream, int what) { return 768 * 16 / dl_ring(what) / stream; }   // of an SM: 192 KB of rings
template <class T, int DO, int STREAM>
__global__ void __launch_bounds__(STREAM, dl_ctas(STREAM, DO)) k_distill_long(const DtArgs a) {
  extern __shared__ __align__(16) unsigned char dt_raw[];
  __shared__ float2 s_part[2][DL_MOST_SHARE * STREAM / 32];
  constexpr int VN = RW_VEC<T>, PARTS = STREAM / 32, RING = dl_ring(DO), STEP = STREAM * 16;
  constexpr bool BOTH = DO == (DT_LOSS | DT_GRAD);
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, K = a.top, V = a.vocab;
  uint32_t rank, share;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(share));
  if ((DO & DT_LOSS) && share > 1) rw_cluster_sync();   // the others are running
  pdl_begin();
  const long long groups = gridDim.x / share;
  const float c = a.c, factor = DO & DT_GRAD ? dt_factor(a) : 0.f;
  const uint64_t cc = rw_pair(c, c);
  double loss_sum = 0.0, weight_sum = 0.0;
  // A row, and what of it is this CTA's: `pieces` of 16 bytes from element `at` on, elements lo to hi; of those pieces t, t + STREAM, ... are thread t's,
  // `count` of them, from `from` on
  struct Row { const T* s; const unsigned char* from; int at, pieces, lo, hi, count; };
  auto place = [&](long long row) {
    Row r;
    r.s = (const T*)a.logits + row * a.stride;
    const int head = min(V, (int)((16 - ((uintptr_t)r.s & 15)) & 15) / (int)sizeof(T)), all = (V - head) / VN;
    const int per = share > 1 ? (all + (int)share - 1) / (int)share : all, p0 = min((int)rank * per, all);
    r.pieces = min(per, all - p0);
    r.at = head + p0 * VN;
    r.lo = rank == 0 ? 0 : r.at;
    r.hi = rank == share - 1 ? V : r.at + r.pieces * VN;
    r.count = t < r.pieces ? (r.pieces - t + STREAM - 1) / STREAM : 0;
    r.from = (const unsigned char*)(r.s + r.at) + 16 * t;
    return r;
  };
  // a row without a weight that counts
  auto pass_over = [&](long long row) {
    if constexpr (DO & DT_LOSS) {
      if (t == 0 && rank == 0 && a.row_loss) a.row_loss[row] = 0.f;
    }
    if constexpr (DO & DT_GRAD) {
      const Row r = place(row);
      T* const grad = (T*)a.grad + row * V;
      for (int j = r.lo + t; j < r.hi; j += STREAM) grad[j] = rw_to<T>(0.f);
    }
  };
  // the next row that counts, its teacher's sums and (of an earlier call) its maximum and sum
  struct Next { long long row; float4 teacher; float2 st; };
  auto look = [&](long long row) {
    Next n = {row, make_float4(0.f, 0.f, 0.f, 0.f), make_float2(0.f, 0.f)};
    if (row < a.rows) {
      n.teacher = a.teachers[row];
      if constexpr (!(DO & DT_LOSS)) n.st = a.stat[row];
    }
    return n;
  };
  Next peeked = look(blockIdx.x / share);   // asked for a row ahead
  auto find = [&] {
    Next n = peeked;
    while (n.row < a.rows && n.teacher.x == 0.f) {
      pass_over(n.row);
      n = look(n.row + groups);
    }
    peeked = look(n.row + groups);
    return n;
  };
  const uint32_t ring = smem_addr(dt_raw) + 16 * t;
  uint32_t in = 0, out = 0;   // places of the ring, as offsets: where the next copy goes, where the next piece is
  auto copy = [&](const unsigned char* from) {
    rw_copy(ring + in, from);
    in = in == (RING - 1) * STEP ? 0 : in + STEP;
  };
  auto take = [&] {
    RwPiece<T, VN> v;
    v.from_shared(ring + out);
    out = out == (RING - 1) * STEP ? 0 : out + STEP;
    return v;
  };
  Next now = find(), next = now;
  Row r = place(now.row < a.rows ? now.row : 0), coming = r;
  if (now.row >= a.rows) r.count = 0;
  int on_way = min(RING, r.count);   // this row's pieces that have been asked for
  for (int i = 0; i < on_way; ++i) { copy(r.from + i * STEP); rw_commit(); }
  auto entry_of = [&](long long row) { return (DO & DT_GRAD) && t < K && row < a.rows ? a.columns[row * K + t] : make_int2(-1, 0); };
  int2 entry1 = entry_of(now.row);   // asked for a row ahead
  int buf = 0;
  for (; now.row < a.rows; now = next, r = coming) {
    const long long row = now.row;
    next = find();
    coming = place(next.row < a.rows ? next.row : 0);
    if (next.row >= a.rows) coming.count = 0;
    const float w = now.teacher.x;
    float2 st = now.st;
    T* const grad = DO & DT_GRAD ? (T*)a.grad + row * V : nullptr;
    const float f = DO & DT_GRAD ? factor * w * (a.upstream && a.per_row ? a.upstream[row] : 1.0f) : 0.f;
    const int2 entry = entry1;   // the teacher's entry whose column is this thread's
    entry1 = entry_of(next.row);
    // an element before the row's first piece or behind its last
    const int head = rank == 0 ? r.at : 0, edge = t < head ? t : r.at + r.pieces * VN + t - head;
    const bool has_edge = t < head || (rank == share - 1 && edge < V);
    T outside = rw_to<T>(0.f);   // (as it comes: anything computed of it would have to wait for it here)
    if (has_edge) outside = r.s[edge];
    static_assert(2 * (VN - 1) <= STREAM, "a thread per element outside of the pieces");
    // One pass over the row's pieces, each of which makes room for another: of this row, then of the next.  A piece was asked for `on_way` pieces before.
    auto sweep = [&](auto&& work) {
      const int rest = r.count - on_way;
      const unsigned char* from = r.from + on_way * STEP;
      if (on_way == RING)
#pragma unroll 2
        for (int k = 0; k < rest; ++k, from += STEP) {
          asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
          const RwPiece<T, VN> v = take();
          work(v);
          copy(from);
          rw_commit();
        }
      from = coming.from;
      const int most = min(on_way, coming.count);
      for (int k = 0; k < on_way; ++k, from += STEP) {
        if (on_way == RING) asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
        else rw_arrived(0);
        const RwPiece<T, VN> v = take();
        work(v);
        if (k < most) copy(from);
        rw_commit();
      }
      // a next row that is longer than this one
      from = coming.from + most * STEP;
      for (int k = most; k < min(RING, coming.count); ++k, from += STEP) {
        copy(from);
        rw_commit();
      }
      on_way = min(RING, coming.count);
    };
    // this thread's part of the gradient, from powers relative to m
    auto gradient = [&](float m, float total, auto&& over) {
      const float g = f * total;
      const uint64_t gg = rw_pair(g, g), mm = rw_pair(-m, -m);
      T* to = grad + r.at + t * VN;
      T logit = rw_to<T>(0.f);
      const bool has_entry = entry.x >= r.lo && entry.x < r.hi;
      if (has_entry) logit = r.s[entry.x];
      auto go = [&](auto aligned) {
        over([&](const RwPiece<T, VN>& v) {
          float x[VN];
#pragma unroll
          for (int j = 0; j < VN; j += 2) {
            rw_unpair(rw_mul2(rw_add2(v.two(j), mm), cc), x[j], x[j + 1]);
            rw_unpair(rw_mul2(gg, rw_pair(dt_exp2(x[j]), dt_exp2(x[j + 1]))), x[j], x[j + 1]);
          }
          RwPiece<T, VN> o;
          o.make([&](int j) { return x[j]; });
          if constexpr (decltype(aligned)::value) o.store(to);
          else
#pragma unroll
            for (int j = 0; j < VN; ++j) to[j] = o.one(j);
          to += STREAM * VN;
        });
      };
      if (((uintptr_t)(grad + r.at) & 15) == 0) go(std::true_type());
      else go(std::false_type());
      if (has_edge) grad[edge] = rw_to<T>(g * dt_exp2((rw_float(outside) - m) * c));
      __syncthreads();   // behind it, the columns of the teacher's entries are written again
      if (has_entry) dt_column(grad, entry.x, __int_as_float(entry.y), rw_float(logit), f, total, m, c);
      for (int k = t + STREAM; k < K; k += STREAM) {
        const int2 q = a.columns[row * K + k];
        if (q.x >= r.lo && q.x < r.hi) dt_column(grad, q.x, __int_as_float(q.y), rw_float(r.s[q.x]), f, total, m, c);
      }
    };
    if constexpr (!(DO & DT_LOSS)) gradient(st.x, st.y, sweep);
    else {
      float m = DT_LOWEST;   // maximum
      uint64_t mm = rw_pair(-m, -m), sum = rw_pair(0.f, 0.f);   // sums of powers relative to it
      auto raise = [&](float to) {
        const float by = dt_exp2((m - to) * c);
        sum = rw_mul2(sum, rw_pair(by, by));
        m = to;
        mm = rw_pair(-m, -m);
      };
      auto add = [&](const RwPiece<T, VN>& v) {
        const float most = rw_most(v);
        if (most > m) raise(most);
#pragma unroll
        for (int j = 0; j < VN; j += 2) {
          float x, y;
          rw_unpair(rw_mul2(rw_add2(v.two(j), mm), cc), x, y);
          sum = rw_add2(sum, rw_pair(dt_exp2(x), dt_exp2(y)));
        }
      };
      if constexpr (!BOTH) sweep(add);
      else {
        // the rest of the row, and as much of the next as there is room for (on_way: of the next from here on)
        const uint32_t first = out;
        for (int k = on_way; k < r.count; ++k) { copy(r.from + k * STEP); rw_commit(); }
        on_way = min(RING - r.count, coming.count);
        for (int k = 0; k < RING - r.count; ++k) {
          if (k < on_way) copy(coming.from + k * STEP);
          rw_commit();
        }
        for (int k = 0; k < r.count; k += 4) {
          rw_arrived(RING - 1 - min(k + 3, RING - 1));
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (k + i < r.count) add(take());
        }
        out = first;
      }
      if (has_edge) {
        const float v = rw_float(outside);
        if (v > m) raise(v);
        sum = rw_add2(sum, rw_pair(dt_exp2((v - m) * c), 0.f));
      }
      const float all = rw_warp_max(m);
      float total = rw_warp_sum(rw_both(sum) * dt_exp2((m - all) * c));
      if (lane < (int)share) {
        const uint32_t to = rw_at_rank(&s_part[buf][rank * PARTS + warp], lane);
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(all), "f"(total) : "memory");
      }
      if (share > 1) rw_cluster_sync();
      else __syncthreads();
      if (BOTH || warp == 0) {
        const int parts = (int)share * PARTS;
        constexpr int EACH = (DL_MOST_SHARE * PARTS + 31) / 32;   // of a lane
        float2 x[EACH];
        m = DT_LOWEST;
        total = 0.f;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          x[i] = lane + 32 * i < parts ? s_part[buf][lane + 32 * i] : make_float2(DT_LOWEST, 0.f);
          m = fmaxf(m, x[i].x);
        }
        m = rw_warp_max(m);
#pragma unroll
        for (int i = 0; i < EACH; ++i) total += x[i].y * dt_exp2((x[i].x - m) * c);
        total = rw_warp_sum(total);
        st = make_float2(m, 1.0f / total);
        if (t == 0 && rank == 0) {
          const float loss = w * a.temperature * a.temperature * DT_LN2 * fmaf(now.teacher.z, (m - now.teacher.w) * c, now.teacher.y + log2f(total));
          if (a.row_loss) a.row_loss[row] = loss;
          if (a.stat) a.stat[row] = st;
          loss_sum += loss;
          weight_sum += w;
        }
      }
      buf ^= 1;
      if constexpr (BOTH)
        // the second pass: each piece makes room for one of the next row
        gradient(st.x, st.y, [&](auto&& work) {
          const int from = on_way;
          on_way = min(from + r.count, coming.count);
          for (int k = 0; k < r.count; ++k) {
            work(take());
            if (from + k < on_way) copy(coming.from + (from + k) * STEP);
            rw_commit();
          }
        });
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if constexpr (DO & DT_LOSS)
    if (t == 0 && rank == 0) a.part[blockIdx.x / share] = make_double2(loss_sum, weight_sum);
}

// The weights that count, before the gradient is scaled by their sum: a row's is zero if it has no teacher.
__global__ void __launch_bounds__(NT) k_distill_weights(const DtArgs a, double* part) {
  pdl_begin();
  __shared__ double s_d[NWARP];
  double w = 0.0;
  for (long long row = (long long)blockIdx.x * NT + threadIdx.x; row < a.rows; row += (long long)gridDim.x * NT) {
    const float weight = a.weights ? a.weights[row] : 1.0f;
    bool any = false;
    for (int k = 0; k < a.top && !any && weight != 0.f; ++k)   // the first entry, nearly always
      any = dt_id(a, row * a.top + k) >= 0 && !(dt_any(a.teacher, a.teacher_type, row * a.top + k) == -CUDART_INF_F);
    if (any) w += weight;
  }
  w = warp_sum_d(w);
  if ((threadIdx.x & 31) == 0) s_d[threadIdx.x >> 5] = w;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < NWARP; ++i) w += s_d[i];
    part[blockIdx.x] = w;
  }
}
// The CTAs' sums: loss[0] their sum, or (mean) over that of the weights; inv[0] one over that
__global__ void __launch_bounds__(NT) k_distill_total(const double2* __restrict__ part, int n, int mean, float* loss, float* inv) {
  pdl_begin();
  __shared__ double s_d[2][NWARP];
  double l = 0.0, w = 0.0;
  for (int i = threadIdx.x; i < n; i += NT) { l += part[i].x; w += part[i].y; }
  l = warp_sum_d(l);
  w = warp_sum_d(w);
  if ((threadIdx.x & 31) == 0) { s_d[0][threadIdx.x >> 5] = l; s_d[1][threadIdx.x >> 5] = w; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < NWARP; ++i) { l += s_d[0][i]; w += s_d[1][i]; }
    if (loss) loss[0] = (float)(!mean ? l : w != 0.0 ? l / w : 0.0);
    if (inv) inv[0] = w != 0.0 ? (float)(1.0 / w) : 0.f;
  }
}

// A call's form.  Threads that stream through a long row: few for short ones, so that more rows' latencies lie side by side.  share: CTAs that share a
// row, until all have work, or (loss and gradient) until DL_KEPT pieces of a thread are its part of the row.
struct DtForm { int stream, share; bool fits; };   // fits: into the rings
static DtForm dt_form(long long rows, int vocab, int type_bytes, bool both) {
  if (vocab <= DT_WARP_VOCAB) return {0, 1, true};
  const long long bytes = (long long)vocab * type_bytes;
  const int stream = bytes <= (both ? 32768 : 131072) ? 128 : 256;
  const long long most = (long long)sm_count() * dl_ctas(stream, both ? DT_LOSS | DT_GRAD : DT_LOSS);
  int share = 1;
  while (share < DL_MOST_SHARE && ((bytes >= share * 2 * 16384 && rows * share * 2 <= most) || (both && bytes > (long long)share * stream * 16 * DL_KEPT))) share *= 2;
  return {stream, share, bytes <= (long long)share * stream * 16 * dl_ring(DT_LOSS | DT_GRAD)};
}
static int dt_weight_ctas(long long rows) { return (int)(rows < 64 * NT ? (rows + NT - 1) / NT : 64); }   // at most as many as rows
static size_t dt_teacher_smem(int top) { return (sizeof(DtEntry) * top + (size_t)4 * dt_slots(top)) * (DT_WARP_THREADS / 32); }
// CTAs whose warps have a row each
static int dt_warp_ctas(long long rows) {
  const long long n = (rows + DT_WARP_THREADS / 32 - 1) / (DT_WARP_THREADS / 32), most = (long long)sm_count() * DT_MOST_CTAS;
  return (int)(n < most ? n : most);
}
// Launches one pass; *groups: CTAs or clusters that begin with different rows, which is also the number of partial sums
template <class T, int DO>
static int dt_run(const DtArgs& a, const DtForm& form, int* groups, cudaStream_t s) {
#define DT_LONG(STREAM)                                                                                                              \
  {                                                                                                                                  \
    constexpr int RING = dl_ring(DO) * STREAM * 16;                                                                                  \
    static bool configured[PYLO_MAX_DEVICES] = {};                                                                                   \
    if (int rc = allow_dynamic_smem(k_distill_long<T, DO, STREAM>, RING, configured)) return rc;                                     \
    const long long most = form.share > 1 ? active_clusters<k_distill_long<T, DO, STREAM>>(STREAM, form.share, RING)                 \
                                          : (long long)sm_count() * dl_ctas(STREAM, DO);                                             \
    *groups = (int)(a.rows < most ? a.rows : most);                                                                                  \
    t_plain_next = true;   /* beside a kernel that needs less shared memory, not as many CTAs would fit an SM as do */               \
    launch_clusters(k_distill_long<T, DO, STREAM>, *groups * form.share, STREAM, form.share, RING, s, a);                            \
    return launch_status();                                                                                                          \
  }
  if (form.stream == 128) DT_LONG(128)
  if (form.stream == 256) DT_LONG(256)
#undef DT_LONG
  static bool configured[PYLO_MAX_DEVICES] = {};
  if (int rc = allow_dynamic_smem(k_distill_short<T, DO>, (int)dt_teacher_smem(DT_MOST_K), configured)) return rc;
  *groups = dt_warp_ctas(a.rows);
  launch(k_distill_short<T, DO>, *groups, DT_WARP_THREADS, dt_teacher_smem(a.top), s, a);
  return launch_status();
}
template <int DO>
static int dt_any_type(const DtArgs& a, int type, const DtForm& form, int* groups, cudaStream_t s) {
  return type == PYLO_FP32 ? dt_run<float, DO>(a, form, groups, s) : type == PYLO_BF16 ? dt_run<__nv_bfloat16, DO>(a, form, groups, s) : dt_run<__half, DO>(a, form, groups, s);
}
template <class T>
static int dt_teachers(const DtArgs& a, double* sums, cudaStream_t s) {
  static bool configured[PYLO_MAX_DEVICES] = {};
  if (int rc = allow_dynamic_smem(k_distill_teachers<T>, (int)dt_teacher_smem(DT_MOST_K), configured)) return rc;
  launch(k_distill_teachers<T>, dt_warp_ctas(a.rows), DT_WARP_THREADS, dt_teacher_smem(a.top), s, a, sums);
  return launch_status();
}
// What lies in a call's workspace: the first is kept for a gradient alone
struct DtWork {
  float2* stat; float* inv; float4* teachers; int2* columns;
  double2* part; double* sums;
  int64_t bytes;
};
static DtWork dt_work(void* base, int64_t rows, int vocab, int top) {
  char* p = (char*)base;
  const bool is_long = vocab > DT_WARP_VOCAB;
  const int64_t most = (int64_t)sm_count() * DT_MOST_CTAS, groups = rows < most ? rows : most;
  auto take = [&](int64_t bytes) { char* q = p; p += (bytes + 15) / 16 * 16; return (void*)q; };
  DtWork w = {};
  w.inv = (float*)take(4);
  w.stat = (float2*)take(8 * rows);
  w.teachers = (float4*)take(is_long ? 16 * rows : 0);
  w.columns = (int2*)take(is_long ? 8 * rows * top : 0);
  w.part = (double2*)take(16 * groups);
  w.sums = (double*)take(8 * groups);
  w.bytes = p - (char*)base;
  return w;
}
static bool dt_good(const pylo_distill* d) {
  return d && d->rows >= 0 && d->rows <= (1ll << 40) && d->vocab > 0 && d->vocab <= (1 << 30) && d->top > 0 && d->top <= DT_MOST_K && rw_type(d->type) &&
         rw_type(d->teacher_type) && (d->ids_bytes == 4 || d->ids_bytes == 8) && d->temperature > 0.f && (d->rows == 0 || (d->logits && d->teacher && d->ids)) &&
         d->stride >= d->vocab && d->reduction >= PYLO_REDUCE_NONE && d->reduction <= PYLO_REDUCE_MEAN && rw_on(rw_bytes(d->type), d->logits, d->grad) &&
         rw_on(rw_bytes(d->teacher_type), d->teacher) && rw_on(d->ids_bytes, d->ids) && rw_on(4, d->weights, d->loss, d->row_loss, d->upstream);
}
static DtArgs dt_args(const pylo_distill* d) {
  DtArgs a = {};
  a.logits = d->logits; a.teacher = d->teacher; a.ids = d->ids; a.weights = d->weights;
  a.row_loss = d->row_loss; a.grad = d->grad; a.upstream = d->upstream; a.per_row = d->reduction == PYLO_REDUCE_NONE;
  a.rows = d->rows; a.stride = d->stride; a.vocab = d->vocab; a.top = d->top; a.teacher_type = d->teacher_type; a.wide_ids = d->ids_bytes == 8;
  a.c = (float)(DT_LOG2E / d->temperature); a.temperature = d->temperature; a.scale = 1.0f;
  return a;
}

static bool ln_good(const pylo_norm* n) {
  return n && n->rows >= 0 && n->width > 0 && n->width <= LN_MOST && rw_type(n->type) && rw_type(n->weight_type) && rw_on(rw_bytes(n->type), n->x, n->y, n->dy, n->dx) &&
         rw_on(rw_bytes(n->weight_type), n->weight, n->bias, n->dweight, n->dbias) && rw_on(4, n->mean, n->rstd, n->work);
}

extern "C" {

int64_t pylo_b200_layer_norm_workspace(int64_t rows, int width) {
  if (rows <= 0 || width <= 0 || width > LN_MOST) return 0;
  const int a = ln_form(rows, width, false, true, true).groups, b = ln_form(rows, width, true, true, true).groups;   // (those without rings have fewer)
  return (int64_t)(a > b ? a : b) * 2 * width;
}

int pylo_b200_layer_norm(const pylo_norm* n, void* stream) {
  CHECK_ARG(ln_good(n) && n->eps >= 0.f);
  if (n->rows == 0) return 0;
  CHECK_ARG(n->x && n->y && (n->mean == nullptr) == (n->rstd == nullptr) && (n->weight || !n->bias) && n->x_stride >= 0);
  LnArgs a = {};
  a.x = n->x; a.weight = n->weight; a.bias = n->bias; a.y = n->y; a.mean = n->mean; a.rstd = n->rstd;
  a.rows = n->rows; a.x_stride = n->x_stride; a.width = n->width; a.eps = n->eps;
  return ln_any(a, n->type, n->weight_type, ln_aligned(n, false), false, (cudaStream_t)stream);
}

int pylo_b200_layer_norm_backward(const pylo_norm* n, void* stream) {
  CHECK_ARG(ln_good(n));
  cudaStream_t s = (cudaStream_t)stream;
  const bool columns = n->dweight || n->dbias, aligned = ln_aligned(n, true);
  const int groups = n->rows ? ln_form(n->rows, n->width, aligned && n->type != PYLO_FP32, true, aligned).groups : 0;
  CHECK_ARG(!columns || groups == 0 || (n->work && n->work_floats >= (int64_t)groups * 2 * n->width));
  if (groups) {
    CHECK_ARG(n->x && n->dy && n->mean && n->rstd && n->x_stride >= 0 && n->dy_stride >= 0);
    LnArgs a = {};
    a.x = n->x; a.dy = n->dy; a.weight = n->weight; a.y = n->dx; a.mean = n->mean; a.rstd = n->rstd; a.part = columns ? n->work : nullptr;
    a.rows = n->rows; a.x_stride = n->x_stride; a.dy_stride = n->dy_stride; a.width = n->width;
    if (n->dx || columns)
      if (int rc = ln_any(a, n->type, n->weight_type, aligned, true, s)) return rc;
  }
  if (columns) {
    const dim3 grid((n->width + 31) / 32, n->dbias ? 2 : 1);
#define LN_COLUMNS(W) launch(k_layer_norm_columns<W>, grid, 32 * LN_COLUMN_GROUPS, 0, s, n->work, groups, n->width, (W*)n->dweight, (W*)n->dbias)
    if (n->weight_type == PYLO_FP32) LN_COLUMNS(float);
    else if (n->weight_type == PYLO_BF16) LN_COLUMNS(__nv_bfloat16);
    else if (n->weight_type == PYLO_FP16) LN_COLUMNS(__half);
    else return -1;
#undef LN_COLUMNS
  }
  return launch_status();
}

int64_t pylo_b200_distill_workspace(int64_t rows, int vocab, int top) { return rows < 0 || vocab <= 0 || top <= 0 ? 0 : dt_work(nullptr, rows, vocab, top).bytes; }

int pylo_b200_distill(const pylo_distill* d, int what, void* stream) {
  CHECK_ARG(dt_good(d) && (what == PYLO_DISTILL_LOSS || what == PYLO_DISTILL_GRAD || what == (PYLO_DISTILL_LOSS | PYLO_DISTILL_GRAD)));
  cudaStream_t s = (cudaStream_t)stream;
  const bool loss = what & PYLO_DISTILL_LOSS, grad = what & PYLO_DISTILL_GRAD, mean = d->reduction == PYLO_REDUCE_MEAN;
  CHECK_ARG(d->work && (uintptr_t)d->work % 16 == 0 && d->work_bytes >= pylo_b200_distill_workspace(d->rows, d->vocab, d->top));
  CHECK_ARG(!grad || d->rows == 0 || d->grad);
  const DtWork w = dt_work(d->work, d->rows, d->vocab, d->top);
  int groups = 0;
  if (d->rows) {
    const DtForm form = dt_form(d->rows, d->vocab, (int)rw_bytes(d->type), loss && grad);
    DtArgs a = dt_args(d);
    a.part = w.part; a.stat = w.stat; a.teachers = w.teachers; a.columns = w.columns;
    if (grad) a.scale = d->scale;
    if (loss && form.stream) {
      const int rc = d->type == PYLO_FP32 ? dt_teachers<float>(a, w.sums, s) : d->type == PYLO_BF16 ? dt_teachers<__nv_bfloat16>(a, w.sums, s) : dt_teachers<__half>(a, w.sums, s);
      if (rc) return rc;
    }
    if (grad && mean) {
      if (!loss) a.inv = w.inv;
      else {
        a.weight_sums = w.sums;
        a.n_sums = form.stream ? dt_warp_ctas(d->rows) : dt_weight_ctas(d->rows);
        if (!form.stream) launch(k_distill_weights, a.n_sums, NT, 0, s, a, w.sums);
      }
    }
    int rc, unused;
    if (loss && grad && form.fits) rc = dt_any_type<DT_LOSS | DT_GRAD>(a, d->type, form, &groups, s);
    else {
      rc = loss ? dt_any_type<DT_LOSS>(a, d->type, form, &groups, s) : 0;
      if (grad && !rc) rc = dt_any_type<DT_GRAD>(a, d->type, form, &unused, s);
    }
    if (rc) return rc;
  }
  if (loss && d->reduction != PYLO_REDUCE_NONE)
    launch(k_distill_total, 1, NT, 0, s, (const double2*)w.part, groups, (int)mean, d->loss, w.inv);
  return launch_status();
}

}  // extern "C"
