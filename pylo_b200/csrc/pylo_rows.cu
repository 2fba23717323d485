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
// Sums over the threads of a row, in every one of them.  buf: 32 floats of shared memory that all threads of the CTA have finished
// reading by the barrier before the last: two calls in a row take two of them.
template <bool BLOCK>
__device__ __forceinline__ float rw_sum(float v, float* buf) {
  v = rw_warp_sum(v);
  if constexpr (BLOCK) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) buf[warp] = v;
    __syncthreads();
    v = rw_warp_sum(lane < (int)(blockDim.x >> 5) ? buf[lane] : 0.f);
  }
  return v;
}
// ------------------------------------------------------------------------------------------------
// Layer norm.  m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), xh = (x - m) r:
//   y = xh w + b;   dx = r (q - mean q - xh mean(q xh)) with q = dy w;   dw = sum over rows dy xh, db = sum over rows dy
//
// A row is read once and stays in registers, 32 elements of each thread at most, so that the variance is that of the differences
// from the mean (a sum of squares less the mean's would lose what rows far off centre have).  The weights stay in registers from row
// to row, the sums of their gradients too; they leave as one partial sum per CTA, and a second kernel adds those up in a fixed order.
// ------------------------------------------------------------------------------------------------
#define LN_ELEMS 32           // of a row per thread at most
#define LN_WARP_THREADS 128   // of a CTA whose warps have a row each
#define LN_MOST 32768         // elements of a row: 1024 threads

struct LnArgs {
  const void *x, *dy, *weight, *bias;
  void *y;               // or dx, or NULL
  float *mean, *rstd;    // written forward (or NULL), read backward
  float* part;           // [CTAs][2][width]: sums for dw, db; or NULL
  long long rows, x_stride, dy_stride;
  int width;
  float eps;
};

template <class T, class W, int VN, int E, int MOST>
__global__ void __launch_bounds__(MOST ? MOST : LN_WARP_THREADS) k_layer_norm(const LnArgs a) {
  pdl_begin();
  constexpr bool BLOCK = MOST > 0;   // a row is a CTA's, of so many threads at most
  constexpr int NV = E / VN;
  __shared__ float s_buf[2][32];
  const int t = BLOCK ? threadIdx.x : threadIdx.x & 31, threads = BLOCK ? blockDim.x : 32, width = a.width;
  const long long step = BLOCK ? gridDim.x : (long long)gridDim.x * (LN_WARP_THREADS / 32);
  long long row = BLOCK ? blockIdx.x : (long long)blockIdx.x * (LN_WARP_THREADS / 32) + (threadIdx.x >> 5);
  const float inv = 1.0f / (float)width;
  const T* const x = (const T*)a.x;
  T* const y = (T*)a.y;
  RwPiece<T, VN> v[NV];
  auto fetch = [&](long long r) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * threads) * VN;
      if (c < width && r < a.rows) v[i].load(x + r * a.x_stride + c);
      else v[i].make([](int) { return 0.f; });
    }
  };
  fetch(row);
  for (; row < a.rows; row += step) {
    float f[E], sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VN; ++j) sum += f[i * VN + j] = v[i].at(j);
    fetch(row + step);
    const float mean = rw_sum<BLOCK>(sum, s_buf[0]) * inv;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((t + i * threads) * VN < width)
#pragma unroll
        for (int j = 0; j < VN; ++j) {
          const float d = f[i * VN + j] - mean;
          f[i * VN + j] = d;
          sq = fmaf(d, d, sq);
        }
    const float rstd = 1.0f / sqrtf(fmaf(rw_sum<BLOCK>(sq, s_buf[1]), inv, a.eps));
    if (t == 0 && a.mean) { a.mean[row] = mean; a.rstd[row] = rstd; }
    T* const out = y + row * width;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * threads) * VN;
      if (c < width) {
        RwPiece<T, VN> o;
        o.make([&](int j) {
          float q = f[i * VN + j] * rstd;
          if (a.weight) q *= rw_float(((const W*)a.weight)[c + j]);
          if (a.bias) q += rw_float(((const W*)a.bias)[c + j]);
          return q;
        });
        o.store(out + c);
      }
    }
  }
}

template <class T, class W, int VN, int E, int MOST>
__global__ void __launch_bounds__(MOST ? MOST : LN_WARP_THREADS) k_layer_norm_backward(const LnArgs a) {
  pdl_begin();
  constexpr bool BLOCK = MOST > 0;   // a row is a CTA's, of so many threads at most
  constexpr int NV = E / VN, WARPS = LN_WARP_THREADS / 32;
  __shared__ float s_buf[4][32];
  __shared__ float s_cols[BLOCK ? 1 : 2 * 32 * E];
  const int t = BLOCK ? threadIdx.x : threadIdx.x & 31, threads = BLOCK ? blockDim.x : 32, width = a.width;
  const long long step = BLOCK ? gridDim.x : (long long)gridDim.x * WARPS;
  const float inv = 1.0f / (float)width;
  float dw[E], db[E];
#pragma unroll
  for (int j = 0; j < E; ++j) dw[j] = db[j] = 0.f;
  int flip = 0;
  for (long long row = BLOCK ? blockIdx.x : (long long)blockIdx.x * WARPS + (threadIdx.x >> 5); row < a.rows; row += step, flip ^= 2) {
    const T* const x = (const T*)a.x + row * a.x_stride;
    const T* const dy = (const T*)a.dy + row * a.dy_stride;
    RwPiece<T, VN> vx[NV], vd[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * threads) * VN;
      if (c < width) { vx[i].load(x + c); vd[i].load(dy + c); }
      else { vx[i].make([](int) { return 0.f; }); vd[i].make([](int) { return 0.f; }); }
    }
    const float mean = a.mean[row], rstd = a.rstd[row];
    float q[E], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * threads) * VN;
      if (c < width)
#pragma unroll
        for (int j = 0; j < VN; ++j) {
          const int e = i * VN + j;
          const float d = vd[i].at(j), xh = (vx[i].at(j) - mean) * rstd;
          dw[e] = fmaf(d, xh, dw[e]);
          db[e] += d;
          q[e] = a.weight ? d * rw_float(((const W*)a.weight)[c + j]) : d;
          s1 += q[e];
          s2 = fmaf(q[e], xh, s2);
        }
    }
    if (a.y == nullptr) continue;
    s1 = rw_sum<BLOCK>(s1, s_buf[flip]) * inv;
    s2 = rw_sum<BLOCK>(s2, s_buf[flip + 1]) * inv;
    T* const out = (T*)a.y + row * width;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (t + i * threads) * VN;
      if (c < width) {
        RwPiece<T, VN> o;
        o.make([&](int j) { return rstd * (q[i * VN + j] - s1 - (vx[i].at(j) - mean) * rstd * s2); });
        o.store(out + c);
      }
    }
  }
  if (a.part == nullptr) return;
  float* const part = a.part + (long long)blockIdx.x * 2 * width;
  if constexpr (BLOCK) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VN; ++j) {
        const int c = (t + i * threads) * VN + j;
        if (c < width) { part[c] = dw[i * VN + j]; part[width + c] = db[i * VN + j]; }
      }
  } else {
    // the warps' sums, one warp after the other
    for (int w = 0; w < WARPS; ++w) {
      if ((int)(threadIdx.x >> 5) == w)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < VN; ++j) {
            const int at = (t + i * 32) * VN + j;
            s_cols[at] = w ? s_cols[at] + dw[i * VN + j] : dw[i * VN + j];
            s_cols[32 * E + at] = w ? s_cols[32 * E + at] + db[i * VN + j] : db[i * VN + j];
          }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < width; c += LN_WARP_THREADS) { part[c] = s_cols[c]; part[width + c] = s_cols[32 * E + c]; }
  }
}

// The partial sums of 32 columns by a CTA: eight rows of threads, each adding up every eighth partial, then those.
template <class W>
__global__ void __launch_bounds__(NT) k_layer_norm_columns(const float* __restrict__ part, int n, int width, W* dweight, W* dbias) {
  pdl_begin();
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  W* const out = blockIdx.y ? dbias : dweight;
  if (out == nullptr) return;
  const float* p = part + (blockIdx.y ? width : 0) + c;
  float sum = 0.f;
  if (c < width)
    for (int i = g; i < n; i += 8) sum += p[(long long)i * 2 * width];
  s[g][lane] = sum;
  __syncthreads();
  if (g == 0 && c < width) {
#pragma unroll
    for (int i = 1; i < 8; ++i) sum += s[i][lane];
    out[c] = rw_to<W>(sum);
  }
}

// CTAs of a call: as many as run at once, by rows of so many threads
static int ln_threads(int width) { return width <= 32 * LN_ELEMS ? LN_WARP_THREADS : (width + 32 * LN_ELEMS - 1) / (32 * LN_ELEMS) * 32; }
static long long ln_groups(long long rows, int width) { return width <= 32 * LN_ELEMS ? (rows + LN_WARP_THREADS / 32 - 1) / (LN_WARP_THREADS / 32) : rows; }
static int ln_ctas(long long rows, int width, int resident) {
  const int t = ln_threads(width), per = resident / t > 1 ? resident / t : 1;
  const long long n = ln_groups(rows, width), most = (long long)sm_count() * per;
  return (int)(n < most ? n : most);
}
#define LN_FORWARD 1024   // threads of an SM: forward, backward
#define LN_BACKWARD 384

template <class T, class W, int VN>
static void ln_launch(const LnArgs& a, bool backward, cudaStream_t s) {
  const int t = ln_threads(a.width), ctas = ln_ctas(a.rows, a.width, backward ? LN_BACKWARD : LN_FORWARD);
  constexpr int FEW = VN > 1 ? RW_VEC<T> : 8;
#define LN_GO(E, MOST) backward ? launch(k_layer_norm_backward<T, W, VN, E, MOST>, ctas, t, 0, s, a) : launch(k_layer_norm<T, W, VN, E, MOST>, ctas, t, 0, s, a)
  if (a.width <= 32 * FEW) LN_GO(FEW, 0);
  else if (a.width <= 32 * LN_ELEMS) LN_GO(LN_ELEMS, 0);
  else if (t <= 256) LN_GO(LN_ELEMS, 256);
  else LN_GO(LN_ELEMS, 1024);
#undef LN_GO
}
template <class T, class W>
static void ln_run(const LnArgs& a, bool backward, cudaStream_t s) {
  // 16 bytes at a time where every row begins on their boundary
  const bool aligned = ((uintptr_t)a.x | (uintptr_t)a.dy | (uintptr_t)a.y) % 16 == 0 &&
                       (a.width | a.x_stride | (backward ? a.dy_stride : 0)) % RW_VEC<T> == 0;
  aligned ? ln_launch<T, W, RW_VEC<T>>(a, backward, s) : ln_launch<T, W, 1>(a, backward, s);
}
static int ln_any(const LnArgs& a, int type, int weight_type, bool backward, cudaStream_t s) {
  if (type == PYLO_FP32 && weight_type == PYLO_FP32) ln_run<float, float>(a, backward, s);
  else if (type == PYLO_BF16 && weight_type == PYLO_BF16) ln_run<__nv_bfloat16, __nv_bfloat16>(a, backward, s);
  else if (type == PYLO_FP16 && weight_type == PYLO_FP16) ln_run<__half, __half>(a, backward, s);
  else if (type == PYLO_BF16 && weight_type == PYLO_FP32) ln_run<__nv_bfloat16, float>(a, backward, s);
  else if (type == PYLO_FP16 && weight_type == PYLO_FP32) ln_run<__half, float>(a, backward, s);
  else return -1;
  return launch_status();
}
static size_t rw_bytes(int type) { return type == PYLO_FP32 ? 4 : 2; }
static bool rw_type(int type) { return type == PYLO_FP32 || type == PYLO_BF16 || type == PYLO_FP16; }

// ------------------------------------------------------------------------------------------------
// Distillation from a teacher's K largest logits t at the ids i, of a student's logits s over V classes, at temperature T:
//   p = softmax(t / T) over the K entries,  q = softmax(s / T) over the V classes
//   loss of a row = T^2 sum_k p_k (log p_k - log q_{i_k});   its gradient: T (q_j - sum of the p_k with i_k = j)
// An id outside of [0, V) is padding, whatever the teacher's logit beside it is; a row whose entries are all padding or -inf has no
// teacher and the weight zero.  Rows of weight zero are not read, whatever they hold: their loss and gradient are zero.
//
// One pass over a row with a running maximum and sum per thread; powers of two of values that are scaled by log2(e) / T.  The
// gradient reads the row again (in the call that makes both, out of the L2 cache: the rows that are being worked on fit it).  The K
// columns with a teacher's entry are written a second time, behind a barrier, with what their entries add up to.
// ------------------------------------------------------------------------------------------------
#define DT_MOST_K 1024
#define DT_WARP_VOCAB 1024     // classes up to which a row is a warp's
#define DT_WARP_THREADS 128
#define DT_LOG2E 1.4426950408889634
#define DT_LN2 0.6931471805599453f
enum { DT_LOSS = 1, DT_GRAD = 2 };

struct DtArgs {
  const void *logits, *teacher, *ids;
  const float* weights;     // [rows] or NULL
  float* row_loss;          // [rows]: weight * loss, or NULL
  float2* stat;             // [rows]: maximum (scaled), 1 / sum of powers; written with the loss, read for a gradient alone; or NULL
  double2* part;            // [CTAs]: sums of weight * loss, of weights
  void* grad;               // [rows][vocab]
  const float* upstream;    // of the loss: a scalar, or (per_row) [rows]; NULL: 1
  const float* inv;         // scalar: 1 / sum of the weights; NULL: 1, or
  const double* weight_sums;// [n_sums]: its parts
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
// A row's K entries, by a warp; slots: dt_slots(K) words.  False if there are none
__device__ __forceinline__ bool dt_teacher(const DtArgs& a, long long row, DtEntry* e, int* slots) {
  const int lane = threadIdx.x & 31, K = a.top, n = dt_slots(K);
  float most = -CUDART_INF_F, sum = 0.f;
  bool any = false;
  for (int i = lane; i < n; i += 32) slots[i] = -1;
  __syncwarp();
  bool twice = false;   // a class that has an entry already
  for (int k = lane; k < K; k += 32) {
    const int id = dt_id(a, row * K + k);
    const float z = id >= 0 ? dt_any(a.teacher, a.teacher_type, row * K + k) * a.c : -CUDART_INF_F;
    e[k].id = id >= 0 ? id : DT_PADDING;
    e[k].lp = z;
    most = fmaxf(most, z);
    any |= !(z == -CUDART_INF_F);
    if (id >= 0)
      for (unsigned at = (unsigned)id * 2654435761u;; ++at) {   // ends: half of the slots stay free
        const int found = atomicCAS(&slots[(at ^ at >> 16) & (n - 1)], -1, id);
        twice |= found == id;
        if (found == -1 || found == id) break;
      }
  }
  if (!__any_sync(0xffffffffu, any)) return false;
  twice = __any_sync(0xffffffffu, twice);
  most = rw_warp_max(most);
  for (int k = lane; k < K; k += 32) sum += dt_exp2(e[k].lp - most);
  const float log_sum = log2f(rw_warp_sum(sum));
  for (int k = lane; k < K; k += 32) {
    const float lp = e[k].lp - most - log_sum, p = dt_exp2(lp);
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
// The loss of a row to base 2, without the student's sum: sum of p (log p - s), by a warp
template <class T>
__device__ __forceinline__ float dt_cross(const DtArgs& a, const T* s, const DtEntry* e, float m) {
  float sum = 0.f;
  for (int k = threadIdx.x & 31; k < a.top; k += 32) {
    const DtEntry q = e[k];
    if (!(q.p == 0.f)) sum = fmaf(q.p, q.lp - fmaf(rw_float(s[q.id < 0 ? ~q.id : q.id]), a.c, -m), sum);
  }
  return rw_warp_sum(sum);
}
// The columns of the teacher's entries among lo to hi, once more
template <class T>
__device__ __forceinline__ void dt_columns(const DtArgs& a, const T* s, T* grad, const DtEntry* e, float f, float total, float m, int t, int threads, int lo, int hi) {
  for (int k = t; k < a.top; k += threads) {
    const DtEntry q = e[k];
    if (q.id >= lo && q.id < hi) grad[q.id] = rw_to<T>(f * (total * dt_exp2(fmaf(rw_float(s[q.id]), a.c, -m)) - q.column));
  }
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
    const bool any = weight != 0.f && dt_teacher(a, row, e, slots);
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
    float m = -CUDART_INF_F, total = 0.f;   // scaled maximum; sum of powers relative to it
    if constexpr (DO & DT_LOSS) {
      auto add = [&](const float (&v)[VN]) {
        float most = v[0];
#pragma unroll
        for (int j = 1; j < VN; ++j) most = fmaxf(most, v[j]);
        const float up = fmaxf(m, most * a.c), ref = up == -CUDART_INF_F ? 0.f : up;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < VN; ++j) sum += dt_exp2(fmaf(v[j], a.c, -ref));
        total = fmaf(total, dt_exp2(m - ref), sum);
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
      const float all = rw_warp_max(m), ref = all == -CUDART_INF_F ? 0.f : all;
      total = rw_warp_sum(total * dt_exp2(m - ref));
      m = ref;
      const float cross = dt_cross(a, r.s, e, m);
      if (t == 0) {
        const float loss = weight * a.temperature * a.temperature * DT_LN2 * (cross + log2f(total));
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
      for (int i = t; i < V; i += 32) grad[i] = rw_to<T>(g * dt_exp2(fmaf(rw_float(r.s[i]), a.c, -m)));
      __syncwarp();   // behind it, the columns of the teacher's entries are written again
      dt_columns(a, r.s, grad, e, f, total, m, t, 32, 0, V);
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

// Long rows: a CTA each, or a cluster's, each CTA with its part of the row.  STREAM threads go through the logits, each with DL_U pieces of
// 16 bytes on their way, the next row's first ones behind this row's last; one more warp has the teacher's entries and the row's loss, so that
// nothing of the stream waits for them.  One barrier per row and pass: what the warps leave for one another lies in two buffers that take turns.
//
// A cluster shares a row where there are too few rows for all CTAs.
#define DL_U 4
#define DL_MOST_SHARE 8
__host__ __device__ constexpr int dl_ctas(int stream) { return stream == 128 ? 7 : stream == 256 ? 4 : 2; }   // of an SM
__device__ __forceinline__ uint64_t dt_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void dt_unpair(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t dt_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t dt_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t dt_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <class T, int DO, int STREAM>
__global__ void __launch_bounds__(STREAM + 32, dl_ctas(STREAM)) k_distill_long(const DtArgs a) {
  extern __shared__ __align__(16) unsigned char dt_raw[];
  __shared__ float2 s_part[2][DL_MOST_SHARE * STREAM / 32];
  __shared__ int s_any[2];
  constexpr int VN = RW_VEC<T>, U = DL_U, SPAN = U * STREAM, PARTS = STREAM / 32;
  constexpr float LOWEST = -3.0e38f;   // in the place of a maximum of -inf
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, K = a.top, V = a.vocab;
  const bool streams = warp < STREAM / 32;
  uint32_t rank, share;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(share));
  if (DO == DT_LOSS || DO == (DT_LOSS | DT_GRAD))
    if (share > 1) rw_cluster_sync();   // the others are running
  pdl_begin();
  const long long groups = gridDim.x / share;
  const float c = a.c, factor = DO & DT_GRAD ? dt_factor(a) : 0.f;
  const uint64_t cc = dt_pair(c, c);
  double loss_sum = 0.0, weight_sum = 0.0;
  RwPiece<T, VN> next[U];
  // A row, and what of it is this CTA's: `pieces` of 16 bytes from body on, elements lo to hi, thread t's element outside of the pieces (or -1)
  struct Row { const T *s, *body; int at, pieces, lo, hi, edge; };
  auto place = [&](long long row) {
    Row r;
    r.s = (const T*)a.logits + (row < a.rows ? row : 0) * a.stride;
    const int head = min(V, (int)((16 - ((uintptr_t)r.s & 15)) & 15) / (int)sizeof(T)), all = (V - head) / VN, tail = head + all * VN;
    const int per = (all + (int)share - 1) / (int)share, p0 = min((int)rank * per, all);
    r.pieces = row < a.rows && streams ? min(per, all - p0) : 0;
    r.at = head + p0 * VN;
    r.body = r.s + r.at;
    r.lo = rank == 0 ? 0 : r.at;
    r.hi = rank == share - 1 ? V : min(r.at + per * VN, tail);
    r.edge = t < head ? t : tail + t - head < V ? tail + t - head : -1;
    if (!streams || row >= a.rows || r.edge < r.lo || r.edge >= r.hi) r.edge = -1;
    return r;
  };
  static_assert(2 * (VN - 1) <= STREAM, "a thread per element outside of the pieces");
  // pieces i, i + STREAM, ...; beyond the last -inf, which adds nothing
  auto fetch = [&](const T* body, int pieces, int i) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * STREAM < pieces) next[u].load(body + (long long)(i + u * STREAM) * VN);
      else next[u].make([](int) { return -CUDART_INF_F; });
    }
  };
  Row coming = place(blockIdx.x / share);
  fetch(coming.body, coming.pieces, t);
  float weight = a.weights && blockIdx.x / share < a.rows ? a.weights[blockIdx.x / share] : 1.0f;
  float edge = coming.edge >= 0 ? rw_float(coming.s[coming.edge]) : -CUDART_INF_F;
  float2 ahead = make_float2(0.f, 0.f);
  if constexpr (!(DO & DT_LOSS))
    if (blockIdx.x / share < a.rows) ahead = a.stat[blockIdx.x / share];
  int buf = 0;
  for (long long row = blockIdx.x / share; row < a.rows; row += groups) {
    const Row r = coming;
    const float w = weight, mine = edge;
    coming = place(row + groups);
    edge = coming.edge >= 0 ? rw_float(coming.s[coming.edge]) : -CUDART_INF_F;
    if (a.weights && row + groups < a.rows) weight = a.weights[row + groups];
    T* const grad = DO & DT_GRAD ? (T*)a.grad + row * V : nullptr;
    float2 st = ahead;
    if constexpr (!(DO & DT_LOSS))
      if (row + groups < a.rows) ahead = a.stat[row + groups];
    auto zeros = [&] {
      if (streams)
        for (int j = r.lo + t; j < r.hi; j += STREAM) grad[j] = rw_to<T>(0.f);
    };
    if (w == 0.f || (!(DO & DT_LOSS) && st.y == 0.f)) {   // (a row without a teacher has left 0 there)
      if constexpr (DO & DT_LOSS) {
        if (t == 0 && rank == 0 && a.row_loss) a.row_loss[row] = 0.f;
        if (t == 0 && rank == 0 && a.stat) a.stat[row] = make_float2(0.f, 0.f);
      }
      if constexpr (DO & DT_GRAD) zeros();
      fetch(coming.body, coming.pieces, t);
      continue;
    }
    DtEntry* const e = (DtEntry*)dt_raw + buf * K;
    const float f = DO & DT_GRAD ? factor * w * (a.upstream && a.per_row ? a.upstream[row] : 1.0f) : 0.f;
    // this CTA's pieces, from those that have been fetched on: work(piece, its number); each one's place is taken by the one SPAN further at once,
    // behind the last ones by those of what comes next
    auto sweep = [&](const T* then, int then_pieces, auto&& work) {
      const int blocks = (r.pieces + SPAN - 1) / SPAN;
      const T* ahead = r.body + (long long)(t + SPAN) * VN;
      int i = t;
      for (int k = 2; k < blocks; ++k, i += SPAN, ahead += SPAN * VN)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const RwPiece<T, VN> v = next[u];
          next[u].load(ahead + u * STREAM * VN);
          work(v, i + u * STREAM);
        }
      if (blocks > 1) {   // the last ones may be fewer
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const RwPiece<T, VN> v = next[u];
          if (i + SPAN + u * STREAM < r.pieces) next[u].load(ahead + u * STREAM * VN);
          else next[u].make([](int) { return -CUDART_INF_F; });
          work(v, i + u * STREAM);
        }
        i += SPAN;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const RwPiece<T, VN> v = next[u];
        if (t + u * STREAM < then_pieces) next[u].load(then + (long long)(t + u * STREAM) * VN);
        else next[u].make([](int) { return -CUDART_INF_F; });
        if (i + u * STREAM < r.pieces) work(v, i + u * STREAM);
      }
    };
    // this thread's part of the gradient, from powers relative to m
    auto gradient = [&](float m, float total) {
      const float g = f * total;
      const uint64_t gg = dt_pair(g, g), mm = dt_pair(-m, -m);
      T* const out = grad + r.at;
      auto go = [&](auto aligned) {
        sweep(coming.body, coming.pieces, [&](const RwPiece<T, VN>& v, int i) {
          float x[VN];
#pragma unroll
          for (int j = 0; j < VN; j += 2) {
            dt_unpair(dt_fma2(dt_pair(v.at(j), v.at(j + 1)), cc, mm), x[j], x[j + 1]);
            dt_unpair(dt_mul2(gg, dt_pair(dt_exp2(x[j]), dt_exp2(x[j + 1]))), x[j], x[j + 1]);
          }
          RwPiece<T, VN> o;
          o.make([&](int j) { return x[j]; });
          T* const to = out + (long long)i * VN;
          if constexpr (decltype(aligned)::value) o.store(to);
          else
#pragma unroll
            for (int j = 0; j < VN; ++j) to[j] = o.one(j);
        });
      };
      if (((uintptr_t)out & 15) == 0) go(std::true_type());
      else go(std::false_type());
      if (r.edge >= 0) grad[r.edge] = rw_to<T>(g * dt_exp2(fmaf(mine, c, -m)));
    };
    if (!streams) {
      const bool any = dt_teacher(a, row, e, (int*)((DtEntry*)dt_raw + 2 * K));
      if (lane == 0) s_any[buf] = any;
    } else if constexpr (DO & DT_LOSS) {
      float m = LOWEST, total = 0.f;   // scaled maximum; sum of powers relative to it
      uint64_t mm = dt_pair(-m, -m), sum = dt_pair(0.f, 0.f);
      auto raise = [&](float to) {
        const float by = dt_exp2(m - to);
        sum = dt_mul2(sum, dt_pair(by, by));
        m = to;
        mm = dt_pair(-m, -m);
      };
      const bool again = DO & DT_GRAD;
      sweep(again ? r.body : coming.body, again ? r.pieces : coming.pieces, [&](const RwPiece<T, VN>& v, int) {
        const float most = rw_most(v) * c;
        if (most > m) raise(most);
#pragma unroll
        for (int j = 0; j < VN; j += 2) {
          float x, y;
          dt_unpair(dt_fma2(dt_pair(v.at(j), v.at(j + 1)), cc, mm), x, y);
          sum = dt_add2(sum, dt_pair(dt_exp2(x), dt_exp2(y)));
        }
      });
      if (r.edge >= 0) {
        if (mine * c > m) raise(mine * c);
        sum = dt_add2(sum, dt_pair(dt_exp2(fmaf(mine, c, -m)), 0.f));
      }
      float other;
      dt_unpair(sum, total, other);
      total += other;
      const float all = rw_warp_max(m);
      total = rw_warp_sum(total * dt_exp2(m - all));
      if (lane < (int)share) {
        const uint32_t to = rw_at_rank(&s_part[buf][rank * PARTS + warp], lane);
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(all), "f"(total) : "memory");
      }
    }
    if constexpr (!(DO & DT_LOSS))
      if (streams) gradient(st.x, st.y);
    if ((DO & DT_LOSS) && share > 1) rw_cluster_sync();
    else __syncthreads();
    if constexpr (DO == DT_LOSS)
      if (streams) { buf ^= 1; continue; }
    if constexpr (DO & DT_LOSS) {
      const int parts = (int)share * PARTS;
      constexpr int EACH = DL_MOST_SHARE * PARTS / 32;   // of a lane
      float2 x[EACH];
      float m = LOWEST, total = 0.f;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        x[i] = lane + 32 * i < parts ? s_part[buf][lane + 32 * i] : make_float2(LOWEST, 0.f);
        m = fmaxf(m, x[i].x);
      }
      m = rw_warp_max(m);
#pragma unroll
      for (int i = 0; i < EACH; ++i) total += x[i].y * dt_exp2(x[i].x - m);
      total = rw_warp_sum(total);
      m = m == LOWEST ? 0.f : m;   // (then all are -inf, and total is 0)
      st = make_float2(m, 1.0f / total);
      const bool any = s_any[buf];
      if (!streams) {
        if (rank == 0) {
          const float cross = any ? dt_cross(a, r.s, e, m) : 0.f;
          if (lane == 0) {
            const float loss = any ? w * a.temperature * a.temperature * DT_LN2 * (cross + log2f(total)) : 0.f;
            if (a.row_loss) a.row_loss[row] = loss;
            if (a.stat) a.stat[row] = any ? st : make_float2(0.f, 0.f);
            loss_sum += loss;
            weight_sum += any ? w : 0.f;
          }
        }
      } else if constexpr (DO & DT_GRAD) {
        if (any) gradient(st.x, st.y);
        else {
          zeros();
          fetch(coming.body, coming.pieces, t);
        }
        asm volatile("bar.sync 1, %0;" ::"n"(STREAM) : "memory");   // the streaming warps
        if (any) dt_columns(a, r.s, grad, e, f, st.y, st.x, t, STREAM, r.lo, r.hi);
      }
    } else if (streams) {
      dt_columns(a, r.s, grad, e, f, st.y, st.x, t, STREAM, r.lo, r.hi);
    }
    buf ^= 1;
  }
  if constexpr (DO & DT_LOSS)
    if (t == STREAM && rank == 0) a.part[blockIdx.x / share] = make_double2(loss_sum, weight_sum);
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
__global__ void __launch_bounds__(NT) k_distill_total(const double2* __restrict__ part, int n, int mean, float scale, float* loss, float* inv) {
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
    if (loss) loss[0] = (float)(mean ? (w != 0.0 ? l / w : 0.0) * scale : l * scale);
    if (inv) inv[0] = w != 0.0 ? (float)(1.0 / w) : 0.f;
  }
}

// Rows' groups of a call, one CTA or a cluster each, which is also the number of its partial sums
// A call's form.  Threads that stream through a long row: few for short ones, so that more rows' latencies lie side by side, many for long ones, so
// that (loss and gradient) the rows being worked on stay in the L2 cache between their two passes.  share: CTAs that share a row, until all have work.
struct DtForm { int stream, share, ctas; };
static DtForm dt_form(long long rows, int vocab, int type_bytes) {
  if (vocab <= DT_WARP_VOCAB) {
    const long long n = (rows + DT_WARP_THREADS / 32 - 1) / (DT_WARP_THREADS / 32), most = (long long)sm_count() * 8;
    return {0, 1, (int)(n < most ? n : most)};
  }
  const long long bytes = (long long)vocab * type_bytes;
  const int stream = bytes <= 16384 ? 128 : bytes <= 131072 ? 256 : 512;
  const long long most = (long long)sm_count() * dl_ctas(stream);
  int share = 1;
  while (share < DL_MOST_SHARE && bytes >= share * 2 * 16384 && rows * share * 2 <= most) share *= 2;
  return {stream, share, (int)(rows < most / share ? rows : most / share)};
}
static int dt_weight_ctas(long long rows) { return (int)(rows < 64 * NT ? (rows + NT - 1) / NT : 64); }
template <class T, int DO>
static int dt_run(const DtArgs& a, const DtForm& form, cudaStream_t s) {
  const size_t slots = (size_t)4 * dt_slots(a.top), entries = sizeof(DtEntry) * a.top;
#define DT_LONG(STREAM)                                                                                                    \
  {                                                                                                                        \
    launch_clusters(k_distill_long<T, DO, STREAM>, form.ctas * form.share, STREAM + 32, form.share, 2 * entries + slots, s, a); \
    return launch_status();                                                                                                \
  }
  if (form.stream == 128) DT_LONG(128)
  if (form.stream == 256) DT_LONG(256)
  if (form.stream == 512) DT_LONG(512)
#undef DT_LONG
  const size_t smem = (entries + slots) * (DT_WARP_THREADS / 32);
  static bool configured[PYLO_MAX_DEVICES] = {};
  if (smem > 48 * 1024)
    if (int rc = allow_dynamic_smem(k_distill_short<T, DO>, (int)(DT_WARP_THREADS / 32 * (sizeof(DtEntry) * DT_MOST_K + 4 * dt_slots(DT_MOST_K))), configured)) return rc;
  launch(k_distill_short<T, DO>, form.ctas, DT_WARP_THREADS, smem, s, a);
  return launch_status();
}
template <int DO>
static int dt_any_type(const DtArgs& a, int type, const DtForm& form, cudaStream_t s) {
  return type == PYLO_FP32 ? dt_run<float, DO>(a, form, s) : type == PYLO_BF16 ? dt_run<__nv_bfloat16, DO>(a, form, s) : dt_run<__half, DO>(a, form, s);
}
static bool dt_good(const pylo_distill* d) {
  return d && d->rows >= 0 && d->rows <= (1ll << 40) && d->vocab > 0 && d->vocab <= (1 << 30) && d->top > 0 && d->top <= DT_MOST_K && rw_type(d->type) &&
         rw_type(d->teacher_type) && (d->ids_bytes == 4 || d->ids_bytes == 8) && d->temperature > 0.f && (d->rows == 0 || (d->logits && d->teacher && d->ids)) &&
         d->stride >= d->vocab && (uintptr_t)d->logits % rw_bytes(d->type) == 0;
}
static DtArgs dt_args(const pylo_distill* d) {
  DtArgs a = {};
  a.logits = d->logits; a.teacher = d->teacher; a.ids = d->ids; a.weights = d->weights;
  a.row_loss = d->row_loss; a.stat = (float2*)d->stat; a.grad = d->grad; a.upstream = d->upstream; a.per_row = d->reduction == PYLO_REDUCE_NONE;
  a.rows = d->rows; a.stride = d->stride; a.vocab = d->vocab; a.top = d->top; a.teacher_type = d->teacher_type; a.wide_ids = d->ids_bytes == 8;
  a.c = (float)(DT_LOG2E / d->temperature); a.temperature = d->temperature; a.scale = 1.0f;
  return a;
}

extern "C" {

int64_t pylo_b200_layer_norm_workspace(int64_t rows, int width) {
  if (rows <= 0 || width <= 0 || width > LN_MOST) return 0;
  return (int64_t)ln_ctas(rows, width, LN_BACKWARD) * 2 * width;
}

int pylo_b200_layer_norm(const pylo_norm* n, void* stream) {
  CHECK_ARG(n && n->rows >= 0 && n->width > 0 && n->width <= LN_MOST && rw_type(n->type) && n->eps >= 0.f);
  if (n->rows == 0) return 0;
  CHECK_ARG(n->x && n->y && (n->mean == nullptr) == (n->rstd == nullptr) && (n->weight || !n->bias) && n->x_stride >= 0);
  LnArgs a = {};
  a.x = n->x; a.weight = n->weight; a.bias = n->bias; a.y = n->y; a.mean = n->mean; a.rstd = n->rstd;
  a.rows = n->rows; a.x_stride = n->x_stride; a.width = n->width; a.eps = n->eps;
  return ln_any(a, n->type, n->weight_type, false, (cudaStream_t)stream);
}

int pylo_b200_layer_norm_backward(const pylo_norm* n, void* stream) {
  CHECK_ARG(n && n->rows >= 0 && n->width > 0 && n->width <= LN_MOST && rw_type(n->type));
  cudaStream_t s = (cudaStream_t)stream;
  const bool columns = n->dweight || n->dbias;
  const int ctas = n->rows ? ln_ctas(n->rows, n->width, LN_BACKWARD) : 0;
  CHECK_ARG(!columns || ctas == 0 || (n->work && n->work_floats >= (int64_t)ctas * 2 * n->width));
  if (ctas) {
    CHECK_ARG(n->x && n->dy && n->mean && n->rstd && n->x_stride >= 0 && n->dy_stride >= 0);
    LnArgs a = {};
    a.x = n->x; a.dy = n->dy; a.weight = n->weight; a.y = n->dx; a.mean = n->mean; a.rstd = n->rstd; a.part = columns ? n->work : nullptr;
    a.rows = n->rows; a.x_stride = n->x_stride; a.dy_stride = n->dy_stride; a.width = n->width;
    if (n->dx || columns)
      if (int rc = ln_any(a, n->type, n->weight_type, true, s)) return rc;
  }
  if (columns) {
    const dim3 grid((n->width + 31) / 32, n->dbias ? 2 : 1);
    if (n->weight_type == PYLO_FP32) launch(k_layer_norm_columns<float>, grid, NT, 0, s, n->work, ctas, n->width, (float*)n->dweight, (float*)n->dbias);
    else if (n->weight_type == PYLO_BF16) launch(k_layer_norm_columns<__nv_bfloat16>, grid, NT, 0, s, n->work, ctas, n->width, (__nv_bfloat16*)n->dweight, (__nv_bfloat16*)n->dbias);
    else if (n->weight_type == PYLO_FP16) launch(k_layer_norm_columns<__half>, grid, NT, 0, s, n->work, ctas, n->width, (__half*)n->dweight, (__half*)n->dbias);
    else return -1;
  }
  return launch_status();
}

int64_t pylo_b200_distill_workspace(int64_t rows, int vocab) {
  if (rows <= 0 || vocab <= 0) return 16;
  const long long most = (long long)sm_count() * 8;   // groups of rows of whatever form
  return 16 * (int64_t)(rows < most ? rows : most) + 8 * (int64_t)dt_weight_ctas(rows);
}

int pylo_b200_distill(const pylo_distill* d, int what, void* stream) {
  CHECK_ARG(dt_good(d) && (what == PYLO_DISTILL_LOSS || what == PYLO_DISTILL_GRAD || what == (PYLO_DISTILL_LOSS | PYLO_DISTILL_GRAD)));
  cudaStream_t s = (cudaStream_t)stream;
  const bool loss = what & PYLO_DISTILL_LOSS, grad = what & PYLO_DISTILL_GRAD, mean = d->reduction == PYLO_REDUCE_MEAN;
  CHECK_ARG(!loss || (d->work && (uintptr_t)d->work % 16 == 0 && d->work_bytes >= pylo_b200_distill_workspace(d->rows, d->vocab)));
  CHECK_ARG(!grad || d->rows == 0 || (d->grad && (uintptr_t)d->grad % rw_bytes(d->type) == 0));
  CHECK_ARG(!grad || loss || d->rows == 0 || (d->stat && (!mean || d->inv)));
  DtArgs a = dt_args(d);
  const DtForm form = d->rows ? dt_form(d->rows, d->vocab, (int)rw_bytes(d->type)) : DtForm{};
  if (d->rows) {
    a.part = (double2*)d->work;
    if (grad) a.scale = d->scale;
    if (grad && mean && loss) {
      double* const sums = (double*)((char*)d->work + 16 * (size_t)form.ctas);
      a.weight_sums = sums;
      a.n_sums = dt_weight_ctas(d->rows);
      launch(k_distill_weights, a.n_sums, NT, 0, s, a, sums);
    } else if (grad && mean) a.inv = d->inv;
    const int rc = !grad ? dt_any_type<DT_LOSS>(a, d->type, form, s) : loss ? dt_any_type<DT_LOSS | DT_GRAD>(a, d->type, form, s) : dt_any_type<DT_GRAD>(a, d->type, form, s);
    if (rc) return rc;
  }
  if (loss && d->reduction != PYLO_REDUCE_NONE)
    launch(k_distill_total, 1, NT, 0, s, (const double2*)d->work, form.ctas, (int)mean, 1.0f, d->loss, d->inv);
  return launch_status();
}

}  // extern "C"
