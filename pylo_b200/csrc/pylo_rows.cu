// Operators on the rows of a matrix that a model's training step needs beside its optimizer: layer norm with its gradients, and the
// loss of a distillation from a teacher's largest logits with its gradient.
//
// Both read and write whole rows once and compute a few operations per element: the memory's bandwidth bounds them, and a small call
// the latency of its launches.  A row belongs to a warp where it is short, else to a CTA; the CTAs are as many as run at once and go
// from row to row.  Everything is computed in fp32 from the elements' own type and rounded once, where it is stored.
#include <cuda_bf16.h>

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

// the largest of some pieces' elements that are numbers
template <class T, int N, int U>
__device__ __forceinline__ float rw_most(const RwPiece<T, N> (&v)[U]) {
  if constexpr (std::is_same_v<T, float>) {
    float most = v[0].at(0);
#pragma unroll
    for (int j = 1; j < N * U; ++j) most = fmaxf(most, v[j / N].at(j % N));
    return most;
  } else {   // two at a time
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    T2 most = *reinterpret_cast<const T2*>(&v[0].w[0]);
#pragma unroll
    for (int j = 1; j < 4 * U; ++j) most = __hmax2(most, *reinterpret_cast<const T2*>(&v[j / 4].w[j % 4]));
    return fmaxf(rw_float(most.x), rw_float(most.y));
  }
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
// A teacher's K entries by a warp: ids (-1 for padding), probabilities and their logarithms to base 2; whether there are any
__device__ __forceinline__ bool dt_teacher(const DtArgs& a, long long row, int* id, float* p, float* lp) {
  const int lane = threadIdx.x & 31, K = a.top;
  float most = -CUDART_INF_F, sum = 0.f;
  bool any = false;
  for (int k = lane; k < K; k += 32) {
    id[k] = dt_id(a, row * K + k);
    const float z = id[k] >= 0 ? dt_any(a.teacher, a.teacher_type, row * K + k) * a.c : -CUDART_INF_F;
    lp[k] = z;
    most = fmaxf(most, z);
    any |= !(z == -CUDART_INF_F);
  }
  any = __any_sync(0xffffffffu, any);
  if (!any) return false;
  most = rw_warp_max(most);
  for (int k = lane; k < K; k += 32) sum += dt_exp2(lp[k] - most);
  const float log_sum = log2f(rw_warp_sum(sum));
  for (int k = lane; k < K; k += 32) {
    lp[k] = lp[k] - most - log_sum;
    p[k] = dt_exp2(lp[k]);
  }
  __syncwarp();
  return true;
}
// The loss of a row to base 2, without the student's sum: sum of p (log p - s), by a warp
template <class T>
__device__ __forceinline__ float dt_cross(const DtArgs& a, const T* s, const int* id, const float* p, const float* lp, float m) {
  float sum = 0.f;
  for (int k = threadIdx.x & 31; k < a.top; k += 32)
    if (!(p[k] == 0.f)) sum = fmaf(p[k], lp[k] - fmaf(rw_float(s[id[k] < 0 ? 0 : id[k]]), a.c, -m), sum);   // (p > 0 has an id)
  return rw_warp_sum(sum);
}
// The columns of the teacher's entries, once more; a class that several entries name takes them all, in their order
template <class T>
__device__ __forceinline__ void dt_columns(const DtArgs& a, const T* s, T* grad, const int* id, const float* p, float f, float total, float m, int t, int threads) {
  for (int k = t; k < a.top; k += threads) {
    const int at = id[k];
    if (at < 0) continue;
    const float v = rw_float(s[at]);
    float sum = 0.f;
    bool first = true;   // of the entries with this id
    for (int j = 0; j < a.top; ++j)
      if (id[j] == at) {
        first &= j >= k;
        sum += p[j];
      }
    if (first) grad[at] = rw_to<T>(f * (total * dt_exp2(fmaf(v, a.c, -m)) - sum));
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
  int* const id = (int*)dt_raw + (size_t)group * 3 * a.top;
  float* const p = (float*)(id + a.top);
  float* const lp = p + a.top;
  const float factor = DO & DT_GRAD ? dt_factor(a) : 0.f;
  double loss_sum = 0.0, weight_sum = 0.0;
  for (long long row = (long long)blockIdx.x * GROUPS + group; row < a.rows; row += (long long)gridDim.x * GROUPS) {
    const float weight = a.weights ? a.weights[row] : 1.0f;
    const bool any = weight != 0.f && dt_teacher(a, row, id, p, lp);
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
      const float cross = dt_cross(a, r.s, id, p, lp, m);
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
      dt_columns(a, r.s, grad, id, p, f, total, m, t, 32);
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

// Long rows: a CTA each.  Eight warps stream through the logits, each thread with four pieces of 16 bytes on their way while it works on four
// others, the next row's first ones behind this row's last; a ninth warp has the teacher's entries and the row's loss, so that nothing of the stream
// waits for them.  One barrier per row and pass: what the warps leave for one another lies in two buffers that take turns.
#define DL_STREAM 256
#define DL_THREADS (DL_STREAM + 32)
#define DL_CTAS 4   // of an SM
#define DL_U 4
template <class T, int DO>
__global__ void __launch_bounds__(DL_THREADS, DL_CTAS) k_distill_long(const DtArgs a) {
  pdl_begin();
  extern __shared__ __align__(16) unsigned char dt_raw[];
  __shared__ float2 s_part[2][DL_STREAM / 32];
  __shared__ int s_any[2];
  constexpr int VN = RW_VEC<T>, U = DL_U, SPAN = U * DL_STREAM;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, K = a.top, V = a.vocab;
  const bool streams = warp < DL_STREAM / 32;
  const float c = a.c, factor = DO & DT_GRAD ? dt_factor(a) : 0.f;
  double loss_sum = 0.0, weight_sum = 0.0;
  RwPiece<T, VN> next[U];
  const T* const logits = (const T*)a.logits;
  // pieces i, i + DL_STREAM, ... of a row; beyond its last -inf, which adds nothing
  auto fetch = [&](const T* body, int pieces, int i) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * DL_STREAM < pieces) next[u].load(body + (long long)(i + u * DL_STREAM) * VN);
      else next[u].make([](int) { return -CUDART_INF_F; });
    }
  };
  auto place = [&](long long row) { return DtRow<T>(logits + (row < a.rows ? row : 0) * a.stride, streams && row < a.rows ? V : 0, t); };
  auto outside = [&](const DtRow<T>& r) { return streams && r.edge >= 0 ? rw_float(r.s[r.edge]) : -CUDART_INF_F; };
  DtRow<T> coming = place(blockIdx.x);
  fetch(coming.s + coming.head, coming.pieces, t);
  float weight = a.weights && blockIdx.x < a.rows ? a.weights[blockIdx.x] : 1.0f, edge = outside(coming);
  int buf = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const long long row1 = row + gridDim.x;
    const DtRow<T> r = coming;
    const float w = weight, mine = edge;
    coming = place(row1);
    edge = outside(coming);
    if (a.weights && row1 < a.rows) weight = a.weights[row1];
    const T* const body = r.s + r.head;
    T* const grad = DO & DT_GRAD ? (T*)a.grad + row * V : nullptr;
    float2 st = make_float2(0.f, 0.f);
    if constexpr (!(DO & DT_LOSS)) st = a.stat[row];
    auto zeros = [&] {
      if (streams)
        for (int j = t; j < V; j += DL_STREAM) grad[j] = rw_to<T>(0.f);
    };
    if (w == 0.f || (!(DO & DT_LOSS) && st.y == 0.f)) {   // (a row without a teacher has left 0 there)
      if constexpr (DO & DT_LOSS) {
        if (t == 0 && a.row_loss) a.row_loss[row] = 0.f;
        if (t == 0 && a.stat) a.stat[row] = make_float2(0.f, 0.f);
      }
      if constexpr (DO & DT_GRAD) zeros();
      fetch(coming.s + coming.head, coming.pieces, t);
      continue;
    }
    int* const id = (int*)dt_raw + (size_t)buf * 3 * K;
    float* const p = (float*)(id + K);
    float* const lp = p + K;
    const float f = DO & DT_GRAD ? factor * w * (a.upstream && a.per_row ? a.upstream[row] : 1.0f) : 0.f;
    // a row's pieces, from those that have been fetched on; behind the last, those of what comes next are
    auto sweep = [&](const T* then, int then_pieces, auto&& work) {
      int i = t;
      do {
        RwPiece<T, VN> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = next[u];
        const bool last = i + SPAN >= r.pieces;
        fetch(last ? then : body, last ? then_pieces : r.pieces, last ? t : i + SPAN);
        work(v, i);
      } while ((i += SPAN) < r.pieces);
    };
    // this thread's part of the gradient, from powers relative to m
    auto gradient = [&](float m, float total) {
      const float g = f * total;
      T* const out = grad + r.head;
      const bool aligned = ((uintptr_t)out & 15) == 0;
      sweep(coming.s + coming.head, coming.pieces, [&](const RwPiece<T, VN> (&v)[U], int i) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (i + u * DL_STREAM < r.pieces) {
            RwPiece<T, VN> o;
            o.make([&](int j) { return g * dt_exp2(fmaf(v[u].at(j), c, -m)); });
            T* const to = out + (long long)(i + u * DL_STREAM) * VN;
            if (aligned) o.store(to);
            else
#pragma unroll
              for (int j = 0; j < VN; ++j) to[j] = o.one(j);
          }
      });
      if (r.edge >= 0) grad[r.edge] = rw_to<T>(g * dt_exp2(fmaf(mine, c, -m)));
    };
    if (!streams) {
      const bool any = dt_teacher(a, row, id, p, lp);
      if (lane == 0) s_any[buf] = any;
    } else if constexpr (DO & DT_LOSS) {
      float m = -CUDART_INF_F, total = 0.f;   // scaled maximum; sum of powers relative to it
      const bool again = DO & DT_GRAD;
      sweep(again ? body : coming.s + coming.head, again ? r.pieces : coming.pieces, [&](const RwPiece<T, VN> (&v)[U], int) {
        const float up = fmaxf(m, rw_most(v) * c), ref = up == -CUDART_INF_F ? 0.f : up;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < U * VN; ++j) sum[j & 1] += dt_exp2(fmaf(v[j / VN].at(j % VN), c, -ref));
        total = fmaf(total, dt_exp2(m - ref), sum[0] + sum[1]);
        m = up;
      });
      if (r.edge >= 0) {
        const float up = fmaxf(m, mine * c), ref = up == -CUDART_INF_F ? 0.f : up;
        total = fmaf(total, dt_exp2(m - ref), dt_exp2(fmaf(mine, c, -ref)));
        m = up;
      }
      const float all = rw_warp_max(m), ref = all == -CUDART_INF_F ? 0.f : all;
      total = rw_warp_sum(total * dt_exp2(m - ref));
      if (lane == 0) s_part[buf][warp] = make_float2(all, total);
    }
    if constexpr (!(DO & DT_LOSS))
      if (streams) gradient(st.x, st.y);
    __syncthreads();
    if constexpr (DO & DT_LOSS) {
      float m = -CUDART_INF_F, total = 0.f;
#pragma unroll
      for (int i = 0; i < DL_STREAM / 32; ++i) m = fmaxf(m, s_part[buf][i].x);
      m = m == -CUDART_INF_F ? 0.f : m;
#pragma unroll
      for (int i = 0; i < DL_STREAM / 32; ++i) {
        const float2 q = s_part[buf][i];
        total += q.y * dt_exp2((q.x == -CUDART_INF_F ? 0.f : q.x) - m);
      }
      st = make_float2(m, 1.0f / total);
      const bool any = s_any[buf];
      if (!streams) {
        const float cross = any ? dt_cross(a, r.s, id, p, lp, m) : 0.f;
        if (lane == 0) {
          const float loss = any ? w * a.temperature * a.temperature * DT_LN2 * (cross + log2f(total)) : 0.f;
          if (a.row_loss) a.row_loss[row] = loss;
          if (a.stat) a.stat[row] = any ? st : make_float2(0.f, 0.f);
          loss_sum += loss;
          weight_sum += any ? w : 0.f;
        }
      } else if constexpr (DO & DT_GRAD) {
        if (any) gradient(st.x, st.y);
        else {
          zeros();
          fetch(coming.s + coming.head, coming.pieces, t);
        }
        asm volatile("bar.sync 1, %0;" ::"n"(DL_STREAM) : "memory");   // the streaming warps
        if (any) dt_columns(a, r.s, grad, id, p, f, st.y, st.x, t, DL_STREAM);
      }
    } else if (streams) {
      dt_columns(a, r.s, grad, id, p, f, st.y, st.x, t, DL_STREAM);
    }
    buf ^= 1;
  }
  if constexpr (DO & DT_LOSS)
    if (t == DL_STREAM) a.part[blockIdx.x] = make_double2(loss_sum, weight_sum);
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

// CTAs of a call, which is also the number of its partial sums
static int dt_ctas(long long rows, int vocab) {
  const bool is_short = vocab <= DT_WARP_VOCAB;
  const long long n = is_short ? (rows + DT_WARP_THREADS / 32 - 1) / (DT_WARP_THREADS / 32) : rows, most = (long long)sm_count() * (is_short ? 8 : DL_CTAS);
  return (int)(n < most ? n : most);
}
static int dt_weight_ctas(long long rows) { return (int)(rows < 64 * NT ? (rows + NT - 1) / NT : 64); }
template <class T, int DO>
static int dt_run(const DtArgs& a, cudaStream_t s) {
  const int ctas = dt_ctas(a.rows, a.vocab);
  if (a.vocab <= DT_WARP_VOCAB) launch(k_distill_short<T, DO>, ctas, DT_WARP_THREADS, (size_t)12 * a.top * (DT_WARP_THREADS / 32), s, a);
  else launch(k_distill_long<T, DO>, ctas, DL_THREADS, (size_t)24 * a.top, s, a);
  return launch_status();
}
template <int DO>
static int dt_any_type(const DtArgs& a, int type, cudaStream_t s) {
  return type == PYLO_FP32 ? dt_run<float, DO>(a, s) : type == PYLO_BF16 ? dt_run<__nv_bfloat16, DO>(a, s) : dt_run<__half, DO>(a, s);
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
  return 16 * (int64_t)dt_ctas(rows, vocab) + 8 * (int64_t)dt_weight_ctas(rows);
}

int pylo_b200_distill(const pylo_distill* d, int what, void* stream) {
  CHECK_ARG(dt_good(d) && (what == PYLO_DISTILL_LOSS || what == PYLO_DISTILL_GRAD || what == (PYLO_DISTILL_LOSS | PYLO_DISTILL_GRAD)));
  cudaStream_t s = (cudaStream_t)stream;
  const bool loss = what & PYLO_DISTILL_LOSS, grad = what & PYLO_DISTILL_GRAD, mean = d->reduction == PYLO_REDUCE_MEAN;
  CHECK_ARG(!loss || (d->work && (uintptr_t)d->work % 16 == 0 && d->work_bytes >= pylo_b200_distill_workspace(d->rows, d->vocab)));
  CHECK_ARG(!grad || d->rows == 0 || (d->grad && (uintptr_t)d->grad % rw_bytes(d->type) == 0));
  CHECK_ARG(!grad || loss || d->rows == 0 || (d->stat && (!mean || d->inv)));
  DtArgs a = dt_args(d);
  if (d->rows) {
    a.part = (double2*)d->work;
    if (grad) a.scale = d->scale;
    if (grad && mean && loss) {
      double* const sums = (double*)((char*)d->work + 16 * (size_t)dt_ctas(d->rows, d->vocab));
      a.weight_sums = sums;
      a.n_sums = dt_weight_ctas(d->rows);
      launch(k_distill_weights, a.n_sums, NT, 0, s, a, sums);
    } else if (grad && mean) a.inv = d->inv;
    const int rc = !grad ? dt_any_type<DT_LOSS>(a, d->type, s) : loss ? dt_any_type<DT_LOSS | DT_GRAD>(a, d->type, s) : dt_any_type<DT_GRAD>(a, d->type, s);
    if (rc) return rc;
  }
  if (loss && d->reduction != PYLO_REDUCE_NONE)
    launch(k_distill_total, 1, NT, 0, s, (const double2*)d->work, d->rows ? dt_ctas(d->rows, d->vocab) : 0, (int)mean, 1.0f, d->loss, d->inv);
  return launch_status();
}

}  // extern "C"
