// Matrix products in 8-bit integers: y[m][n] = xs[m] ws[n] sum_k cx[m][k] cw[n][k], codes -127 .. 127, the sum exact in 32-bit integers
// (K up to 32,768), rounded once as it is scaled.  And what stands in front of them: a row of activations quantised, its scale
// the largest magnitude / 127, as it is, behind an RMS norm, or behind the gate of a feed-forward.
// (reference: the nn.Linear calls of model/llama.py:175,184,195 are the same products in the model's precision; it has no form in fewer bits)
//
// The weight is laid out once, in pieces of 1 KiB that are an operand of v_mfma_i32_16x16x64_i8 in lane order:
//   wt[row tile rt][piece kc][lane = 16 g + r][16 bytes] = cw[16 rt + r][64 kc + 16 g + {0 .. 15}]
// rows padded to a multiple of 16 and K to KP, a multiple of 256 and at least 512, with zeros.  Activations are plain rows, KP bytes apart;
// what lies in them beyond K is multiplied with zeros.
#include "common.h"
#include "lds_loads.h"

typedef __attribute__((__vector_size__(4 * sizeof(int)))) int i32x4;

#define INT8_TINY 0x1p-100f
#define INT8_MAX_K 32768  // (a row in the registers of a workgroup)

// ------------------------------------------------------------------------------------------------------------------------------------
// Rows into codes.  Bound by memory: a row is read once and kept in registers (up to 16 values a thread) between its maximum and its codes.
//   SRC 0: x;  1: w * (r * rsqrt(mean(r^2) + eps)), r = resid + x rounded to T, which is stored if resid_out;  2: silu(x[:K]) * x[K:]
// all in 32-bit and not rounded before the codes.  A row with an infinity or no number has the scale "no number": its products are none.
struct Int8RowsParams {
  int8_t* codes;   // [rows][kp]
  float* scales;   // [rows]
  const void *x, *resid, *weight;
  void* resid_out;
  int x_stride, k, kp;
  float eps;
};

template <typename T, int SRC, int V, int CHUNKS>
__global__ void int8_rows_kernel(const Int8RowsParams p) {
  typedef T vec_t __attribute__((ext_vector_type(V)));
  __shared__ float scratch[16], scratch2[16];
  const size_t row = blockIdx.x;
  const T* x = (const T*)p.x + row * p.x_stride;
  const T* resid = SRC == 1 && p.resid ? (const T*)p.resid + row * p.k : nullptr;
  const int pieces = p.k / V;
  float val[CHUNKS][V];
  float square = 0.f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = threadIdx.x + c * blockDim.x;
    if (i >= pieces) {
#pragma unroll
      for (int e = 0; e < V; ++e) val[c][e] = 0.f;
      continue;
    }
    vec_t a = reinterpret_cast<const vec_t*>(x)[i];
    if constexpr (SRC == 1) {
      if (resid) {
        const vec_t b = reinterpret_cast<const vec_t*>(resid)[i];
#pragma unroll
        for (int e = 0; e < V; ++e) a[e] = from_f<T>(to_f((T)b[e]) + to_f((T)a[e]));
      }
      if (p.resid_out) reinterpret_cast<vec_t*>((T*)p.resid_out + row * p.k)[i] = a;
    }
    if constexpr (SRC == 2) {
      const vec_t up = reinterpret_cast<const vec_t*>(x + p.k)[i];
#pragma unroll
      for (int e = 0; e < V; ++e) val[c][e] = silu_of(to_f((T)a[e])) * to_f((T)up[e]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        val[c][e] = to_f((T)a[e]);
        if constexpr (SRC == 1) square += val[c][e] * val[c][e];
      }
    }
  }
  if constexpr (SRC == 1) {
    const float inv = rsqrtf(block_sum(square, scratch) / (float)p.k + p.eps);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int i = threadIdx.x + c * blockDim.x;
      if (i >= pieces) continue;
      const vec_t w = reinterpret_cast<const vec_t*>(p.weight)[i];
#pragma unroll
      for (int e = 0; e < V; ++e) val[c][e] = to_f((T)w[e]) * (val[c][e] * inv);
    }
  }
  float most = 0.f;
  int bad = 0;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      most = fmaxf(most, fabsf(val[c][e]));
      bad |= !(fabsf(val[c][e]) < INFINITY);
    }
  most = block_max(bad ? INFINITY : most, scratch2);
  const bool fine = most < INFINITY, some = fine && most >= INT8_TINY;
  const float inverse = some ? 127.f / most : 0.f;
  typedef int8_t code_t __attribute__((ext_vector_type(V)));
  code_t* to = reinterpret_cast<code_t*>(p.codes + row * p.kp);
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = threadIdx.x + c * blockDim.x;
    if (i >= pieces) continue;
    code_t o;
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = some ? (int8_t)fminf(fmaxf(rintf(val[c][e] * inverse), -127.f), 127.f) : (int8_t)0;
    to[i] = o;
  }
  if (threadIdx.x == 0) p.scales[row] = fine ? (some ? most / 127.f : 0.f) : NAN;
}

template <typename T, int SRC, int V>
static int launch_rows(const Int8RowsParams& p, int rows, hipStream_t stream) {
  const int pieces = p.k / V;
  // (a wave for little, 1,024 threads for the widest rows: as many pieces a thread as there must be)
  const int chunks = (pieces + 1023) / 1024;
  int threads = (pieces + chunks - 1) / chunks;
  threads = (threads + 63) / 64 * 64;
  if (chunks == 1)
    int8_rows_kernel<T, SRC, V, 1><<<rows, threads, 0, stream>>>(p);
  else if (chunks == 2)
    int8_rows_kernel<T, SRC, V, 2><<<rows, threads, 0, stream>>>(p);
  else if (chunks <= 4)
    int8_rows_kernel<T, SRC, V, 4><<<rows, threads, 0, stream>>>(p);
  else if (chunks <= 8)
    int8_rows_kernel<T, SRC, V, 8><<<rows, threads, 0, stream>>>(p);
  else if constexpr (V == 1)
    int8_rows_kernel<T, SRC, V, INT8_MAX_K / 1024><<<rows, threads, 0, stream>>>(p);
  else
    return NS_ERR_UNSUPPORTED;
  return ns_launch_status();
}
template <typename T>
static int launch_rows(const Int8RowsParams& p, int rows, int src, hipStream_t stream) {
  // pieces of 16 bytes where the rows allow them, of one value otherwise
  constexpr int V = 16 / sizeof(T);
  const bool wide = p.k % V == 0 && p.x_stride % V == 0 && !(((uintptr_t)p.x | (uintptr_t)p.resid | (uintptr_t)p.resid_out | (uintptr_t)p.weight) & 15);
  switch (src) {
    case 0: return wide ? launch_rows<T, 0, V>(p, rows, stream) : launch_rows<T, 0, 1>(p, rows, stream);
    case 1: return wide ? launch_rows<T, 1, V>(p, rows, stream) : launch_rows<T, 1, 1>(p, rows, stream);
    case 2: return wide ? launch_rows<T, 2, V>(p, rows, stream) : launch_rows<T, 2, 1>(p, rows, stream);
  }
  return NS_ERR_BAD_ARG;
}

extern "C" int ns_int8_rows(void* codes, float* scales, const void* x, int x_stride, const void* resid, void* resid_out, const void* weight, float eps, int rows, int k,
                            int kp, int src, int dtype, hipStream_t stream) {
  if (rows < 0 || k <= 0 || kp < k || k > INT8_MAX_K || src < 0 || src > 2 || x_stride < (src == 2 ? 2 * k : k) || (src == 1 && !weight)) return NS_ERR_BAD_ARG;
  if (((uintptr_t)codes & 15) || kp % 16) return NS_ERR_UNSUPPORTED;
  if (rows == 0) return NS_OK;
  const Int8RowsParams p{(int8_t*)codes, scales, x, resid, weight, resid_out, x_stride, k, kp, eps};
  if (dtype == NS_DTYPE_F32) return launch_rows<float>(p, rows, src, stream);
  if (dtype == NS_DTYPE_BF16) return launch_rows<bf16_t>(p, rows, src, stream);
  return NS_ERR_UNSUPPORTED;
}

// ------------------------------------------------------------------------------------------------------------------------------------
// Up to 16 rows: the weight streams once, a workgroup a tile of 16 of its rows, its waves the pieces of K in turn; their sums meet in LDS.
struct Int8Params {
  void* out;
  const int8_t *x, *w;
  const float *xs, *ws;
  int M, N, KP, out_stride, ranges;
};

template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void gemm_int8_few_kernel(const Int8Params p) {
  __shared__ i32x4 sums[WAVES][64];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), r = lane % 16, g = lane / 16;
  const int m0 = blockIdx.y * 16, pieces = p.KP / 64;
  const i32x4* w = reinterpret_cast<const i32x4*>(p.w + (size_t)blockIdx.x * 16 * p.KP) + lane;
  const i32x4* x = reinterpret_cast<const i32x4*>(p.x + (size_t)min(m0 + r, p.M - 1) * p.KP) + g;
  i32x4 acc = {0, 0, 0, 0};
#pragma unroll 4
  for (int kc = wave; kc < pieces; kc += WAVES) {
    const i32x4 a = __builtin_nontemporal_load(w + (size_t)kc * 64), b = x[kc * 4];
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc, 0, 0, 0);
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int v = 1; v < WAVES; ++v) acc += sums[v][lane];
  const int row = m0 + r, col = blockIdx.x * 16 + 4 * g;
  if (row >= p.M) return;
  const float xs = p.xs[row];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < p.N) ((T*)p.out)[(size_t)row * p.out_stride + col + e] = from_f<T>((float)acc[e] * xs * p.ws[col + e]);
}

extern "C" int ns_gemm_int8(void* out, const void* x, const float* xs, const void* w, const float* ws, int M, int N, int KP, int out_stride, int dtype, hipStream_t stream) {
  if (M < 0 || N <= 0 || KP < 512 || KP % 256 || KP > INT8_MAX_K || out_stride < N) return NS_ERR_BAD_ARG;
  if ((((uintptr_t)x | (uintptr_t)w) & 15) || (M + 15) / 16 > 65535) return NS_ERR_UNSUPPORTED;
  if (M == 0) return NS_OK;
  const Int8Params p{out, (const int8_t*)x, (const int8_t*)w, xs, ws, M, N, KP, out_stride, 1};
  const dim3 grid((N + 15) / 16, (M + 15) / 16);
  if (dtype == NS_DTYPE_F32)
    gemm_int8_few_kernel<float, 8><<<grid, 512, 0, stream>>>(p);
  else if (dtype == NS_DTYPE_BF16)
    gemm_int8_few_kernel<bf16_t, 8><<<grid, 512, 0, stream>>>(p);
  else
    return NS_ERR_UNSUPPORTED;
  return ns_launch_status();
}
