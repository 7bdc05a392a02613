// Matrix products in 8-bit integers: y[m][n] = xs[m] ws[n] sum_k cx[m][k] cw[n][k], codes -127 .. 127, the sum exact in 32-bit integers
// (K up to 32,768), rounded once as it is scaled.  And what stands in front of them: a row of activations quantised, its scale
// the largest magnitude / 127, as it is, behind an RMS norm, or behind the gate of a feed-forward.
// (reference: the nn.Linear calls of model/llama.py:175,184,195 are the same products in the model's precision; it has no form in fewer bits)
//
// Both operands lie in fragments, pieces of 1 KiB that are an operand of v_mfma_i32_16x16x64_i8 in lane order:
//   wt[row block rt][kc][lane = 16 g + r][16 bytes] = cw[16 rt + r][64 kc + 16 g + {0 .. 15}]
// the weight's laid out once, the activations' by the kernels that quantise them.  Rows are padded to a multiple of 16 and K to KP, a multiple of 256 and at least 512; the weight's
// padding is zeros, the activations' may be anything (beyond K it is multiplied with zeros, rows beyond M are not written).
#include "common.h"
#include "lds_loads.h"

typedef __attribute__((__vector_size__(4 * sizeof(int)))) int i32x4;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4;

#define INT8_TINY 0x1p-100f
#define INT8_MAX_K 32768  // (a row in the registers of a workgroup)

// ------------------------------------------------------------------------------------------------------------------------------------
// Rows into codes.  Bound by memory: a row is read once and kept in registers (up to 16 values a thread) between its maximum and its codes.
//   SRC 0: x;  1: w * (r * rsqrt(mean(r^2) + eps)), r = resid + x rounded to T, which is stored if resid_out;  2: silu(x[:K]) * x[K:]
// all in 32-bit and not rounded before the codes.  A row with an infinity or no number has the scale "no number": its products are none.
struct Int8RowsParams {
  int8_t* codes;   // fragments [rows up to a multiple of 16][kp]
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
  int8_t* to = p.codes + row / 16 * 16 * p.kp + row % 16 * 16;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = threadIdx.x + c * blockDim.x;
    if (i >= pieces) continue;
    code_t o;
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = some ? (int8_t)fminf(fmaxf(rintf(val[c][e] * inverse), -127.f), 127.f) : (int8_t)0;
    // (k = V i: its fragment, its lane group and its place among the lane's 16)
    *reinterpret_cast<code_t*>(to + V * i / 16 * 256 + V * i % 16) = o;
  }
  if (threadIdx.x == 0) p.scales[row] = fine ? (some ? most / 127.f : 0.f) : NAN;
}

template <typename T, int SRC, int V>
static int launch_rows(const Int8RowsParams& p, int rows, hipStream_t stream) {
  const int pieces = p.k / V;
  // (a wave for little, 1,024 threads for the widest rows: as many pieces a thread as there must be; four of fewer threads are no faster with many rows: 2,048 of 4,096 10.8 us and 10.7)
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
// Few rows: the weight streams, a workgroup a tile of 16 of its rows and 16 RB of x, its waves the pieces of K in turn; their sums meet in LDS.  Bound by memory with up to 16 rows: of
// 28,672 x 4,096 21 us, 5.6 TB/s of weights; with more by what a compute unit reads of both operands, some 60 bytes a ns (64 rows of 4,096 x 4,096 in RB 1, 2, 4: 12.8, 9.8, 8.1 us).
struct Int8Params {
  void* out;
  const int8_t *x, *w;
  const float *xs, *ws;
  int M, N, KP, out_stride, ranges;
  int quads;  // rows of the result are whole pieces of four values, side by side in memory
  int whole;  // ... of 16 bytes
};
static int int8_whole(const void* out, int N, int out_stride, int dtype) {
  const int v = dtype == NS_DTYPE_F32 ? 4 : 8;
  return N % v == 0 && out_stride % v == 0 && ((uintptr_t)out & 15) == 0;
}
static int int8_quads(const void* out, int N, int out_stride, int dtype) {
  return N % 4 == 0 && out_stride % 4 == 0 && ((uintptr_t)out & (dtype == NS_DTYPE_F32 ? 15 : 7)) == 0;
}

// the scales of four neighbours (there are as many as the weight has rows with its padding)
__device__ __forceinline__ f32x4 int8_scales(const Int8Params& p, int col) { return *reinterpret_cast<const f32x4*>(p.ws + col); }
// four neighbours of a row of the result; at once where rows lie so that they may be
template <typename T>
__device__ __forceinline__ void int8_store(const Int8Params& p, int row, int col, const i32x4 sum, float xs, const f32x4 ws) {
  typedef T vec_t __attribute__((ext_vector_type(4)));
  T* to = (T*)p.out + (size_t)row * p.out_stride + col;
  vec_t r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = from_f<T>((float)sum[e] * xs * ws[e]);
  if (p.quads) {
    *reinterpret_cast<vec_t*>(to) = r;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < p.N) to[e] = r[e];
  }
}

// AHEAD: pieces of a wave whose loads are on their way at a time.  Eight from K 4,096 on (16 rows of 4,096 x 4,096 5.1 us, four 5.3; of 57,344 x 8,192 78.0 and 78.9), four below
// (16,384 x 2,048 7.9, eight 10.5: half of them beyond the end), and four with more rows (64 rows of 4,096 x 14,336 21.6, eight 23.3).
template <typename T, int WAVES, int AHEAD, int RB>
__global__ __launch_bounds__(WAVES * 64) void gemm_int8_few_kernel(const Int8Params p) {
  __shared__ i32x4 sums[WAVES][RB][64];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), r = lane % 16, g = lane / 16;
  const int m0 = blockIdx.y * 16 * RB, pieces = p.KP / 64, blocks = (p.M - 1 - m0) / 16 + 1;
  const i32x4* w = reinterpret_cast<const i32x4*>(p.w + (size_t)blockIdx.x * 16 * p.KP) + lane;
  const i32x4* x[RB];  // (row blocks beyond the last are the last; their sums are not written)
#pragma unroll
  for (int i = 0; i < RB; ++i) x[i] = reinterpret_cast<const i32x4*>(p.x + (size_t)(m0 + 16 * min(i, blocks - 1)) * p.KP) + lane;
  i32x4 acc[RB];
#pragma unroll
  for (int i = 0; i < RB; ++i) acc[i] = i32x4{0, 0, 0, 0};
  int kc = wave;
  i32x4 a[AHEAD], b[AHEAD][RB];
  for (; kc + (AHEAD - 1) * WAVES < pieces; kc += AHEAD * WAVES) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      a[u] = __builtin_nontemporal_load(w + (size_t)(kc + u * WAVES) * 64);
#pragma unroll
      for (int i = 0; i < RB; ++i) b[u][i] = x[i][(size_t)(kc + u * WAVES) * 64];
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
      for (int i = 0; i < RB; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u], b[u][i], acc[i], 0, 0, 0);
  }
  if (kc < pieces) {  // the rest (beyond it the last piece is read once more and not multiplied)
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int at = min(kc + u * WAVES, pieces - 1);
      a[u] = __builtin_nontemporal_load(w + (size_t)at * 64);
#pragma unroll
      for (int i = 0; i < RB; ++i) b[u][i] = x[i][(size_t)at * 64];
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (kc + u * WAVES < pieces)
#pragma unroll
        for (int i = 0; i < RB; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u], b[u][i], acc[i], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < RB; ++i) sums[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave >= RB) return;
  i32x4 sum = sums[0][wave][lane];
#pragma unroll
  for (int v = 1; v < WAVES; ++v) sum += sums[v][wave][lane];
  const int row = m0 + 16 * wave + r, col = blockIdx.x * 16 + 4 * g;
  if (row < p.M && col < p.N) int8_store<T>(p, row, col, sum, p.xs[row], int8_scales(p, col));
}

template <typename T>
static int launch_int8_few(const Int8Params& p, int blocks, hipStream_t stream) {
  const dim3 grid((p.N + 15) / 16, (p.M + 16 * blocks - 1) / (16 * blocks));
  if (blocks == 4)
    gemm_int8_few_kernel<T, 8, 4, 4><<<grid, 512, 0, stream>>>(p);
  else if (blocks == 2)
    gemm_int8_few_kernel<T, 8, 4, 2><<<grid, 512, 0, stream>>>(p);
  else if (p.KP >= 4096)
    gemm_int8_few_kernel<T, 8, 8, 1><<<grid, 512, 0, stream>>>(p);
  else
    gemm_int8_few_kernel<T, 8, 4, 1><<<grid, 512, 0, stream>>>(p);
  return ns_launch_status();
}

// ``blocks``: row blocks of 16 of a workgroup's tile, 1, 2 or 4.
extern "C" int ns_gemm_int8(void* out, const void* x, const float* xs, const void* w, const float* ws, int M, int N, int KP, int out_stride, int blocks, int dtype, hipStream_t stream) {
  if (M < 0 || N <= 0 || KP < 512 || KP % 256 || KP > INT8_MAX_K || out_stride < N || (blocks != 1 && blocks != 2 && blocks != 4)) return NS_ERR_BAD_ARG;
  if ((((uintptr_t)x | (uintptr_t)w | (uintptr_t)ws) & 15) || (M - 1) / (16 * blocks) >= 65535) return NS_ERR_UNSUPPORTED;  // (a grid's rows)
  if (M == 0) return NS_OK;
  const Int8Params p{out, (const int8_t*)x, (const int8_t*)w, xs, ws, M, N, KP, out_stride, 1, int8_quads(out, N, out_stride, dtype), 0};
  if (dtype == NS_DTYPE_F32) return launch_int8_few<float>(p, blocks, stream);
  if (dtype == NS_DTYPE_BF16) return launch_int8_few<bf16_t>(p, blocks, stream);
  return NS_ERR_UNSUPPORTED;
}

// ------------------------------------------------------------------------------------------------------------------------------------
// More rows: a workgroup a tile of BM rows of x by BN of the weight, its WM x WN waves a part of the tile each.  The operands go straight from memory into LDS, a fragment a load, and
// from there a fragment a read, both linear in the lane: no bank is asked twice, and no address is a vector's.  ST stages of 64 k lie in LDS.  While the matrix unit works on stage
// s, out of registers, stage s + 1 is read into others.  Stages go in pairs with one barrier each (it costs a wave some 300 clocks, a pair of the largest tile's 2,048): at the
// beginning of pair (s, s + 1) the loads of stages s + ST - 1 and s + ST go out, into the places of stages s - 1 and s, which all have read; behind its end all waves' loads up to
// stage s + 4 have landed.  The waits are counted by hand (lds_loads.h): no other vector load may be on its way in run(), scratch memory's among them.
// Few tiles take ranges of K each, whose sums, whole numbers, a second kernel adds.
template <int BM_, int BN_, int WM, int WN, int ST_>
struct Int8Tile {
  static constexpr int BM = BM_, BN = BN_, ST = ST_, WAVES = WM * WN;
  static constexpr int FA = BM / 16, FB = BN / 16, MI = FA / WM, NJ = FB / WN;  // fragments of a stage; of a wave
  static constexpr int LA = FA / WAVES, LB = FB / WAVES, LOADS = LA + LB;      // loads of a wave and stage
  static constexpr int STAGE = (FA + FB) * 1024, BYTES = ST * STAGE;
  static_assert(LA * WAVES == FA && LB * WAVES == FB && MI * WM == FA && NJ * WN == FB && ST >= 4 && BYTES <= 160 * 1024, "whole fragments");

  uint8_t* lds;
  int lane, wave, wm, wn;
  int off[LOADS];  // the same in a wave's lanes: where its fragments begin
  __amdgpu_buffer_rsrc_t xr, wr;
  i32x4 acc[MI][NJ];

  __device__ __forceinline__ void init(uint8_t* lds_, const int8_t* x, const int8_t* w, int x_blocks, int w_blocks, int KP) {
    lds = lds_;
    lane = threadIdx.x % NS_WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / NS_WAVE), wm = wave / WN, wn = wave % WN;
    xr = __builtin_amdgcn_make_buffer_rsrc((void*)x, 0, 0xffffffff, 0x00020000);
    wr = __builtin_amdgcn_make_buffer_rsrc((void*)w, 0, 0xffffffff, 0x00020000);
    // (row blocks beyond the last are the last; their sums are not written)
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
      const int f = (q < LA ? q : q - LA) * WAVES + wave;
      off[q] = __builtin_amdgcn_readfirstlane(min(f, (q < LA ? x_blocks : w_blocks) - 1) * 16 * KP);
    }
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void load(int stage, int slot) const {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((address_space(3))) void* lds_ptr;
#pragma unroll
    for (int q = 0; q < LOADS; ++q) {
      const int f = (q < LA ? q : q - LA + FA / WAVES) * WAVES + wave;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(q < LA ? xr : wr, (lds_ptr)(lds + slot + f * 1024), 16, lane * 16, off[q] + stage * 1024, 0, 0);
    }
#endif
  }
  __device__ __forceinline__ i32x4 fragment(int slot, int f) const { return *reinterpret_cast<const i32x4*>(lds + slot + f * 1024 + lane * 16); }
  __device__ __forceinline__ i32x4 read(int slot, int e) const { return fragment(slot, e < MI ? wm * MI + e : FA + wn * NJ + e - MI); }

  static __device__ __forceinline__ int behind(int slot) { return slot + STAGE == BYTES ? 0 : slot + STAGE; }
  // a stage out of ``now``; the one behind it is read from ``from`` into ``then`` (behind the last: what nobody uses)
  __device__ __forceinline__ void stage(int from, const i32x4* now, i32x4* then) {
    // the reads are spread over most of the products: LDS gives a wave's fragment in 8 clocks, and all waves ask
    constexpr int READS = MI + NJ, SPAN = MI * NJ > 8 ? MI * NJ - MI * NJ / 8 : MI * NJ;
    int reads = 0;
#pragma unroll
    for (int m = 0; m < MI * NJ; ++m) {
      acc[m / NJ][m % NJ] = __builtin_amdgcn_mfma_i32_16x16x64_i8(now[MI + m % NJ], now[m / NJ], acc[m / NJ][m % NJ], 0, 0, 0);
      // (behind a product, not in front of the first: the compiler would have that wait for the read)
#pragma unroll
      for (int e = 0; e < READS; ++e)
        if (e == reads && e * SPAN < (m + 1) * READS) then[e] = read(from, e), ++reads;
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // an even number of stages, at least ST
  __device__ __forceinline__ void run(int stages) {
    i32x4 one[MI + NJ], two[MI + NJ];
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) load(s, s * STAGE);
    TILE_WAIT_LOADS((ST - 4) * LOADS);  // stages 0 to 2
    TILE_BARRIER();
#pragma unroll
    for (int e = 0; e < MI + NJ; ++e) one[e] = read(0, e);
    TILE_WAIT_LDS();  // stage 0 has been read by all before its place is loaded into
    TILE_BARRIER();
    int slot = 0, before = BYTES - STAGE;  // of stage s, and of the one before it
    for (int s = 0; s < stages; s += 2) {
      const int second = behind(slot), third = behind(second);
      if (s + ST - 1 < stages) load(s + ST - 1, before);
      if (s + ST < stages) load(s + ST, slot);  // (stage s has been read by all in the pair before)
      __builtin_amdgcn_sched_barrier(0);
      stage(second, one, two);
      stage(third, two, one);
      // the loads that may be on their way: those behind stage s + 4
      if (s + ST < stages) TILE_WAIT_LOADS((ST - 4) * LOADS);
      else TILE_WAIT_LOADS(0);
      TILE_WAIT_LDS();
      TILE_BARRIER();
      __builtin_amdgcn_sched_barrier(0);
      before = second, slot = third;
    }
  }
};

struct Int8ManyParams {
  Int8Params p;
  int* parts;  // [ranges][M][NP]: sums of the ranges (ranges > 1), NP = N up to a multiple of 4
  int m_tiles, n_tiles;
};

#define INT8_PATCH_M 4
#define INT8_PATCH_N 8

template <class Q, typename T, bool RANGES>
__global__ __launch_bounds__(Q::WAVES * NS_WAVE) __attribute__((amdgpu_waves_per_eu(2))) void gemm_int8_many_kernel(const Int8ManyParams a) {
  __shared__ __attribute__((aligned(16))) uint8_t int8_tiles[Q::BYTES];
  const Int8Params& p = a.p;
  // tiles go to the eight XCDs in eighths, range by range of K, within a range in patches of 4 x 8 tiles whose rows of both operands share an L2
  const int tiles = a.m_tiles * a.n_tiles, items = tiles * p.ranges, share = (items + 7) / 8;
  const int item = (blockIdx.x & 7) * share + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= share || item >= items) return;
  const int range = item / tiles;
  int tile = item - range * tiles;
  const int band = tile / (INT8_PATCH_M * a.n_tiles);
  tile -= band * INT8_PATCH_M * a.n_tiles;
  const int high = min(INT8_PATCH_M, a.m_tiles - band * INT8_PATCH_M), patch = tile / (high * INT8_PATCH_N);
  tile -= patch * high * INT8_PATCH_N;
  const int m0 = (band * INT8_PATCH_M + tile % high) * Q::BM, n0 = (patch * INT8_PATCH_N + tile / high) * Q::BN;
  // ranges of whole quarters of 1,024 bytes of a row block's 16, as even as they go
  const int quads = p.KP / 256, k0 = (int)((long long)quads * range / p.ranges) * 4, k1 = (int)((long long)quads * (range + 1) / p.ranges) * 4;  // in pieces of 64
  Q t;
  t.init(int8_tiles, p.x + (size_t)m0 * p.KP + (size_t)k0 * 1024, p.w + (size_t)n0 * p.KP + (size_t)k0 * 1024, (p.M - 1 - m0) / 16 + 1, (p.N - 1 - n0) / 16 + 1, p.KP);
  t.run(k1 - k0);

  const int r = t.lane % 16, g = t.lane / 16, np = (p.N + 3) & ~3;
  if constexpr (RANGES) {
#pragma unroll
    for (int i = 0; i < Q::MI; ++i) {
      const int row = m0 + 16 * (t.wm * Q::MI + i) + r;
      if (row >= p.M) continue;
#pragma unroll
      for (int j = 0; j < Q::NJ; ++j) {
        const int col = n0 + 16 * (t.wn * Q::NJ + j) + 4 * g;
        if (col < p.N) *reinterpret_cast<i32x4*>(a.parts + ((size_t)range * p.M + row) * np + col) = t.acc[i][j];
      }
    }
    return;
  }
  // all scales before the first result goes out: a load behind a store waits until that has been written (4 us a tile of 256 x 256)
  float xs[Q::MI];
  f32x4 ws[Q::NJ];
#pragma unroll
  for (int i = 0; i < Q::MI; ++i) xs[i] = p.xs[min(m0 + 16 * (t.wm * Q::MI + i) + r, p.M - 1)];
#pragma unroll
  for (int j = 0; j < Q::NJ; ++j) ws[j] = int8_scales(p, min(n0 + 16 * (t.wn * Q::NJ + j) + 4 * g, (p.N - 1) & ~3));
  const int row0 = m0 + 16 * t.wm * Q::MI, col0 = n0 + 16 * t.wn * Q::NJ;  // of this wave's part
  if (p.whole) {
    // by way of LDS, which nobody reads any more, a fragment's 16 rows at a time: pieces of 16 bytes, a row's side by side (2,048 x 24,576 with K 1,024 59 us; of 8 bytes from the
    // registers, four of a row side by side, 67)
    constexpr int V = 16 / sizeof(T), COLS = Q::NJ * 16, LINE = COLS * (int)sizeof(T) + 16, LANES = COLS / V, ROWS = NS_WAVE / LANES, DEEP = 2;
    static_assert(Q::WAVES * DEEP * 16 * LINE <= Q::BYTES && 16 % ROWS == 0, "a wave's lines");
    typedef T four_t __attribute__((ext_vector_type(4)));
    uint8_t* lines = int8_tiles + t.wave * (DEEP * 16 * LINE);
#pragma unroll
    for (int i = 0; i < Q::MI; ++i) {
      uint8_t* at = lines + i % DEEP * (16 * LINE);
#pragma unroll
      for (int j = 0; j < Q::NJ; ++j) {
        four_t v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = from_f<T>((float)t.acc[i][j][e] * xs[i] * ws[j][e]);
        *reinterpret_cast<four_t*>(at + r * LINE + (16 * j + 4 * g) * (int)sizeof(T)) = v;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int q = 0; q < 16 / ROWS; ++q) {
        const int line = q * ROWS + t.lane / LANES, row = row0 + 16 * i + line, col = col0 + t.lane % LANES * V;
        const i32x4 v = *reinterpret_cast<const i32x4*>(at + line * LINE + t.lane % LANES * 16);
        if (row < p.M && col < p.N) *reinterpret_cast<i32x4*>((T*)p.out + (size_t)row * p.out_stride + col) = v;
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < Q::MI; ++i) {
    const int row = row0 + 16 * i + r;
    if (row >= p.M) continue;
#pragma unroll
    for (int j = 0; j < Q::NJ; ++j) {
      const int col = col0 + 16 * j + 4 * g;
      if (col < p.N) int8_store<T>(p, row, col, t.acc[i][j], xs[i], ws[j]);
    }
  }
}

#define INT8_JOIN_ROWS 65535  // a row of workgroups each

template <typename T>
__global__ __launch_bounds__(256) void gemm_int8_join_kernel(const Int8ManyParams a) {
  const Int8Params& p = a.p;
  const int np = (p.N + 3) & ~3, col = (blockIdx.x * 256 + threadIdx.x) * 4, row = blockIdx.y;
  if (col >= p.N) return;
  i32x4 sum = {0, 0, 0, 0};
  for (int s = 0; s < p.ranges; ++s) sum += *reinterpret_cast<const i32x4*>(a.parts + ((size_t)s * p.M + row) * np + col);
  int8_store<T>(p, row, col, sum, p.xs[row], int8_scales(p, col));
}

template <class Q, typename T>
static int launch_int8_many(Int8ManyParams a, hipStream_t stream) {
  const Int8Params& p = a.p;
  a.m_tiles = (p.M + Q::BM - 1) / Q::BM, a.n_tiles = (p.N + Q::BN - 1) / Q::BN;
  const long long items = (long long)a.m_tiles * a.n_tiles * p.ranges;
  if (p.KP / 256 / p.ranges * 4 < Q::ST || items > (1 << 22) || (p.ranges > 1 && p.M > INT8_JOIN_ROWS)) return NS_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)((items + 7) / 8 * 8);
  if (p.ranges == 1) {
    gemm_int8_many_kernel<Q, T, false><<<grid, Q::WAVES * NS_WAVE, 0, stream>>>(a);
  } else {
    gemm_int8_many_kernel<Q, T, true><<<grid, Q::WAVES * NS_WAVE, 0, stream>>>(a);
    gemm_int8_join_kernel<T><<<dim3((p.N + 1023) / 1024, p.M), 256, 0, stream>>>(a);
  }
  return ns_launch_status();
}

template <typename T>
static int launch_int8_many(const Int8ManyParams& a, int form, hipStream_t stream) {
  switch (form) {
    case 0: return launch_int8_many<Int8Tile<64, 64, 2, 2, 8>, T>(a, stream);
    case 1: return launch_int8_many<Int8Tile<64, 128, 2, 2, 6>, T>(a, stream);
    case 2: return launch_int8_many<Int8Tile<128, 64, 2, 2, 6>, T>(a, stream);
    case 3: return launch_int8_many<Int8Tile<128, 128, 2, 2, 5>, T>(a, stream);
    case 4: return launch_int8_many<Int8Tile<256, 128, 4, 2, 5>, T>(a, stream);
    case 5: return launch_int8_many<Int8Tile<256, 256, 2, 4, 5>, T>(a, stream);
  }
  return NS_ERR_BAD_ARG;
}

// ``form``: the tile, rows of x by rows of w: 0 64 x 64, 1 64 x 128, 2 128 x 64, 3 128 x 128, 4 256 x 128, 5 256 x 256.  ``parts``: int32 [ranges * M * N up to a multiple of 4] on 16 bytes,
// with more ranges of K than one; a range has at least 512 of K.
extern "C" int ns_gemm_int8_many(void* out, void* parts, const void* x, const float* xs, const void* w, const float* ws, int M, int N, int KP, int out_stride, int form, int ranges,
                                 int dtype, hipStream_t stream) {
  if (M < 0 || N <= 0 || KP < 512 || KP % 256 || KP > INT8_MAX_K || out_stride < N || ranges < 1 || (ranges > 1 && !parts)) return NS_ERR_BAD_ARG;
  if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)ws | (uintptr_t)parts) & 15) return NS_ERR_UNSUPPORTED;
  if (M == 0) return NS_OK;
  const Int8ManyParams a{{out, (const int8_t*)x, (const int8_t*)w, xs, ws, M, N, KP, out_stride, ranges, int8_quads(out, N, out_stride, dtype), int8_whole(out, N, out_stride, dtype)}, (int*)parts, 0, 0};
  if (dtype == NS_DTYPE_F32) return launch_int8_many<float>(a, form, stream);
  if (dtype == NS_DTYPE_BF16) return launch_int8_many<bf16_t>(a, form, stream);
  return NS_ERR_UNSUPPORTED;
}
