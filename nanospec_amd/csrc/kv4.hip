// What a layer's new tokens put into pages of 4 bits (kv4.h says how those lie): queries and keys are rotated, and keys and values of
// every head quantised and packed; and the way back, keys and values as the pages hold them.
// (reference: kv/cache.py:23-26 writes them in the model's precision; it has no form in fewer bits)
#include "kv4.h"
#include "rope.h"

// The token of a workgroup: workgroups go to the eight XCDs in turn, and tokens in eighths, so that the eight neighbours whose values share every 16 bytes of a record meet in one L2
// (4,095 tokens written in 24 us and read in 8.8; as they come 25 and 9.7).
__device__ __forceinline__ int kv4_token(int n) {
  const int share = (n + 7) / 8;
  return (blockIdx.x & 7) * share + (blockIdx.x >> 3);
}
static unsigned kv4_token_grid(int n) { return (unsigned)((n + 7) / 8 * 8); }

// One wave's lanes in groups of W (a power of two, hd / 8 <= W <= 32): lane o of a group has channels 8 o .. 8 o + 7 of one row (the key
// or the value of one head); lanes from hd / 8 on have none.
struct Kv4Row {
  float low, step;
};
__device__ __forceinline__ Kv4Row kv4_marks_of(const float* x, bool has, int W) {
  float lo = INFINITY, hi = -INFINITY;
  int bad = 0;
  if (has) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo = fminf(lo, x[e]);
      hi = fmaxf(hi, x[e]);
      bad |= !(fabsf(x[e]) < INFINITY);
    }
  }
  for (int o = 1; o < W; o <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, o, NS_WAVE));
    hi = fmaxf(hi, __shfl_xor(hi, o, NS_WAVE));
    bad |= __shfl_xor(bad, o, NS_WAVE);
  }
  const float low = bf16_floor(lo), reach = hi - low;
  if (bad || !(reach < KV4_HUGE)) return {__uint_as_float(0x7fc00000u), 0.f};
  const float step = bf16_ceil(reach / 15.f);
  return {low, step < KV4_TINY ? 0.f : step};
}
// Divided, not times 1 / step: of short numbers (bfloat16 inputs) many lie half way between two codes exactly, and the quotient keeps that.  With y = 1 / step rounded to nearest, and q a
// quotient that is off by no more than its last bit, q + (a - q step) y is the quotient rounded to nearest (Markstein 1990): a reciprocal a row and three operations a value.
__device__ __forceinline__ uint32_t kv4_code(float x, const Kv4Row r, float y) {
  const float a = x - r.low, q = a * y;
  return (uint32_t)fminf(fmaxf(rintf(fmaf(fmaf(-q, r.step, a), y, q)), 0.f), 15.f);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x, bool wide) {
  constexpr int V = 16 / sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(V)));
  if (wide) {
#pragma unroll
    for (int i = 0; i < 8 / V; ++i) {
      vec_t v;
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = from_f<T>(x[i * V + e]);
      reinterpret_cast<vec_t*>(p)[i] = v;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = from_f<T>(x[e]);
  }
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x, bool wide) {
  constexpr int V = 16 / sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(V)));
  if (wide) {
#pragma unroll
    for (int i = 0; i < 8 / V; ++i) {
      const vec_t v = reinterpret_cast<const vec_t*>(p)[i];
#pragma unroll
      for (int e = 0; e < V; ++e) x[i * V + e] = to_f(v[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f(p[e]);
  }
}

// Channels 8 o .. 8 o + 7 of a head, and those that the rotation pairs them with, as they are read.  WIDE: whole vectors of 16 bytes, as the partners of 8 channels of a half are 8 of the
// other.
template <typename T, bool WIDE>
struct Kv4Piece {
  static constexpr int V = 16 / sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(V)));
  vec_t own[8 / V], other[8 / V];
  __device__ __forceinline__ void load(const T* p, int o, const RopeForm f, bool turns, bool) {
    const int half = f.rot / 2, c0 = 8 * o;
    const vec_t *a = reinterpret_cast<const vec_t*>(p + c0), *b = reinterpret_cast<const vec_t*>(p + (c0 < half ? c0 + half : c0 - half));
#pragma unroll
    for (int i = 0; i < 8 / V; ++i) own[i] = a[i];
    if (turns && c0 < f.rot)
#pragma unroll
      for (int i = 0; i < 8 / V; ++i) other[i] = b[i];
  }
  __device__ __forceinline__ void values(float* x, int o, const RopeForm f, bool turns, const float* cs) const {
#pragma clang fp contract(off)
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f((T)own[e / V][e % V]);
    const int half = f.rot / 2, c0 = 8 * o;
    if (!turns || c0 >= f.rot) return;
    const bool second = c0 >= half;
    typedef float four __attribute__((ext_vector_type(4)));
    const four *c = reinterpret_cast<const four*>(cs + (second ? c0 - half : c0)), *s = reinterpret_cast<const four*>(cs + (second ? c0 : c0 + half));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float turned = x[e] * c[e / 4][e % 4], cross = to_f((T)other[e / V][e % V]) * s[e / 4][e % 4];
      x[e] = second ? turned + cross : turned - cross;
    }
  }
};
template <typename T>
struct Kv4Piece<T, false> {
  float own[8], other[8];
  __device__ __forceinline__ void load(const T* p, int o, const RopeForm f, bool turns, bool aligned) {
    load8(p + 8 * o, own, aligned);
    const int half = f.rot / 2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int ch = 8 * o + e;
      other[e] = 0.f;
      if (!turns || ch >= f.rot) continue;
      int d1, d2;
      rope_pair_channels(f, f.interleaved ? ch / 2 : ch % half, d1, d2);
      other[e] = to_f(p[ch == d1 ? d2 : d1]);
    }
  }
  __device__ __forceinline__ void values(float* x, int o, const RopeForm f, bool turns, const float* cs) const {
#pragma clang fp contract(off)
    const int half = f.rot / 2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int ch = 8 * o + e;
      x[e] = own[e];
      if (!turns || ch >= f.rot) continue;
      const bool first = f.interleaved ? ch % 2 == 0 : ch < half;
      const int j = f.interleaved ? ch / 2 : first ? ch : ch - half;
      const float turned = x[e] * cs[j], cross = other[e] * cs[half + j];
      x[e] = first ? turned - cross : turned + cross;
    }
  }
};
// (the products and their sum are rounded one by one, with no fused multiply-add: a key's codes are then those of the formula's own 32-bit operations)

struct Kv4WriteParams {
  const void* qkv;  // [tokens][heads + 2 kv_heads][hd], rows row_stride apart
  void* q_out;      // the rotated queries, rows q_stride apart (qkv itself: in place)
  const int *positions, *token_req, *block_table;
  const float* inv_freq;
  uint8_t* pool;
  int tokens, row_stride, q_stride, table_stride, heads, kv_heads, hd, page, write_kv, wide, aligned, width;  // width: lanes of a row
  RopeForm form;
};

// A workgroup a token; its groups of W lanes take the rows (queries, keys, values, as they lie in qkv) in turn, UNITS of them at once: all that a thread reads is on its way before the
// token's angles are made and before anything is written (in place, the partners are each other's).
// Bound by memory with many tokens (4,095 of 32 heads on 8 of 128 channels, 88 MB: 23 us, 3.8 TB/s; a row after the other 29, with eight divisions a lane 24), by one chain of loads with few.
template <typename T, bool WIDE, int UNITS>
__global__ __launch_bounds__(256) void rope_kv4_kernel(const Kv4WriteParams p) {
  extern __shared__ __attribute__((aligned(16))) float cs[];  // cos[half] | sin[half] of this token's angles
  const int t = kv4_token(p.tokens);
  if (t >= p.tokens) return;
  const int pos = p.positions[t], half = p.form.rot / 2;
  const T* row = (const T*)p.qkv + (size_t)t * p.row_stride;
  T* qo = (T*)p.q_out + (size_t)t * p.q_stride;
  const int W = p.width, o = threadIdx.x % W, first = threadIdx.x / W, step = blockDim.x / W;
  const int rows = p.write_kv ? p.heads + 2 * p.kv_heads : p.heads, keys = p.heads + p.kv_heads;
  const bool has = 8 * o < p.hd, whole = p.q_out != p.qkv;
  const int record = kv4_record(p.hd), groups = p.hd / 32, off = pos % p.page, j = off % KV4_TOKENS;
  const int page = p.write_kv ? p.block_table[(size_t)p.token_req[t] * p.table_stride + pos / p.page] : 0;
  for (int r0 = 0; r0 < rows; r0 += UNITS * step) {
    Kv4Piece<T, WIDE> piece[UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int r = r0 + u * step + first;
      if (has && r < rows) piece[u].load(row + (size_t)r * p.hd, o, p.form, r < keys, p.aligned);
    }
    if (r0 == 0)
      for (int i = threadIdx.x; i < 2 * half; i += blockDim.x) {
        const float angle = (float)pos * p.inv_freq[i < half ? i : i - half];
        cs[i] = (i < half ? cosf(angle) : sinf(angle)) * p.form.factor;
      }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int r = r0 + u * step + first;
      const bool live = has && r < rows, value = r >= keys;
      float x[8];
      if (live) piece[u].values(x, o, p.form, !value, cs);
      if (r < p.heads) {
        if (live && (whole || 8 * o < p.form.rot)) store8(qo + (size_t)r * p.hd + 8 * o, x, p.aligned);
        continue;
      }
      const Kv4Row m = kv4_marks_of(x, live, W);
      if (!live) continue;
      const float y = m.step > 0.f ? 1.f / m.step : 0.f;  // (0: all codes are 0)
      const int h = r - (value ? keys : p.heads);
      uint8_t* to = p.pool + kv4_at(page, p.kv_heads, h, p.page / KV4_TOKENS, off / KV4_TOKENS) * record;
      if (value) {
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          lo |= kv4_code(x[e], m, y) << (4 * e);
          hi |= kv4_code(x[4 + e], m, y) << (4 * e);
        }
        uint16_t* d = reinterpret_cast<uint16_t*>(to + kv4_values_at(p.hd) + 2 * o * 16 + j * 2);
        d[0] = (uint16_t)lo;
        d[8] = (uint16_t)hi;
      } else {
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) w |= kv4_code(x[e], m, y) << (4 * (e / 2) + 16 * (e % 2));
        reinterpret_cast<uint32_t*>(to + j * (p.hd / 2))[o % 4 * groups + o / 4] = w;
      }
      if (o == 0)
        reinterpret_cast<uint32_t*>(to + kv4_marks_at(p.hd))[(value ? KV4_TOKENS : 0) + j] = (__float_as_uint(m.step) & 0xffff0000u) | (__float_as_uint(m.low) >> 16);
    }
  }
}

template <typename T>
static void launch_write(const Kv4WriteParams& p, size_t lds, hipStream_t stream) {
  // the rows of a group of lanes, in as few passes of at most three as they take
  const int step = 256 / p.width, rows = p.write_kv ? p.heads + 2 * p.kv_heads : p.heads, each = (rows + step - 1) / step, passes = (each + 2) / 3;
  const int units = (each + passes - 1) / passes;
  const unsigned grid = kv4_token_grid(p.tokens);
  if (!p.wide || !p.aligned)
    rope_kv4_kernel<T, false, 1><<<grid, 256, lds, stream>>>(p);
  else if (units == 1)
    rope_kv4_kernel<T, true, 1><<<grid, 256, lds, stream>>>(p);
  else if (units == 2)
    rope_kv4_kernel<T, true, 2><<<grid, 256, lds, stream>>>(p);
  else
    rope_kv4_kernel<T, true, 3><<<grid, 256, lds, stream>>>(p);
}

static bool kv4_sizes(int kv_heads, int hd, int page) {
  return kv_heads > 0 && hd >= 32 && hd <= KV4_MAX_HD && hd % 32 == 0 && page >= KV4_TOKENS && (page & (page - 1)) == 0;
}

// q (rotated) into ``q_out`` [tokens][heads][hd] (rows q_stride apart; the same tensor as qkv, with its stride, rotates in place); k (rotated)
// and v of every token into the pages block_table[token_req[t]][position / page].
extern "C" int ns_rope_kv4_write(const void* qkv, int row_stride, void* q_out, int q_stride, const int* positions, const int* token_req, const int* block_table,
                                 int table_stride, const float* inv_freq, void* pool, int n_tokens, int heads, int kv_heads, int hd, int rot, int interleaved,
                                 float factor, int page, int write_kv, int dtype, hipStream_t stream) {
  if (n_tokens < 0 || heads <= 0 || !kv4_sizes(kv_heads, hd, page) || rot < 0 || rot > hd || (rot & 1)) return NS_ERR_BAD_ARG;
  if (n_tokens == 0) return NS_OK;
  const int v = dtype == NS_DTYPE_F32 ? 4 : 8;
  int width = 4;
  while (width < hd / 8) width *= 2;
  const int aligned = (((uintptr_t)qkv | (uintptr_t)q_out) & 15) == 0 && row_stride % v == 0 && q_stride % v == 0;
  const int wide = !interleaved && rot / 2 % 8 == 0;
  const Kv4WriteParams p{qkv, q_out, positions, token_req, block_table, inv_freq, (uint8_t*)pool, n_tokens, row_stride, q_stride, table_stride, heads, kv_heads, hd, page,
                         write_kv, wide, aligned, width, {rot, interleaved ? 1 : 0, factor}};
  const size_t lds = (size_t)(rot + 2) * sizeof(float);
  if (dtype == NS_DTYPE_F32)
    launch_write<float>(p, lds, stream);
  else if (dtype == NS_DTYPE_BF16)
    launch_write<bf16_t>(p, lds, stream);
  else
    return NS_ERR_UNSUPPORTED;
  return ns_launch_status();
}

// the value of a code as 32 bits make it, rounded once
template <typename T>
__global__ __launch_bounds__(256) void kv4_read_kernel(T* __restrict__ k, T* __restrict__ v, const uint8_t* __restrict__ pool, const int* __restrict__ positions,
                                                       const int* __restrict__ token_req, const int* __restrict__ block_table, int table_stride, int kv_heads,
                                                       int hd, int page, bool aligned, int tokens) {
  const int t = kv4_token(tokens);
  if (t >= tokens) return;
  const int pos = positions[t];
  const int at = block_table[(size_t)token_req[t] * table_stride + pos / page], off = pos % page, j = off % KV4_TOKENS, parts = hd / 8, groups = hd / 32;
  for (int u = threadIdx.x; u < 2 * kv_heads * parts; u += blockDim.x) {
    const int r = u / parts, o = u % parts;
    const bool value = r >= kv_heads;
    const int h = value ? r - kv_heads : r;
    const uint8_t* from = pool + kv4_at(at, kv_heads, h, page / KV4_TOKENS, off / KV4_TOKENS) * kv4_record(hd);
    const uint32_t mark = reinterpret_cast<const uint32_t*>(from + kv4_marks_at(hd))[(value ? KV4_TOKENS : 0) + j];
    const float low = kv4_low(mark), step = kv4_step(mark);
    uint32_t code[8];
    if (value) {
      const uint16_t* w = reinterpret_cast<const uint16_t*>(from + kv4_values_at(hd) + 2 * o * 16 + j * 2);
#pragma unroll
      for (int e = 0; e < 8; ++e) code[e] = (uint32_t)w[e / 4 * 8] >> (4 * (e % 4)) & 15u;
    } else {
      const uint32_t w = reinterpret_cast<const uint32_t*>(from + j * (hd / 2))[o % 4 * groups + o / 4];
#pragma unroll
      for (int e = 0; e < 8; ++e) code[e] = w >> (4 * (e / 2) + 16 * (e % 2)) & 15u;
    }
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma clang fp contract(off)
      const float part = step * (float)code[e];
      x[e] = part + low;
    }
    store8((value ? v : k) + ((size_t)t * kv_heads + h) * hd + 8 * o, x, aligned);
  }
}

extern "C" int ns_kv4_read(void* k, void* v, const void* pool, const int* positions, const int* token_req, const int* block_table, int table_stride,
                           int n_tokens, int kv_heads, int hd, int page, int dtype, hipStream_t stream) {
  if (n_tokens < 0 || !kv4_sizes(kv_heads, hd, page)) return NS_ERR_BAD_ARG;
  if (n_tokens == 0) return NS_OK;
  const bool aligned = (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
  if (dtype == NS_DTYPE_F32)
    kv4_read_kernel<float><<<kv4_token_grid(n_tokens), 256, 0, stream>>>((float*)k, (float*)v, (const uint8_t*)pool, positions, token_req, block_table, table_stride, kv_heads, hd, page, aligned, n_tokens);
  else if (dtype == NS_DTYPE_BF16)
    kv4_read_kernel<bf16_t><<<kv4_token_grid(n_tokens), 256, 0, stream>>>((bf16_t*)k, (bf16_t*)v, (const uint8_t*)pool, positions, token_req, block_table, table_stride, kv_heads, hd, page, aligned, n_tokens);
  else
    return NS_ERR_UNSUPPORTED;
  return ns_launch_status();
}
