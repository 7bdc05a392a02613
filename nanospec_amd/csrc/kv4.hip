// What a layer's new tokens put into pages of 4 bits (kv4.h says how those lie): queries and keys are rotated, and keys and values of
// every head quantised and packed; and the way back, keys and values as the pages hold them.
// (reference: kv/cache.py:23-26 writes them in the model's precision; it has no form in fewer bits)
#include "kv4.h"
#include "rope.h"

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
// Divided, not times 1 / step: of short numbers (bfloat16 inputs) many lie half way between two codes exactly, and the quotient keeps that
__device__ __forceinline__ uint32_t kv4_code(float x, const Kv4Row r) {
  return r.step > 0.f ? (uint32_t)fminf(fmaxf(rintf((x - r.low) / r.step), 0.f), 15.f) : 0u;
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

// Channels 8 o .. 8 o + 7 of a rotated head at p.  The products and their sum are rounded one by one (no fused multiply-add): a key's codes
// are then those of the formula's own 32-bit operations.  ``wide``: 8 channels of a half have their partners in 8 of the other.
template <typename T>
__device__ __forceinline__ void rotated8(const T* p, int o, int hd, const RopeForm f, const float* cs, bool wide, bool aligned, float* x) {
#pragma clang fp contract(off)
  const int half = f.rot / 2, c0 = 8 * o;
  load8(p + c0, x, aligned);
  if (c0 >= f.rot) return;
  if (wide) {
    const bool second = c0 >= half;
    const int j0 = second ? c0 - half : c0;
    float other[8];
    load8(p + (second ? j0 : j0 + half), other, aligned);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float c = cs[j0 + e], s = cs[half + j0 + e];
      const float own = x[e] * c, cross = other[e] * s;
      x[e] = second ? own + cross : own - cross;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int ch = c0 + e;
    if (ch >= f.rot) continue;
    const int j = f.interleaved ? ch / 2 : ch % half;
    int d1, d2;
    rope_pair_channels(f, j, d1, d2);
    const float c = cs[j], s = cs[half + j];
    const float own = x[e] * c, cross = to_f(p[ch == d1 ? d2 : d1]) * s;
    x[e] = ch == d1 ? own - cross : own + cross;
  }
}

struct Kv4WriteParams {
  const void* qkv;  // [tokens][heads + 2 kv_heads][hd], rows row_stride apart
  void* q_out;      // the rotated queries, rows q_stride apart (qkv itself: in place)
  const int *positions, *token_req, *block_table;
  const float* inv_freq;
  uint8_t* pool;
  int row_stride, q_stride, table_stride, heads, kv_heads, hd, page, write_kv, wide, aligned, width;  // width: lanes of a row
  RopeForm form;
};

template <typename T>
__global__ __launch_bounds__(256) void rope_kv4_kernel(const Kv4WriteParams p) {
  extern __shared__ float cs[];  // cos[half] | sin[half] of this token's angles
  const int t = blockIdx.x, pos = p.positions[t], half = p.form.rot / 2;
  for (int j = threadIdx.x; j < half; j += blockDim.x) rope_cos_sin(p.form, pos, p.inv_freq[j], cs[j], cs[half + j]);
  __syncthreads();
  const T* row = (const T*)p.qkv + (size_t)t * p.row_stride;
  const int W = p.width, o = threadIdx.x % W, first = threadIdx.x / W, step = blockDim.x / W, parts = p.hd / 8;
  const bool has = o < parts;
  // queries; a group's lanes read a whole head before they write it (in place the partners are each other's)
  T* qo = (T*)p.q_out + (size_t)t * p.q_stride;
  const bool in_place = p.q_out == p.qkv;
  for (int h0 = 0; h0 < p.heads; h0 += step) {
    const int h = h0 + first;
    float x[8];
    const bool mine = has && h < p.heads && (!in_place || 8 * o < p.form.rot);
    if (mine) rotated8(row + h * p.hd, o, p.hd, p.form, cs, p.wide, p.aligned, x);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (mine) store8(qo + h * p.hd + 8 * o, x, p.aligned);
  }
  if (!p.write_kv) return;
  const int page = p.block_table[(size_t)p.token_req[t] * p.table_stride + pos / p.page], off = pos % p.page, j = off % KV4_TOKENS;
  const int record = kv4_record(p.hd), groups = p.hd / 32;
  // keys, then values: rows 0 .. 2 kv_heads - 1
  for (int r0 = 0; r0 < 2 * p.kv_heads; r0 += step) {
    const int r = r0 + first;
    const bool live = r < 2 * p.kv_heads, value = r >= p.kv_heads;
    const int h = value ? r - p.kv_heads : r;
    float x[8];
    if (live && has) {
      const T* from = row + (size_t)(p.heads + r) * p.hd;
      if (value)
        load8(from + 8 * o, x, p.aligned);
      else
        rotated8(from, o, p.hd, p.form, cs, p.wide, p.aligned, x);
    }
    const Kv4Row m = kv4_marks_of(x, live && has, W);
    if (!live || !has) continue;
    uint8_t* to = p.pool + kv4_at(page, p.kv_heads, h, p.page / KV4_TOKENS, off / KV4_TOKENS) * record;
    if (value) {
      uint32_t lo = 0, hi = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo |= kv4_code(x[e], m) << (4 * e);
        hi |= kv4_code(x[4 + e], m) << (4 * e);
      }
      uint16_t* d = reinterpret_cast<uint16_t*>(to + kv4_values_at(p.hd) + 2 * o * 16 + j * 2);
      d[0] = (uint16_t)lo;
      d[8] = (uint16_t)hi;
    } else {
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) w |= kv4_code(x[e], m) << (4 * (e / 2) + 16 * (e % 2));
      reinterpret_cast<uint32_t*>(to + j * (p.hd / 2))[o % 4 * groups + o / 4] = w;
    }
    if (o == 0)
      reinterpret_cast<uint32_t*>(to + kv4_marks_at(p.hd))[(value ? KV4_TOKENS : 0) + j] = (__float_as_uint(m.step) & 0xffff0000u) | (__float_as_uint(m.low) >> 16);
  }
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
  const Kv4WriteParams p{qkv, q_out, positions, token_req, block_table, inv_freq, (uint8_t*)pool, row_stride, q_stride, table_stride, heads, kv_heads, hd, page,
                         write_kv, wide, aligned, width, {rot, interleaved ? 1 : 0, factor}};
  const size_t lds = (size_t)(rot + 2) * sizeof(float);
  if (dtype == NS_DTYPE_F32)
    rope_kv4_kernel<float><<<n_tokens, 256, lds, stream>>>(p);
  else if (dtype == NS_DTYPE_BF16)
    rope_kv4_kernel<bf16_t><<<n_tokens, 256, lds, stream>>>(p);
  else
    return NS_ERR_UNSUPPORTED;
  return ns_launch_status();
}

// the value of a code as 32 bits make it, rounded once
template <typename T>
__global__ __launch_bounds__(256) void kv4_read_kernel(T* __restrict__ k, T* __restrict__ v, const uint8_t* __restrict__ pool, const int* __restrict__ positions,
                                                       const int* __restrict__ token_req, const int* __restrict__ block_table, int table_stride, int kv_heads,
                                                       int hd, int page) {
  const int t = blockIdx.x, pos = positions[t];
  const int at = block_table[(size_t)token_req[t] * table_stride + pos / page], off = pos % page, j = off % KV4_TOKENS, parts = hd / 8, groups = hd / 32;
  for (int u = threadIdx.x; u < 2 * kv_heads * parts; u += blockDim.x) {
    const int r = u / parts, o = u % parts;
    const bool value = r >= kv_heads;
    const int h = value ? r - kv_heads : r;
    const uint8_t* from = pool + kv4_at(at, kv_heads, h, page / KV4_TOKENS, off / KV4_TOKENS) * kv4_record(hd);
    const uint32_t mark = reinterpret_cast<const uint32_t*>(from + kv4_marks_at(hd))[(value ? KV4_TOKENS : 0) + j];
    const float low = kv4_low(mark), step = kv4_step(mark);
    T* to = (value ? v : k) + ((size_t)t * kv_heads + h) * hd + 8 * o;
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
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma clang fp contract(off)
      const float part = step * (float)code[e];
      to[e] = from_f<T>(part + low);
    }
  }
}

extern "C" int ns_kv4_read(void* k, void* v, const void* pool, const int* positions, const int* token_req, const int* block_table, int table_stride,
                           int n_tokens, int kv_heads, int hd, int page, int dtype, hipStream_t stream) {
  if (n_tokens < 0 || !kv4_sizes(kv_heads, hd, page)) return NS_ERR_BAD_ARG;
  if (n_tokens == 0) return NS_OK;
  if (dtype == NS_DTYPE_F32)
    kv4_read_kernel<float><<<n_tokens, 256, 0, stream>>>((float*)k, (float*)v, (const uint8_t*)pool, positions, token_req, block_table, table_stride, kv_heads, hd, page);
  else if (dtype == NS_DTYPE_BF16)
    kv4_read_kernel<bf16_t><<<n_tokens, 256, 0, stream>>>((bf16_t*)k, (bf16_t*)v, (const uint8_t*)pool, positions, token_req, block_table, table_stride, kv_heads, hd, page);
  else
    return NS_ERR_UNSUPPORTED;
  return ns_launch_status();
}
