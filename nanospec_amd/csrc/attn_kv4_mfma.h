// Attention over 4-bit pages on the matrix cores, head sizes 64 and 128.  Included by attn_kv4.hip.
//
// A wave walks 32 keys at a time with CT tiles of 16 columns, a column a (token, query head) pair of one request and key/value head:
//   S^T[key][col] = K[key][:] . Q[col][:]          A = 16 keys, B = the columns' queries
//   O^T[channel][col] += V^T[channel][key] . P^T   A = 16 channels, B = the columns' weights, in the layout that S^T came out in
// Keys go to the rows of the first product in the order that makes its result the second's operand: row 4 t + r of tile a is key 8 t + 4 a + r of
// the 32, so that lane (col, t) holds the weights of keys 8 t .. 8 t + 7, one octet, whose values and marks it reads in whole records.
// Nothing passes through LDS on the way (a wave's operands are 4.25 bits a value, from L2): the waves need no barriers.
//
// From codes to operands.  A code in the lowest four bits of a float16, all others zero, is that many 2^-24, a number below the normal range, which the matrix instruction multiplies
// exactly (in the next four bits: times 16).  A mask makes two codes of a dword operands, and nothing has to be taken off: the products are 2^-24 (2^-20) times the sums of whole
// numbers that are meant.  The queries' channels that meet codes times 16 carry a factor of 1/16, exactly; the outputs' channels that do are multiplied by it at the end.
//   s = step (q . u) + low sum(q):      two operations a score, as both are a key's
//   out = sum p step u + sum p low:     p step is the weight in the second product, the rest a sum of numbers
// Of a lane's octet the last four keys have their codes turned round, 15 - u, and their weights' signs with them:
//   sum p step u = sum over the first four p step u - sum over the last four p step (15 - u) + sum over the last four p (15 step),   15 step added to those keys' low
// The sums of whole numbers, all positive, would grow with the keys, and a mean of many values is many times smaller: the instruction cuts off what lies some 20 bits below its largest product, towards zero, which of
// such sums is always the same way (-1.2e-3 of the result over 400,000 keys).  So half of the products have the other sign, and what is cut off of them cancels (under 1e-4; one instruction for eight codes and one for
// each of four keys, 1% of a portion's time; codes less 8 everywhere, an instruction for two codes, 9 to 17%).
// Queries are float16 on their way in, scaled by a power of two of their own so that the largest lies at 256: what is 2^-22 of it is exact.  Weights are
// rounded to float16 (2^-12 of themselves).
// float32 (EXACT) takes the 32-bit matrix instructions, with codes as the numbers 16 (u - 8), bytes that a mask and a sign bit make, low + 8 step in the place of low, and everything in 32 bits.  (Queries and weights as two
// float16 values each were faster and 1e-4 of the result off at 4,000 keys: with all codes positive the two sums above are many times what is left of them, and the instruction cuts off what lies below its largest
// product.)
//
// The soft-max's reference R is one number a column for weights and steps together: R >= (score + log2 of its value's step) - 15 of every key so far, so
// that p step, p = 2^(s - R), fits float16 whatever the steps' size, and is only raised when that no longer holds (then every sum shrinks).  (Key by key: by the largest score and the largest step
// apart, a value of great size whose key has next to no weight would cost the others their bits; that costs a portion 5%.)
// It knows of the keys that the column sees, and of no others.  (kv4_log has what is taken for a step that is next to nothing, or small beside its value.)
#pragma once

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

#define KV4_TILE_INTS 8
#define KV4_TILE_TOKENS 32  // of a portion's tile
#define KV4_TOP 7.f    // log2 of the largest weight times step where the reference is raised to it, so that of small ones float16's subnormal numbers cost as little as may be ...
#define KV4_SLACK 8.f  // ... and how far above that another may come before it is raised again: 2^15 is below float16's largest
#define KV4_RANGE_BLOCKS 8  // of 32 keys: the fewest of a range of a single token's keys
#define KV4_PORTION_BLOCKS 4  // ... and of a portion's (KV4_PORTION_KEYS of parts/attention.py)

__device__ __forceinline__ f16x8 as_f16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __builtin_bit_cast(f16x8, u32x4{a, b, c, d}); }
// two codes of a dword as 2^-24 u, and as 2^-20 u
__device__ __forceinline__ uint32_t kv4_ones(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t kv4_sixteens(uint32_t w) { return w & 0x00f000f0u; }
// log2 + 127, up to 0.09 below it, of a value's step, or of what its lowest value makes of that: weights go up to 2^15 over it, and sums of them, and of them times lowest values, are to fit 32 bits.  So it counts as at
// least 2^-64 of the lowest value (2^79 a key; what a smaller step adds is below its last bit anyway), and as at least 2^-88 (2^103 a key, for 2^24 keys; steps go down to 2^-100, whose weights of 2^-5 and more float16
// still holds).  A lowest value that is no number counts for nothing here.
__device__ __forceinline__ float kv4_log(float step, float low) { return (float)__float_as_uint(fmaxf(fmaxf(step, fabsf(low) * 0x1p-64f), 0x1p-88f)) * 0x1p-23f; }
// the upper codes of a dword's bytes as signed bytes 16 (u - 8), and one of them as a number
__device__ __forceinline__ uint32_t kv4_signed(uint32_t w) { return (w & 0xf0f0f0f0u) ^ 0x80808080u; }
__device__ __forceinline__ float kv4_byte(uint32_t w, int y) { return (float)(int8_t)(w >> (8 * y)); }
__device__ __forceinline__ float quarters_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, NS_WAVE));
  return fmaxf(v, __shfl_xor(v, 32, NS_WAVE));
}
__device__ __forceinline__ float quarters_sum(float v) {
  v += __shfl_xor(v, 16, NS_WAVE);
  return v + __shfl_xor(v, 32, NS_WAVE);
}

// 32 keys as they lie in the pages
template <int HD>
struct Kv4Block {
  uint32_t k[2][HD / 32];  // [tile a]: this lane's dwords of its key
  u32x4 v[HD / 64];        // its octet's values, four channels of each 64
  u32x4 km[2], vm[2];      // its octet's marks
};

// CT: tiles of 16 columns.  EXACT: float32.
template <typename T, int HD, int CT, bool EXACT>
struct Kv4Wave {
  static constexpr int NG = HD / 32, NB = HD / 64;
  static constexpr int REC = 8 * HD + 64;
  f16x8 q[CT][EXACT ? 1 : NG];
  float q32[EXACT ? CT : 1][EXACT ? NG : 1][8];
  float qsum[CT], unscale[CT];  // sum of the scaled queries, times 2^-24 as the products are; what a score is multiplied with: the scale, log2(e), the queries' own scale and the 2^-24 taken off (EXACT: neither)
  float R[CT], l[CT], z[CT];
  f32x4v o[CT][NB][4];
  int lane, col, t;
  int kpos[CT], kfirst[CT];  // the last and the first key that this lane's column sees

  __device__ __forceinline__ void init() {
    lane = threadIdx.x % NS_WAVE, col = lane % 16, t = lane / 16;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      R[c] = -INFINITY, l[c] = 0.f, z[c] = 0.f;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[c][b][i] = f32x4v{0.f, 0.f, 0.f, 0.f};
    }
  }

  // this lane's column of tile c: its query's channels (nullptr: a column of zeros).  ``wide``: they lie at a multiple of 16 bytes.
  __device__ __forceinline__ void query(int c, const T* from, float scale_log2, bool wide) {
    float x[NG][8], most = 0.f;
    if (!from) {
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[g][e] = 0.f;
    } else if (wide) {
      constexpr int V = 16 / sizeof(T);
      typedef T vec_t __attribute__((ext_vector_type(V)));
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 8 / V; ++i) {
          const vec_t v = *reinterpret_cast<const vec_t*>(from + 32 * g + 8 * t + V * i);
#pragma unroll
          for (int e = 0; e < V; ++e) x[g][V * i + e] = to_f((T)v[e]);
        }
    } else {
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[g][e] = to_f(from[32 * g + 8 * t + e]);
    }
    if constexpr (EXACT) {
      float sum = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) q32[c][g][e] = x[g][e], sum += x[g][e];
      qsum[c] = quarters_sum(sum);
      unscale[c] = scale_log2;
      return;
    }
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[g][e]));
    most = quarters_max(most);
    // 2^(8 - exponent): exact; nothing to scale in zeros and where the largest is infinite (the products are then no numbers by themselves)
    const int ex = (int)(__float_as_uint(most) >> 23);
    const int up = ex == 0 || ex == 255 ? 127 : min(max(127 + 127 + 8 - ex, 1), 254);
    const float by = __uint_as_float((uint32_t)up << 23);
    unscale[c] = scale_log2 * 0x1p24f * __uint_as_float((uint32_t)max(1, 254 - up) << 23);
    float sum = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f16x8 hi;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // channels 2, 3, 6, 7 of the eight meet codes times 16
        const float y = x[g][e] * by, s = e & 2 ? y * 0.0625f : y;
        hi[e] = (_Float16)s;
        // what a lowest value meets are the queries as they are multiplied
        sum += e & 2 ? 16.f * (float)hi[e] : (float)hi[e];
      }
      q[c][g] = hi;
    }
    qsum[c] = quarters_sum(sum) * 0x1p-24f;
  }

  // The records of a block's four octets, in records from the pool's start, found through the scalar unit; a lane picks those of the octet of its key (a row of the first product) and of
  // its octet of values.  Octets outside low .. high are their neighbours: nobody sees those keys, and they may have no page.
  struct Octets {
    int r[4];
  };
  struct At {
    const uint8_t *k, *v;
  };
  __device__ __forceinline__ Octets octets(int block, int low, int high, const int* table, int kv_heads, int kvh, int shift) const {
    typedef const __attribute__((address_space(4))) int* scalar_ints;  // (this kernel does not write the table)
    const scalar_ints ids = (scalar_ints)(unsigned long long)table;
    Octets o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int oct = min(max(4 * block + j, low), high);
      o.r[j] = ((ids[oct >> shift] * kv_heads + kvh) << shift) | (oct & ((1 << shift) - 1));
    }
    return o;
  }
  static __device__ __forceinline__ int pick(const Octets& o, int j) {
    const int a = j & 1 ? o.r[1] : o.r[0], b = j & 1 ? o.r[3] : o.r[2];
    return j & 2 ? b : a;
  }
  __device__ __forceinline__ At at(const Octets& o, const uint8_t* pool) const {
    return {pool + (uint32_t)pick(o, col / 4) * (uint64_t)REC + ((col % 4) * (HD / 2) + t * (HD / 8)), pool + (uint32_t)pick(o, t) * (uint64_t)REC};
  }
  __device__ __forceinline__ void load_keys(Kv4Block<HD>& b, const At& p) const {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      if constexpr (HD == 128) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(p.k + a * 4 * (HD / 2));
        b.k[a][0] = w[0], b.k[a][1] = w[1], b.k[a][2] = w[2], b.k[a][3] = w[3];
      } else {
        const u32x2 w = *reinterpret_cast<const u32x2*>(p.k + a * 4 * (HD / 2));
        b.k[a][0] = w[0], b.k[a][1] = w[1];
      }
    }
  }
  __device__ __forceinline__ void load_values(Kv4Block<HD>& b, const At& p) const {
#pragma unroll
    for (int n = 0; n < NB; ++n) b.v[n] = *reinterpret_cast<const u32x4*>(p.v + 4 * HD + (16 * n + col) * 16);
  }
  __device__ __forceinline__ void load_marks(u32x4* m, const At& p, int of_values) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) m[i] = *reinterpret_cast<const u32x4*>(p.v + 8 * HD + 32 * of_values + 16 * i);
  }

  // From the products of 8 keys with a column of tile c to its weights, in p.  ``v_log``: about log2 of the keys' steps for values, + 127.
  __device__ __forceinline__ void soften(int c, const f32x4v* d, const float* k_step, const float* k_low, const float* v_step, const float* v_low, const float* v_log, int k0, bool mask,
                                         float* p) {
    float s[8], reach = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = fmaf(k_step[e], d[e / 4][e % 4], k_low[e] * qsum[c]);
    if (mask) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = k0 + 8 * t + e;
        s[e] = key <= kpos[c] && key >= kfirst[c] ? s[e] : -INFINITY;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) reach = fmaxf(reach, fmaf(s[e], unscale[c], v_log[e]));
    reach -= 127.f + KV4_TOP;
    if (__any(reach > R[c] + KV4_SLACK)) {
      const float want = quarters_max(reach), next = want > R[c] + KV4_SLACK ? want : R[c], base = next == -INFINITY ? 0.f : next;
      const float shrink = __builtin_amdgcn_exp2f(R[c] - base);
      R[c] = next;
      l[c] *= shrink;
      z[c] *= shrink;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[c][n][i] *= shrink;
    }
    const float base = R[c] == -INFINITY ? 0.f : R[c];
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = __builtin_amdgcn_exp2f(fmaf(s[e], unscale[c], -base));
      l[c] += w[e];
    }
    if (mask) {  // (what a column does not see may be no number)
#pragma unroll
      for (int e = 0; e < 8; ++e) z[c] += s[e] != -INFINITY ? w[e] * v_low[e] : 0.f;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) z[c] = fmaf(w[e], v_low[e], z[c]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = w[e] * v_step[e];
  }

  // The 32 keys from k0 on.  ``mask``: some column may not see all of them.  What has been used of the block is loaded anew, from ``then``, at once: a load has most
  // of a block's time to arrive, and there is one set of registers for them.
  __device__ __forceinline__ void block(Kv4Block<HD>& b, int k0, bool mask, const At& then) {
    // keys as operands
    f16x8 ka[2][EXACT ? 1 : NG];
    uint32_t kw[2][EXACT ? NG : 1];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t w = b.k[a][g], w8 = w >> 8;
        if constexpr (EXACT)
          kw[a][g] = w;
        else
          ka[a][g] = as_f16x8(kv4_ones(w), kv4_sixteens(w), kv4_ones(w8), kv4_sixteens(w8));
      }
    load_keys(b, then);
    // (with two tiles of columns, whose registers are all in use, the order that the compiler finds is the better one: 2,048 tokens at 16,000 keys 818 us, 852 with it; with one tile 1 to 2% the other way)
    if constexpr (CT == 1) __builtin_amdgcn_sched_barrier(0);
    float k_step[8], k_low[8], v_step[8], v_low[8];
    float v_log[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t km = b.km[e / 4][e % 4], vm = b.vm[e / 4][e % 4];
      k_step[e] = kv4_step(km);
      k_low[e] = kv4_low(km);
      // (what a column does not see may be anything, a place that nobody has written to in a pool that was not cleared: its weight is 0, and so is 0 times any finite number; scores and lowest values are looked at in soften)
      v_step[e] = __uint_as_float(min(vm & 0xffff0000u, 0x7f7f0000u));
      v_low[e] = kv4_low(vm);
      v_log[e] = kv4_log(v_step[e], v_low[e]);
      if (!EXACT && e >= 4) {
        v_low[e] = fmaf(15.f, v_step[e], v_low[e]);
        v_step[e] = __uint_as_float(__float_as_uint(v_step[e]) | 0x80000000u);  // the weight's sign
      }
      if constexpr (EXACT) {
        k_low[e] = fmaf(8.f, k_step[e], k_low[e]);
        v_low[e] = fmaf(8.f, v_step[e], v_low[e]);
        k_step[e] *= 0.0625f;
      }
    }
    load_marks(b.km, then, 0);
    load_marks(b.vm, then, 1);
    f16x8 p[CT];
    float p32[CT][8];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      f32x4v d[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        d[a] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          if constexpr (EXACT) {
            // bytes: channels 2, 6, 3, 7 of the eight, and 0, 4, 1, 5
            const uint32_t upper = kv4_signed(kw[a][g]), lower = kv4_signed(kw[a][g] << 4);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int e = y % 2 * 4 + y / 2;
              d[a] = __builtin_amdgcn_mfma_f32_16x16x4f32(kv4_byte(lower, y), q32[c][g][e], d[a], 0, 0, 0);
              d[a] = __builtin_amdgcn_mfma_f32_16x16x4f32(kv4_byte(upper, y), q32[c][g][e + 2], d[a], 0, 0, 0);
            }
          } else {
            d[a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[a][g], q[c][g], d[a], 0, 0, 0);
          }
        }
      }
      soften(c, d, k_step, k_low, v_step, v_low, v_log, k0, mask, p32[c]);
      if constexpr (!EXACT)
#pragma unroll
        for (int e = 0; e < 8; ++e) p[c][e] = (_Float16)p32[c][e];
      __builtin_amdgcn_sched_barrier(0);
    }
    // values as operands, four channels of each 64 a lane
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      u32x4 w = b.v[n];
      if constexpr (EXACT) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          // bytes: channels 1 and 3 of key 2 x, then of 2 x + 1; channels 0 and 2
          const uint32_t upper = kv4_signed(w[x]), lower = kv4_signed(w[x] << 4);
#pragma unroll
          for (int y = 0; y < 4; ++y)
#pragma unroll
            for (int c = 0; c < CT; ++c) {
              f32x4v* to = o[c][n] + y % 2 * 2;
              to[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kv4_byte(lower, y), p32[c][2 * x + y / 2], to[0], 0, 0, 0);
              to[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kv4_byte(upper, y), p32[c][2 * x + y / 2], to[1], 0, 0, 0);
            }
        }
        continue;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t r[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t y = i >= 2 ? w[x] >> 8 : w[x];
          r[x] = i & 1 ? kv4_sixteens(x < 2 ? y : ~y) : kv4_ones(x < 2 ? y : ~y);  // the last four keys' as 15 - u
        }
        const f16x8 va = as_f16x8(r[0], r[1], r[2], r[3]);
#pragma unroll
        for (int c = 0; c < CT; ++c) o[c][n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, p[c], o[c][n][i], 0, 0, 0);
        if (i & 1) __builtin_amdgcn_sched_barrier(0);
      }
    }
    load_values(b, then);
  }

  // Blocks b0, b0 + by, .. before b1 of 32 keys; columns of tile c see keys kfirst[c] .. kpos[c] of their lane.  ``whole0`` .. ``whole1``: blocks that every column sees whole.
  __device__ __forceinline__ void walk(int b0, int b1, int by, int whole0, int whole1, int low, int high, const int* table, const uint8_t* pool, int kv_heads, int kvh,
                                       int shift) {
    if (b0 >= b1) return;
    Kv4Block<HD> held;
    const At to = at(octets(b0, low, high, table, kv_heads, kvh, shift), pool);
    load_keys(held, to), load_marks(held.km, to, 0), load_marks(held.vm, to, 1), load_values(held, to);
    Octets next = octets(b0 + by, low, high, table, kv_heads, kvh, shift);  // (ids a block ahead of the loads)
    for (int b = b0; b < b1; b += by) {
      const At then = at(next, pool);
      next = octets(b + 2 * by, low, high, table, kv_heads, kvh, shift);
      block(held, 32 * b, b < whole0 || b >= whole1, then);
    }
  }

  // this lane's share of column c's result: channels 64 n + 16 t + {0 .. 15} as out(n, 4 r + i), and log2 of the column's weight
  __device__ __forceinline__ float weight(int c, float& total, float& low) const {
    total = quarters_sum(l[c]);
    low = quarters_sum(z[c]);
    return total == 0.f ? -INFINITY : R[c] + __log2f(total);
  }
  __device__ __forceinline__ float sum_of(int c, int n, int e) const { return (EXACT ? 0.0625f : e & 1 ? 0x1p20f : 0x1p24f) * o[c][n][e % 4][e / 4]; }
};

// Single tokens: a workgroup a (token, key/value head, 16 query heads of its group, range of keys), whose waves take blocks of 32 keys in turn and meet in LDS.  Ranges are even and as many
// as give ``a.groups`` workgroups over all tokens: a row twice as long as others has twice as many.
// Bound by memory where the rows are long and many (61 rows of 200 to 12,000 keys, 8 key/value heads of 128 channels: 96 us, 4.2 TB/s; 64 rows of 6,000: 90 us, 4.65), by one workgroup's
// chain of loads where they are few (a row of 1,000, in eight waves: 8.9 us).  Two blocks on their way at a time were slower everywhere (their registers cost a wave a SIMD).
template <typename T, int HD, bool EXACT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) __attribute__((amdgpu_waves_per_eu(3))) void attn_kv4_rows_kernel(const Kv4AttnParams a) {
  typedef Kv4Wave<T, HD, 1, EXACT> Wave;
  __shared__ float outs[WAVES][16][HD + 4];
  __shared__ float weights[WAVES][16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / NS_WAVE);
  const int group = a.heads / a.kv_heads, hblks = (group + 15) / 16, ny = a.kv_heads * hblks;
  const int y = blockIdx.x, tile = blockIdx.y, split = blockIdx.z, kvh = hblks == 1 ? y : y / hblks, head0 = kvh * group + (y - kvh * hblks) * 16;
  const int heads = min(16, (kvh + 1) * group - head0);
  const int* info = a.tiles + (size_t)tile * KV4_TILE_INTS;
  const int req = info[0], t0 = info[1], row = info[2] + t0, n = info[3], kv = info[4], all = info[6];
  if (t0 >= n) return;
  const int pos = kv - n + t0, first = a.window ? max(0, pos - a.window + 1) : 0, shift = 31 - __clz(a.page) - 3;
  const int b0 = first / 32, blocks = pos / 32 + 1 - b0;
  // (quotients by reciprocals: a share that is one block too long does no harm, and the same for all of a row's ranges)
  const float every = (float)ny * (a.window ? fminf((float)all, (float)a.n_tiles * (float)(a.window / 32 + 2)) : (float)all);
  const float wanted = fmaxf((float)KV4_RANGE_BLOCKS, every * __builtin_amdgcn_rcpf((float)a.groups)), ranges = fminf((float)a.splits, ceilf((float)blocks * __builtin_amdgcn_rcpf(wanted)));
  const int share = __builtin_amdgcn_readfirstlane((int)((float)blocks * __builtin_amdgcn_rcpf(fmaxf(ranges, 1.f))) + 1);
  if (split * share >= blocks) {
    if ((int)threadIdx.x < heads) a.part_l[((size_t)tile * a.heads + head0 + threadIdx.x) * a.splits + split] = -INFINITY;
    return;
  }
  const bool whole = share >= blocks;
  const int from = b0 + split * share, to = min(b0 + blocks, from + share);
  Wave w;
  w.init();
  w.kpos[0] = pos, w.kfirst[0] = first;
  w.query(0, w.col < heads ? (const T*)a.q + (size_t)row * a.q_stride + (head0 + w.col) * HD : nullptr, a.scale_log2, a.wide);
  w.walk(from + wave, to, WAVES, (first + 31) / 32, (pos + 1) / 32, first / 8, pos / 8, a.block_table + (size_t)req * a.table_stride, a.pool, a.kv_heads, kvh, shift);
  float total, low;
  const float weight = w.weight(0, total, low), inv = total == 0.f ? 0.f : 1.f / total;
  if (w.t == 0) weights[wave][w.col] = weight;
  if (w.col < heads) {
#pragma unroll
    for (int nb = 0; nb < Wave::NB; ++nb)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        f32x4v x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (w.sum_of(0, nb, e + i) + low) * inv;
        *reinterpret_cast<f32x4v*>(&outs[wave][w.col][64 * nb + 16 * w.t + e]) = x;
      }
  }
  __syncthreads();
  const size_t pc0 = ((size_t)tile * a.heads + head0) * a.splits;
  for (int i = threadIdx.x; i < heads * (HD / 4); i += WAVES * 64) {
    const int c = i / (HD / 4), ch = i % (HD / 4) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) top = fmaxf(top, weights[v][c]);
    const float base = top == -INFINITY ? 0.f : top;
    f32x4v sum = {0.f, 0.f, 0.f, 0.f};
    float every_weight = 0.f, x[WAVES];
#pragma unroll
    for (int v = 0; v < WAVES; ++v) x[v] = __builtin_amdgcn_exp2f(weights[v][c] - base), every_weight += x[v];
    const float by = every_weight == 0.f ? 0.f : 1.f / every_weight;
#pragma unroll
    for (int v = 0; v < WAVES; ++v)  // (a mean of means: no sum is larger than they are.  A wave without weight may hold no number: who sees such a value has none, however small its weight)
      sum += (x[v] * by) * *reinterpret_cast<const f32x4v*>(&outs[v][c][ch]);
    const size_t pc = pc0 + (size_t)c * a.splits + split;
    if (whole) {
      typedef T vec_t __attribute__((ext_vector_type(4)));
      vec_t r;
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = from_f<T>(sum[e]);
      *reinterpret_cast<vec_t*>((T*)a.out + ((size_t)row * a.heads + head0 + c) * HD + ch) = r;
      if (a.splits > 1 && ch == 0) a.part_l[pc] = KV4_WHOLE;  // (the second kernel leaves the row alone)
    } else {
      *reinterpret_cast<f32x4v*>(a.part_o + pc * HD + ch) = sum;
      if (ch == 0) a.part_l[pc] = every_weight == 0.f ? -INFINITY : base + __log2f(every_weight);
    }
  }
}

// The results of a wave's columns, ``tokens`` tokens of a head from row ``row`` on, ``whole`` or as a range of theirs (``column``: its first token among all tiles').
template <typename T, int HD, int CT, class Wave>
__device__ __forceinline__ void kv4_columns_out(const Wave& w, const Kv4AttnParams& a, int row, int tokens, int column, int head, int split, bool whole) {
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    float total, low;
    const float weight = w.weight(c, total, low), inv = total == 0.f ? 0.f : 1.f / total;
    const int token = 16 * c + w.col;
    if (token >= tokens) continue;
    const size_t pc = (((size_t)column + token) * a.heads + head) * a.splits + split;
    if (whole) {
      if (a.splits > 1 && w.t == 0) a.part_l[pc] = KV4_WHOLE;
      T* to_ = (T*)a.out + ((size_t)(row + token) * a.heads + head) * HD;
#pragma unroll
      for (int nb = 0; nb < Wave::NB; ++nb) {
        typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T))));
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int e0 = 0; e0 < 16; e0 += V) {
          vec_t r;
#pragma unroll
          for (int e = 0; e < V; ++e) r[e] = from_f<T>((w.sum_of(c, nb, e0 + e) + low) * inv);
          *reinterpret_cast<vec_t*>(to_ + 64 * nb + 16 * w.t + e0) = r;
        }
      }
    } else {
#pragma unroll
      for (int nb = 0; nb < Wave::NB; ++nb)
#pragma unroll
        for (int e0 = 0; e0 < 16; e0 += 4) {
          f32x4v r;
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] = (w.sum_of(c, nb, e0 + e) + low) * inv;
          *reinterpret_cast<f32x4v*>(a.part_o + pc * HD + 64 * nb + 16 * w.t + e0) = r;
        }
      if (w.t == 0) a.part_l[pc] = weight;
    }
  }
}

// Portions: a wave 16 CT tokens of a head, four waves a workgroup that share nothing but their place.
// Bound by vector instructions: a block of 32 keys and 32 columns of 128 channels has 32 matrix instructions (512 cycles) and 355 others (counted; 1,610 cycles), of which 80 make operands of the
// codes and 16 are exponentials; they are under way 84% of the time.  2,048 tokens at 16,000 keys: 811 us, 704 TFLOP/s; 2,048 at none, 16 columns a wave, 72 us.  Four tiles of columns a wave (each operand made
// for twice as many) leave one wave a SIMD and nothing to fill its waits: 1,203 and 149 us.  Operands made by four waves for each other, by way of LDS, with a barrier a block: 828 and 90, where these took 772 and 75.
template <typename T, int HD, int CT, bool EXACT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void attn_kv4_tiles_kernel(const Kv4AttnParams a) {
  typedef Kv4Wave<T, HD, CT, EXACT> Wave;
  constexpr int TOKENS = 16 * CT, PIECES = KV4_TILE_TOKENS / TOKENS;  // of a wave; of a tile
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / NS_WAVE);
  // (late tiles see the most keys: they begin first)
  const int item = blockIdx.x * 4 + wave, columns = a.heads * PIECES, tile = a.n_tiles - 1 - item / (columns * a.splits), rest = item % (columns * a.splits);
  const int split = rest / columns, head = rest % columns / PIECES, piece = rest % PIECES;
  if (tile < 0) return;
  const int kvh = head / (a.heads / a.kv_heads);
  const int* info = a.tiles + (size_t)tile * KV4_TILE_INTS;
  const int req = info[0], t0 = info[1] + piece * TOKENS, row0 = info[2], n = info[3], kv = info[4];
  if (t0 >= n) return;
  const int tokens = min(TOKENS, n - t0), pos0 = kv - n + t0, last = pos0 + tokens - 1, shift = 31 - __clz(a.page) - 3;
  const int first = a.window ? max(0, pos0 - a.window + 1) : 0, first_of_last = a.window ? max(0, last - a.window + 1) : 0;
  // (ranges are chosen on the host for the most keys that a portion may have, in a captured step those of its table; of fewer keys there are as many ranges as are worth joining)
  const int b0 = first / 32, blocks = last / 32 + 1 - b0, share = a.splits == 1 ? blocks : max((blocks + a.splits - 1) / a.splits, KV4_PORTION_BLOCKS);
  const int column = tile * KV4_TILE_TOKENS + piece * TOKENS;
  if (split * share >= blocks) {  // nothing to do: neither queries nor keys are read, and no result is written
    for (int i = threadIdx.x % NS_WAVE; i < tokens; i += NS_WAVE) a.part_l[(((size_t)column + i) * a.heads + head) * a.splits + split] = -INFINITY;
    return;
  }
  const int from = b0 + split * share, to = min(b0 + blocks, from + share);
  Wave w;
  w.init();
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int token = min(16 * c + w.col, tokens - 1);  // (beyond the last: the last once more, not written)
    w.kpos[c] = pos0 + token;
    w.kfirst[c] = a.window ? max(0, pos0 + token - a.window + 1) : 0;
    w.query(c, (const T*)a.q + (size_t)(row0 + t0 + token) * a.q_stride + head * HD, a.scale_log2, a.wide);
  }
  w.walk(from, to, 1, (first_of_last + 31) / 32, (pos0 + 1) / 32, first / 8, last / 8, a.block_table + (size_t)req * a.table_stride, a.pool, a.kv_heads, kvh, shift);
  kv4_columns_out<T, HD, CT>(w, a, row0 + t0, tokens, column, head, split, share >= blocks);
}
