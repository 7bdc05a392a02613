// Attention over 4-bit pages on the matrix cores, head sizes 64 and 128.  Included by attn_kv4.hip.
//
// A wave walks 32 keys at a time with CT tiles of 16 columns, a column a (token, query head) pair of one request and key/value head:
//   S^T[key][col] = K[key][:] . Q[col][:]          A = 16 keys, B = the columns' queries
//   O^T[channel][col] += V^T[channel][key] . P^T   A = 16 channels, B = the columns' weights, in the layout that S^T came out in
// Keys go to the rows of the first product in the order that makes its result the second's operand: row 4 t + r of tile a is key 8 t + 4 a + r of
// the 32, so that lane (col, t) holds the weights of keys 8 t .. 8 t + 7, one octet, whose values and marks it reads in whole records.
// Nothing passes through LDS on the way (a wave's operands are 4.25 bits a value, from L2): the waves need no barriers.
//
// From codes to operands.  Float16 of 1,024 + u has u in its lowest four bits, and of 1,024 + 16 u in the next four: a mask and an or make two
// codes at a time, and the queries' channels at the second kind of place carry a factor of 1/16, exactly.  The 1,024s are taken off in the first
// sum: it starts at -1,024 times the sum of the queries.  That rounds at 2^-24 of 1,024 |q|, 2^-14 of a step of the key, less than bfloat16
// queries hold; float32 (PARTS 2) and the values, whose sums over many keys that may cancel, take it off before (codes of -8 .. 7, exactly).
//   s = step (q . u) + low sum(q):      two operations a score, as both are a key's
//   out = sum p step (u - 8) + sum p (low + 8 step):   p step is the weight in the second product, the rest a sum of numbers
// Queries are float16 on their way in, scaled by a power of two of their own so that the largest lies at 256: what is 2^-22 of it is exact.  Weights are
// rounded to float16 (2^-12 of themselves).  PARTS 2: queries and weights as the sum of two float16 values each, two products for one.
//
// The soft-max's reference R is one number a column for weights and steps together: R >= (largest score so far) + (exponent of the steps seen) - 8, so
// that p step, p = 2^(s - R), fits float16 whatever the steps' size, and is only raised when that no longer holds (then every sum shrinks).
// It knows of the keys that the column sees, and of no others.
#pragma once

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

#define KV4_TILE_INTS 8
#define KV4_TILE_TOKENS 32  // of a portion's tile
#define KV4_SLACK 8.f

__device__ __forceinline__ f16x8 as_f16x8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __builtin_bit_cast(f16x8, u32x4{a, b, c, d}); }
// two codes of a dword as 1,024 + u, and as 1,024 + 16 u
// (one instruction: the compiler makes two of it, as an instruction may name one constant only, and the other has to be in a register of its own)
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t set) {
  uint32_t r;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(mask), "v"(set));
  return r;
}
__device__ __forceinline__ uint32_t kv4_ones(uint32_t w) { return and_or(w, 0x000f000fu, 0x64006400u); }
__device__ __forceinline__ uint32_t kv4_sixteens(uint32_t w) { return and_or(w, 0x00f000f0u, 0x64006400u); }
// the same less 1,024 and 8 (128): u - 8, 16 (u - 8)
__device__ __forceinline__ uint32_t kv4_centred(uint32_t w, bool sixteens) {
  const _Float16 off = sixteens ? (_Float16)-1152.f : (_Float16)-1032.f;
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, w) + f16x2{off, off});
}
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

// CT: tiles of 16 columns.  PARTS: 1 for bfloat16, 2 for float32.
template <typename T, int HD, int CT, int PARTS>
struct Kv4Wave {
  static constexpr int NG = HD / 32, NB = HD / 64;
  static constexpr int REC = 8 * HD + 64;
  f16x8 q[CT][PARTS][NG];
  float qsum[CT], unscale[CT];  // sum of the scaled queries; scale * log2(e) and the queries' own scale taken off
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

  // this lane's column of tile c: its query's channels (nullptr: a column of zeros)
  __device__ __forceinline__ void query(int c, const T* from, float scale_log2) {
    float x[NG][8], most = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[g][e] = from ? to_f(from[32 * g + 8 * t + e]) : 0.f;
        most = fmaxf(most, fabsf(x[g][e]));
      }
    most = quarters_max(most);
    // 2^(8 - exponent): exact; nothing to scale in zeros and where the largest is infinite (the products are then no numbers by themselves)
    const int ex = (int)(__float_as_uint(most) >> 23);
    const int up = ex == 0 || ex == 255 ? 127 : min(max(127 + 127 + 8 - ex, 1), 254);
    const float by = __uint_as_float((uint32_t)up << 23);
    unscale[c] = scale_log2 * __uint_as_float((uint32_t)max(1, 254 - up) << 23);
    float sum = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f16x8 hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // channels 2, 3, 6, 7 of the eight meet codes times 16
        const float y = x[g][e] * by, s = e & 2 ? y * 0.0625f : y;
        hi[e] = (_Float16)s;
        lo[e] = (_Float16)(s - (float)hi[e]);
        // what is taken off, and what a lowest value meets, are the queries as they are multiplied
        sum += PARTS == 1 ? (e & 2 ? 16.f * (float)hi[e] : (float)hi[e]) : y;
      }
      q[c][0][g] = hi;
      if constexpr (PARTS == 2) q[c][1][g] = lo;
    }
    qsum[c] = quarters_sum(sum);
  }
  // -1,024 times the sum of what the first product multiplies (channels with a factor of 1/16 count as such)
  __device__ __forceinline__ float start(int c) const {
    float s = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += (float)q[c][0][g][e];
    return -1024.f * quarters_sum(s);
  }

  // records of the octet of this lane's key (a row of the first product) and of its octet of values, of the 32 keys from ``k0`` on
  struct At {
    const uint8_t *k, *v;
  };
  // ``low``, ``high``: the first and the last octet that may be read (outside them their neighbours are: nobody sees those keys)
  __device__ __forceinline__ void pages_of(int k0, int low, int high, const int* table, int shift, int& pk, int& pv) const {
    const int ok = min(max(k0 / 8 + col / 4, low), high), ov = min(max(k0 / 8 + t, low), high);
    pk = table[ok >> shift];
    pv = table[ov >> shift];
  }
  __device__ __forceinline__ At at(int k0, int low, int high, int pk, int pv, const uint8_t* pool, int kv_heads, int kvh, int shift) const {
    const int ok = min(max(k0 / 8 + col / 4, low), high), ov = min(max(k0 / 8 + t, low), high), mask = (1 << shift) - 1;
    return {pool + ((((size_t)pk * kv_heads + kvh) << shift) + (ok & mask)) * REC + (col % 4) * (HD / 2) + t * (HD / 8),
            pool + ((((size_t)pv * kv_heads + kvh) << shift) + (ov & mask)) * REC};
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

  // The 32 keys from k0 on.  ``mask``: some column may not see all of them.  What has been used of the block is loaded anew, from ``then``, at once: a load has most
  // of a block's time to arrive, and there is one set of registers for them.
  __device__ __forceinline__ void block(Kv4Block<HD>& b, int k0, bool mask, const float* cinit, const At& then) {
    // keys as operands
    f16x8 ka[2][NG];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t w = b.k[a][g], w8 = w >> 8;
        uint32_t r0 = kv4_ones(w), r1 = kv4_sixteens(w), r2 = kv4_ones(w8), r3 = kv4_sixteens(w8);
        if constexpr (PARTS == 2) r0 = kv4_centred(r0, false), r1 = kv4_centred(r1, true), r2 = kv4_centred(r2, false), r3 = kv4_centred(r3, true);
        ka[a][g] = as_f16x8(r0, r1, r2, r3);
      }
    load_keys(b, then);
    __builtin_amdgcn_sched_barrier(0);
    f16x8 p[CT][PARTS];
    float k_step[8], k_low[8], v_step[8], v_mid[8];
    uint32_t v_mark[8], most_of = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t km = b.km[e / 4][e % 4], vm = b.vm[e / 4][e % 4];
      k_step[e] = kv4_step(km);
      k_low[e] = PARTS == 1 ? kv4_low(km) : fmaf(8.f, k_step[e], kv4_low(km));
      v_mark[e] = vm;
      v_step[e] = kv4_step(vm);
      v_mid[e] = fmaf(8.f, v_step[e], kv4_low(vm));
      most_of = max(most_of, vm);
    }
    load_marks(b.km, then, 0);
    load_marks(b.vm, then, 1);
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      f32x4v d[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const float from = PARTS == 1 ? cinit[c] : 0.f;
        d[a] = f32x4v{from, from, from, from};
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int h = 0; h < PARTS; ++h) d[a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[a][g], q[c][h][g], d[a], 0, 0, 0);
      }
      float s[8], top = -INFINITY;
      uint32_t most = most_of;
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = fmaf(k_step[e], d[e / 4][e % 4], k_low[e] * qsum[c]) * unscale[c];
      if (mask) {
        most = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int key = k0 + 8 * t + e;
          const bool seen = key <= kpos[c] && key >= kfirst[c];
          s[e] = seen ? s[e] : -INFINITY;
          most = max(most, seen ? v_mark[e] : 0u);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, s[e]);
      // the exponent above the largest step, at least -64 (smaller ones lose what float16 does not hold of them)
      const float reach = top + fmaxf((float)(int)(most >> 23) - 126.f, -64.f);
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
        w[e] = __builtin_amdgcn_exp2f(s[e] - base);
        l[c] += w[e];
      }
      if (mask) {  // (what a column does not see may be no number)
#pragma unroll
        for (int e = 0; e < 8; ++e) z[c] += s[e] != -INFINITY ? w[e] * v_mid[e] : 0.f;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) z[c] = fmaf(w[e], v_mid[e], z[c]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float ps = w[e] * v_step[e];
        p[c][0][e] = (_Float16)ps;
        if constexpr (PARTS == 2) p[c][1][e] = (_Float16)(ps - (float)p[c][0][e]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    // values as operands, four channels of each 64 a lane
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      u32x4 w = b.v[n];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t r[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t y = i >= 2 ? w[x] >> 8 : w[x];
          r[x] = kv4_centred(i & 1 ? kv4_sixteens(y) : kv4_ones(y), i & 1);
        }
        const f16x8 va = as_f16x8(r[0], r[1], r[2], r[3]);
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
          for (int h = 0; h < PARTS; ++h) o[c][n][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, p[c][h], o[c][n][i], 0, 0, 0);
        if (i & 1) __builtin_amdgcn_sched_barrier(0);
      }
    }
    load_values(b, then);
  }

  // Blocks b0, b0 + by, .. before b1 of 32 keys; columns of tile c see keys kfirst[c] .. kpos[c] of their lane.  ``whole0`` .. ``whole1``: blocks that every column sees whole.
  __device__ __forceinline__ void walk(int b0, int b1, int by, int whole0, int whole1, int low, int high, const int* table, const uint8_t* pool, int kv_heads, int kvh,
                                       int shift) {
    if (b0 >= b1) return;
    float cinit[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) cinit[c] = PARTS == 1 ? start(c) : 0.f;
    Kv4Block<HD> now;
    int pk, pv;
    pages_of(32 * b0, low, high, table, shift, pk, pv);
    const At first = at(32 * b0, low, high, pk, pv, pool, kv_heads, kvh, shift);
    pages_of(32 * (b0 + by), low, high, table, shift, pk, pv);
    load_keys(now, first), load_marks(now.km, first, 0), load_marks(now.vm, first, 1), load_values(now, first);
    for (int b = b0; b < b1; b += by) {
      const At then = at(32 * (b + by), low, high, pk, pv, pool, kv_heads, kvh, shift);
      pages_of(32 * (b + 2 * by), low, high, table, shift, pk, pv);
      block(now, 32 * b, b < whole0 || b >= whole1, cinit, then);
    }
  }

  // this lane's share of column c's result: channels 64 n + 16 t + {0 .. 15} as out(n, 4 r + i), and log2 of the column's weight
  __device__ __forceinline__ float weight(int c, float& total, float& low) const {
    total = quarters_sum(l[c]);
    low = quarters_sum(z[c]);
    return total == 0.f ? -INFINITY : R[c] + __log2f(total);
  }
  __device__ __forceinline__ float sum_of(int c, int n, int e) const { return (e & 1 ? 0.0625f : 1.f) * o[c][n][e % 4][e / 4]; }
};

// Single tokens: a workgroup a (token, key/value head, 16 query heads of its group, range of keys), whose four waves take blocks of 32 keys in turn and meet in LDS.
template <typename T, int HD, int PARTS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PARTS == 2 ? 2 : 3))) void attn_kv4_rows_kernel(const Kv4AttnParams a) {
  typedef Kv4Wave<T, HD, 1, PARTS> Wave;
  __shared__ float outs[4][16][HD + 4];
  __shared__ float weights[4][16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / NS_WAVE);
  const int group = a.heads / a.kv_heads, hblks = (group + 15) / 16, ny = a.kv_heads * hblks;
  const int y = blockIdx.x % ny, tile = blockIdx.x / ny, split = blockIdx.y, kvh = y / hblks, head0 = kvh * group + y % hblks * 16;
  const int heads = min(16, (kvh + 1) * group - head0);
  const int* info = a.tiles + (size_t)tile * KV4_TILE_INTS;
  const int req = info[0], t0 = info[1], row = info[2] + t0, n = info[3], kv = info[4];
  if (t0 >= n) return;
  const int pos = kv - n + t0, first = a.window ? max(0, pos - a.window + 1) : 0, shift = 31 - __clz(a.page) - 3;
  const int b0 = first / 32, blocks = pos / 32 + 1 - b0, share = (blocks + a.splits - 1) / a.splits;
  const int from = b0 + split * share, to = min(b0 + blocks, from + share);
  Wave w;
  w.init();
  w.kpos[0] = pos, w.kfirst[0] = first;
  w.query(0, w.col < heads ? (const T*)a.q + (size_t)row * a.q_stride + (head0 + w.col) * HD : nullptr, a.scale_log2);
  w.walk(from + wave, to, 4, (first + 31) / 32, (pos + 1) / 32, first / 8, pos / 8, a.block_table + (size_t)req * a.table_stride, a.pool, a.kv_heads, kvh, shift);
  float total, low;
  const float weight = w.weight(0, total, low), inv = total == 0.f ? 0.f : 1.f / total;
  if (w.t == 0) weights[wave][w.col] = weight;
#pragma unroll
  for (int nb = 0; nb < Wave::NB; ++nb)
#pragma unroll
    for (int e = 0; e < 16; ++e) outs[wave][w.col][64 * nb + 16 * w.t + e] = (w.sum_of(0, nb, e) + low) * inv;
  __syncthreads();
  for (int i = threadIdx.x; i < heads * HD; i += 256) {
    const int c = i / HD, ch = i % HD;
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < 4; ++v) top = fmaxf(top, weights[v][c]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, all = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float x = exp2f(weights[v][c] - base);
      all += x;
      sum += x == 0.f ? 0.f : x * outs[v][c][ch];
    }
    const float r = all == 0.f ? 0.f : sum / all;
    if (a.splits == 1) {
      ((T*)a.out)[((size_t)row * a.heads + head0 + c) * HD + ch] = from_f<T>(r);
    } else {
      const size_t pc = ((size_t)tile * a.heads + head0 + c) * a.splits + split;
      a.part_o[pc * HD + ch] = r;
      if (ch == 0) a.part_l[pc] = all == 0.f ? -INFINITY : base + log2f(all);
    }
  }
}

// Portions: a wave 32 tokens of CT / 2 heads of a group, four waves a workgroup that share nothing but their place.
template <typename T, int HD, int CT, int PARTS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(CT == 2 && !(PARTS == 2 && HD == 128) ? 2 : 1))) void attn_kv4_tiles_kernel(const Kv4AttnParams a) {
  typedef Kv4Wave<T, HD, CT, PARTS> Wave;
  constexpr int HEADS = CT / 2;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / NS_WAVE);
  const int group = a.heads / a.kv_heads, hblks = (group + HEADS - 1) / HEADS, ny = a.kv_heads * hblks;
  // (late tiles see the most keys: they begin first)
  const long long item = (long long)blockIdx.x * 4 + wave, per = (long long)ny * a.splits;
  const int tile = a.n_tiles - 1 - (int)(item / per), rest = (int)(item % per), split = rest / ny, y = rest % ny;
  if (tile < 0) return;
  const int kvh = y / hblks, head0 = kvh * group + y % hblks * HEADS, heads = min(HEADS, (kvh + 1) * group - head0);
  const int* info = a.tiles + (size_t)tile * KV4_TILE_INTS;
  const int req = info[0], t0 = info[1], row0 = info[2], n = info[3], kv = info[4];
  if (t0 >= n) return;
  const int tokens = min(KV4_TILE_TOKENS, n - t0), pos0 = kv - n + t0, last = pos0 + tokens - 1, shift = 31 - __clz(a.page) - 3;
  const int first = a.window ? max(0, pos0 - a.window + 1) : 0, first_of_last = a.window ? max(0, last - a.window + 1) : 0;
  const int b0 = first / 32, blocks = last / 32 + 1 - b0, share = (blocks + a.splits - 1) / a.splits;
  const int from = b0 + split * share, to = min(b0 + blocks, from + share);
  Wave w;
  w.init();
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int token = min(16 * (c % 2) + w.col, tokens - 1);  // (beyond the last: the last once more, not written)
    w.kpos[c] = pos0 + token;
    w.kfirst[c] = a.window ? max(0, pos0 + token - a.window + 1) : 0;
    w.query(c, c / 2 < heads ? (const T*)a.q + (size_t)(row0 + t0 + token) * a.q_stride + (head0 + c / 2) * HD : nullptr, a.scale_log2);
  }
  w.walk(from, to, 1, (first_of_last + 31) / 32, (pos0 + 1) / 32, first / 8, last / 8, a.block_table + (size_t)req * a.table_stride, a.pool, a.kv_heads, kvh, shift);
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    float total, low;
    const float weight = w.weight(c, total, low), inv = total == 0.f ? 0.f : 1.f / total;
    const int token = 16 * (c % 2) + w.col, head = head0 + c / 2;
    if (token >= tokens || c / 2 >= heads) continue;
    if (a.splits == 1) {
      T* to_ = (T*)a.out + ((size_t)(row0 + t0 + token) * a.heads + head) * HD;
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
      const size_t pc = (((size_t)tile * KV4_TILE_TOKENS + token) * a.heads + head) * a.splits + split;
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
