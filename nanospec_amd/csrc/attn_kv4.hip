// Soft-max attention over pages that hold keys and values in 4 bits (kv4.h):
//   s = scale * q . (step_k u_k + low_k) = scale * (step_k (q . u_k) + low_k sum(q));   p = softmax(s) over the keys that a query sees;
//   out = sum p (step_v u_v + low_v)
// A query at position i sees keys max(0, i - window + 1) .. i (window 0: all).  Scores, soft-max and sums are 32-bit.
// The keys of a query may be cut into ranges, which leave a result of their own each, with the logarithm of its weight, for a second kernel.
// (reference: model/attention.py:22-43 for what is computed, over pages in the model's precision)
#include "kv4.h"

#define KV4_WHOLE INFINITY  // in part_l: the column's result has been written, there is nothing to join.  (No range's own: its weight is a finite number or none.)

struct Kv4AttnParams {
  void* out;        // [tokens, heads, hd]
  float* part_o;    // [columns][splits][hd]: a range's result          (splits > 1)
  float* part_l;    // [columns][splits]: log2 of its weight, -inf of an empty range, KV4_WHOLE
  const void* q;    // row t at q + t * q_stride, head h at + h * hd
  const uint8_t* pool;
  const int *tiles, *token_req, *positions, *block_table;
  int q_stride, table_stride, n_tiles, heads, kv_heads, hd, page, splits, window, groups;  // groups: workgroups that share single tokens' keys
  float scale_log2;  // softmax scale * log2(e)
  int wide;          // every query begins at a multiple of 16 bytes
};

// ------------------------------------------------------------------------------------------------------------------------------------
// Any head size that is a multiple of 32: a workgroup a (token, head, range of keys); its four waves take blocks of 64 keys in turn, a lane
// a key for the scores, then a lane a channel (and up to four) for the values.  All arithmetic is plain 32-bit.
#define KV4_PLAIN_TOP 32.f  // the largest weight is 2^-32, so that sums of weights times values fit 32 bits where the values do
template <typename T, int CH>  // CH: channels of a lane, hd <= 64 CH
__global__ __launch_bounds__(256) void attn_kv4_plain_kernel(const Kv4AttnParams a) {
  __shared__ float qs[KV4_MAX_HD];
  __shared__ float sums[4][3];
  __shared__ float outs[4][KV4_MAX_HD];
  const int lane = threadIdx.x % NS_WAVE, wave = threadIdx.x / NS_WAVE;
  const int t = blockIdx.x / a.heads, head = blockIdx.x % a.heads, split = blockIdx.y;
  const int kvh = head / (a.heads / a.kv_heads), hd = a.hd, groups = hd / 32, octets = a.page / KV4_TOKENS, record = kv4_record(hd);
  const int pos = a.positions[t], first = a.window ? max(0, pos - a.window + 1) : 0;
  const int* table = a.block_table + (size_t)a.token_req[t] * a.table_stride;
  const T* q = (const T*)a.q + (size_t)t * a.q_stride + head * hd;
  float qsum = 0.f;
  for (int c = threadIdx.x; c < hd; c += blockDim.x) {
    const int g = c / 32, o = c % 32 / 8;
    qs[(o * groups + g) * 8 + c % 8] = to_f(q[c]);  // in the order of a key's dwords
  }
  __syncthreads();
  for (int c = 0; c < hd; ++c) qsum += qs[c];
  // blocks of 64 keys, and this range's share of them
  const int b0 = first / 64, blocks = pos / 64 + 1 - b0, share = (blocks + a.splits - 1) / a.splits;
  const int from = b0 + split * share, to = min(b0 + blocks, from + share);
  float m = -INFINITY, l = 0.f, z = 0.f, acc[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) acc[c] = 0.f;
  for (int b = from + wave; b < to; b += 4) {
    const int key = 64 * b + lane;
    const bool seen = key >= first && key <= pos;
    const int at = min(max(key, first), pos), oct = at / KV4_TOKENS, j = at % KV4_TOKENS;
    const uint8_t* rec = a.pool + kv4_at(table[oct / octets], a.kv_heads, kvh, octets, oct % octets) * record;
    const uint32_t* kw = reinterpret_cast<const uint32_t*>(rec + j * (hd / 2));
    float dot = 0.f;
    for (int i = 0; i < hd / 8; ++i) {
      const uint32_t w = kw[i];
#pragma unroll
      for (int e = 0; e < 8; ++e) dot = fmaf(qs[8 * i + e], (float)(w >> (4 * (e / 2) + 16 * (e % 2)) & 15u), dot);
    }
    const uint32_t km = reinterpret_cast<const uint32_t*>(rec + kv4_marks_at(hd))[j], vm = reinterpret_cast<const uint32_t*>(rec + kv4_marks_at(hd))[KV4_TOKENS + j];
    const float s = seen ? (kv4_step(km) * dot + kv4_low(km) * qsum) * a.scale_log2 : -INFINITY;
    const float top = fmaxf(m, wave_max(s)), base = top == -INFINITY ? 0.f : top, shrink = exp2f(m - base);
    const float p = exp2f(s - base - KV4_PLAIN_TOP), ps = seen ? p * kv4_step(vm) : 0.f;
    l = l * shrink + p;
    z = z * shrink + (seen ? p * fmaf(8.f, kv4_step(vm), kv4_low(vm)) : 0.f);  // (codes less 8: the two sums would be many times their own)
    m = top;
#pragma unroll
    for (int c = 0; c < CH; ++c) acc[c] *= shrink;
    for (int o = 0; o < 8; ++o) {  // the block's octets
      const int k0 = 64 * b + 8 * o;
      if (k0 > pos || k0 + 7 < first) continue;
      const int vo = k0 / KV4_TOKENS;
      const uint8_t* vr = a.pool + kv4_at(table[vo / octets], a.kv_heads, kvh, octets, vo % octets) * record + kv4_values_at(hd);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int ch = min(lane + 64 * c, hd - 1);
        const uint4 w = *reinterpret_cast<const uint4*>(vr + ch / 4 * 16);
        const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[c] = fmaf(__shfl(ps, 8 * o + e, NS_WAVE), (float)((int)(d[e / 2] >> (16 * (e % 2) + 4 * (ch % 4)) & 15u) - 8), acc[c]);
      }
    }
  }
  l = wave_sum(l);
  z = wave_sum(z);
  if (lane == 0) sums[wave][0] = m, sums[wave][1] = l, sums[wave][2] = z;
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if (lane + 64 * c < hd) outs[wave][lane + 64 * c] = acc[c];
  __syncthreads();
  float top = -INFINITY;
  for (int w = 0; w < 4; ++w) top = fmaxf(top, sums[w][0]);
  const float base = top == -INFINITY ? 0.f : top;
  float total = 0.f, low = 0.f, weight[4];
  bool bad = false;  // (a maximum that is no number is lost in fmaxf; its sum is not)
  for (int w = 0; w < 4; ++w) {
    weight[w] = exp2f(sums[w][0] - base);
    total += sums[w][1] * weight[w];
    low += sums[w][2] * weight[w];
    bad |= !(sums[w][0] < INFINITY);
  }
  for (int c = threadIdx.x; c < hd; c += blockDim.x) {
    float o = low;
    for (int w = 0; w < 4; ++w) o += outs[w][c] * weight[w];
    o = bad ? NAN : total > 0.f ? o / total : total == 0.f ? 0.f : NAN;
    if (a.splits == 1)
      ((T*)a.out)[((size_t)t * a.heads + head) * hd + c] = from_f<T>(o);
    else
      a.part_o[((size_t)blockIdx.x * a.splits + split) * hd + c] = o;
  }
  if (a.splits > 1 && threadIdx.x == 0) a.part_l[(size_t)blockIdx.x * a.splits + split] = bad ? NAN : top + log2f(total);
}

// Joining the ranges of a column: out = sum_s o_s 2^(l_s - max l) / sum_s 2^(l_s - max l).  A workgroup a column: a wave, or, of few columns in many ranges, four that take eight ranges each in turn (2 rows of 64 heads in 32
// ranges each: 6.0 us, by a wave each 9.2); a range whose weight is no number makes it so.
// ``tile_tokens`` 0: columns are (token, head); otherwise (tile, token of the tile, head), and of a tile with fewer tokens nothing is written.
template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES * NS_WAVE) void attn_kv4_join_kernel(const Kv4AttnParams a, int tile_tokens) {
  __shared__ float sums[WAVES][WAVES > 1 ? KV4_MAX_HD : 1];
  const size_t col = blockIdx.x;
  const int lane = threadIdx.x % NS_WAVE, wave = WAVES > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NS_WAVE) : 0, head = col % a.heads;
  size_t row = col / a.heads;
  if (tile_tokens) {
    const int* info = a.tiles + row / tile_tokens * 8;
    const int token = info[1] + (int)(row % tile_tokens);
    if (token >= info[3]) return;
    row = info[2] + token;
  }
  const float* from = a.part_o + col * a.splits * a.hd;
  // a wave's first eight results are asked for before it is known which count
  float x[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int s = 0; s < 8; ++s) x[i][s] = lane + 64 * i < a.hd && 8 * wave + s < a.splits ? from[(size_t)(8 * wave + s) * a.hd + lane + 64 * i] : 0.f;
  const float ls = lane < a.splits ? a.part_l[col * a.splits + lane] : -INFINITY;
  if (__any(ls == INFINITY)) return;  // written whole (KV4_WHOLE)
  // (results are there up to the last that counts, those in front of a token's window of weight 0)
  const uint64_t counts = __ballot(ls != -INFINITY);
  const int used = counts ? 64 - __clzll(counts) : 0;
  const float top = wave_max(ls), base = top == -INFINITY ? 0.f : top;
  // (shares: no sum of them times the ranges' results is larger than those; no key has a weight: 0, as of one range)
  const float part = exp2f(ls - base), weight = used ? part / wave_sum(part) : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = lane + 64 * i;
    if (64 * i >= a.hd) break;
    float o = 0.f;
#pragma unroll
    for (int s = 0; s < 8; ++s) o += 8 * wave + s < used ? x[i][s] * __shfl(weight, 8 * wave + s, NS_WAVE) : 0.f;
    for (int s0 = 8 * (wave + WAVES); s0 < used; s0 += 8 * WAVES) {  // eight results' loads on their way at a time
      float more[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) more[s] = c < a.hd ? from[(size_t)min(s0 + s, used - 1) * a.hd + c] : 0.f;
#pragma unroll
      for (int s = 0; s < 8; ++s) o += s0 + s < used ? more[s] * __shfl(weight, (s0 + s) & 63, NS_WAVE) : 0.f;
    }
    if constexpr (WAVES > 1)
      sums[wave][c] = o;
    else if (c < a.hd)
      ((T*)a.out)[(row * a.heads + head) * a.hd + c] = from_f<T>(o);
  }
  if constexpr (WAVES == 1) return;
  __syncthreads();
  for (int c = threadIdx.x; c < a.hd; c += blockDim.x) {
    float o = sums[0][c];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) o += sums[v][c];
    ((T*)a.out)[(row * a.heads + head) * a.hd + c] = from_f<T>(o);
  }
}
template <typename T>
static void launch_join(const Kv4AttnParams& a, unsigned columns, int tile_tokens, hipStream_t stream) {
  // (many columns fill the card with a wave each: 22,500 of 11 ranges 18 us; as first measured, 21,000 of 9, 24, with four 47)
  if (a.splits <= 8 || columns > 4096)
    attn_kv4_join_kernel<T, 1><<<columns, NS_WAVE, 0, stream>>>(a, tile_tokens);
  else
    attn_kv4_join_kernel<T, 4><<<columns, 4 * NS_WAVE, 0, stream>>>(a, tile_tokens);
}

template <typename T>
static void launch_plain(const Kv4AttnParams& a, int tokens, hipStream_t stream) {
  const dim3 grid((unsigned)(tokens * a.heads), (unsigned)a.splits);
  switch ((a.hd + 63) / 64) {
    case 1: attn_kv4_plain_kernel<T, 1><<<grid, 256, 0, stream>>>(a); break;
    case 2: attn_kv4_plain_kernel<T, 2><<<grid, 256, 0, stream>>>(a); break;
    case 3: attn_kv4_plain_kernel<T, 3><<<grid, 256, 0, stream>>>(a); break;
    default: attn_kv4_plain_kernel<T, 4><<<grid, 256, 0, stream>>>(a);
  }
  if (a.splits > 1) launch_join<T>(a, (unsigned)(tokens * a.heads), 0, stream);
}

extern "C" int ns_attn_kv4_plain(void* out, void* part_o, void* part_l, const void* q, int q_stride, const void* pool, const int* token_req, const int* positions,
                                 const int* block_table, int table_stride, int tokens, int heads, int kv_heads, int hd, int page, int splits, int window, float scale,
                                 int dtype, hipStream_t stream) {
  if (tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || hd < 32 || hd > KV4_MAX_HD || hd % 32 || page < KV4_TOKENS || (page & (page - 1)) || window < 0)
    return NS_ERR_BAD_ARG;
  if (splits < 1 || splits > 64 || (splits > 1 && (!part_o || !part_l)) || (long long)tokens * heads > 0x7fffffff) return NS_ERR_BAD_ARG;
  if (tokens == 0) return NS_OK;
  const Kv4AttnParams a{out, (float*)part_o, (float*)part_l, q, (const uint8_t*)pool, nullptr, token_req, positions, block_table, q_stride, table_stride, 0, heads, kv_heads,
                        hd, page, splits, window, 0, scale * 1.4426950408889634f, 0};
  if (dtype == NS_DTYPE_F32)
    launch_plain<float>(a, tokens, stream);
  else if (dtype == NS_DTYPE_BF16)
    launch_plain<bf16_t>(a, tokens, stream);
  else
    return NS_ERR_UNSUPPORTED;
  return ns_launch_status();
}

#include "attn_kv4_mfma.h"

template <typename T, int HD, bool EXACT>
static int launch_tiles(const Kv4AttnParams& a, int rows, int form, hipStream_t stream) {
  const int group = a.heads / a.kv_heads;
  if (rows) {
    if (a.n_tiles > 65535) return NS_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)(a.kv_heads * ((group + 15) / 16)), (unsigned)a.n_tiles, (unsigned)a.splits);
    if (form == 8)
      attn_kv4_rows_kernel<T, HD, EXACT, 8><<<grid, 512, 0, stream>>>(a);
    else
      attn_kv4_rows_kernel<T, HD, EXACT, 4><<<grid, 256, 0, stream>>>(a);
  } else {
    const long long items = (long long)a.n_tiles * a.splits * a.heads * (KV4_TILE_TOKENS / form);
    if (items > 0x7fffffff - 4) return NS_ERR_UNSUPPORTED;
    const unsigned grid = (unsigned)((items + 3) / 4);
    if constexpr (!EXACT) {
      if (form == 32) attn_kv4_tiles_kernel<T, HD, 2, EXACT><<<grid, 256, 0, stream>>>(a);
    }
    if (form == 16) attn_kv4_tiles_kernel<T, HD, 1, EXACT><<<grid, 256, 0, stream>>>(a);
  }
  if (a.splits > 1) {
    const long long cols = (long long)a.n_tiles * (rows ? 1 : KV4_TILE_TOKENS) * a.heads;
    if (cols > 0x7fffffff) return NS_ERR_UNSUPPORTED;
    launch_join<T>(a, (unsigned)cols, rows ? 1 : KV4_TILE_TOKENS, stream);
  }
  return ns_launch_status();
}

// Attention of the tokens that ``tiles`` [n_tiles][8] names: request, first token of the tile among the request's tokens of this step, row of the request's first token, tokens of the
// request in this step, keys after it, one more, of single tokens the blocks of 32 keys of all of them, one more.  rows 1: a tile is one token, and a workgroup has ``form`` waves (4, 8); 0: up to 32 tokens, of which a
// wave takes ``form`` (16; with bfloat16 also 32).  part_o: float32 [n_tiles * tokens of a tile * heads * splits * hd] and part_l
// [n_tiles * tokens of a tile * heads * splits] with splits > 1.
extern "C" int ns_attn_kv4(void* out, void* part_o, void* part_l, const void* q, int q_stride, const void* pool, const int* tiles, const int* block_table, int table_stride,
                           int n_tiles, int heads, int kv_heads, int hd, int page, int rows, int form, int splits, int groups, int window, float scale, int dtype, hipStream_t stream) {
  if (n_tiles < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || page < KV4_TOKENS || (page & (page - 1)) || window < 0) return NS_ERR_BAD_ARG;
  if (splits < 1 || splits > 64 || (splits > 1 && (!part_o || !part_l)) || groups < 1) return NS_ERR_BAD_ARG;
  if (rows ? form != 4 && form != 8 : form != 16 && (form != 32 || dtype == NS_DTYPE_F32)) return NS_ERR_BAD_ARG;
  if (hd != 64 && hd != 128) return NS_ERR_UNSUPPORTED;
  if ((((uintptr_t)out | (uintptr_t)pool | (uintptr_t)part_o) & 15) != 0) return NS_ERR_UNSUPPORTED;
  if (n_tiles == 0) return NS_OK;
  const Kv4AttnParams a{out, (float*)part_o, (float*)part_l, q, (const uint8_t*)pool, tiles, nullptr, nullptr, block_table, q_stride, table_stride, n_tiles, heads, kv_heads,
                        hd, page, splits, window, groups, scale * 1.4426950408889634f,
                        ((uintptr_t)q & 15) == 0 && q_stride % (dtype == NS_DTYPE_F32 ? 4 : 8) == 0};
  if (dtype == NS_DTYPE_F32) return hd == 64 ? launch_tiles<float, 64, true>(a, rows, form, stream) : launch_tiles<float, 128, true>(a, rows, form, stream);
  if (dtype == NS_DTYPE_BF16) return hd == 64 ? launch_tiles<bf16_t, 64, false>(a, rows, form, stream) : launch_tiles<bf16_t, 128, false>(a, rows, form, stream);
  return NS_ERR_UNSUPPORTED;
}
