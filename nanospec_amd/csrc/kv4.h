// Pages of keys and values held in 4 bits: the layout, shared by the kernels that write, read and attend over them.
//
// The channels of a head's key (or value) of one token share a step and a lowest value, both bfloat16, rounded outwards so that the
// range holds every channel: a code u of 0 to 15 stands for step * u + low.  A group that holds an infinity or no number, or reaches
// further than 2^100, has step 0 and low = no number, so that whoever sees it gets no number and nobody else; a step below 2^-100 is 0.
//
// Eight consecutive tokens of a head (an octet; octets begin at multiples of 8 in a page) lie together in one record, everything that
// attention reads of them in one run of 8 hd + 64 bytes:
//   keys     at j * hd / 2, token j of the octet: dword t * (hd / 32) + g holds channels 32 g + 8 t + {0 .. 7}: what lane (key, t) of
//            a 16x16x32 matrix instruction wants of its key for all hd channels is one load; channel c of the 8 at bit 4 (c / 2) + 16 (c % 2),
//            so that a mask leaves two neighbours in the halves of a dword
//   values   at 4 hd + 16 * (channel / 4): 8 x 16 bits, token j's channels 4 m + {0 .. 3} at bits 4 i: what lane (m, t) wants of eight
//            keys for four channels is one load, two keys of a channel side by side in the halves of a dword
//   marks    at 8 hd: 8 dwords of the keys, 8 of the values: low in the low half, step in the high one (as a whole number a mark orders
//            by its step)
// A pool is [pages][kv heads][page / 8] such records.
#pragma once
#include "common.h"

#define KV4_TOKENS 8       // tokens of a record
#define KV4_MAX_HD 256
#define KV4_TINY 0x1p-100f
#define KV4_HUGE 0x1p100f

__host__ __device__ __forceinline__ int kv4_record(int hd) { return KV4_TOKENS * hd + 2 * KV4_TOKENS * 4; }
__host__ __device__ __forceinline__ int kv4_values_at(int hd) { return KV4_TOKENS / 2 * hd; }
__host__ __device__ __forceinline__ int kv4_marks_at(int hd) { return KV4_TOKENS * hd; }

__device__ __forceinline__ float kv4_low(uint32_t mark) { return __uint_as_float(mark << 16); }
__device__ __forceinline__ float kv4_step(uint32_t mark) { return __uint_as_float(mark & 0xffff0000u); }

// a float's neighbour among the bfloat16 values, downwards or upwards (itself if it is one)
__device__ __forceinline__ float bf16_floor(float x) {
  const uint32_t b = __float_as_uint(x), cut = b & 0xffff0000u;
  return __uint_as_float((b >> 31) && (b & 0xffffu) ? cut + 0x10000u : cut);
}
__device__ __forceinline__ float bf16_ceil(float x) { return -bf16_floor(-x); }

// the record of octet ``oct`` of head ``h`` of page ``page``, in records from the pool's start
__device__ __forceinline__ size_t kv4_at(int page, int kv_heads, int h, int octets, int oct) {
  return ((size_t)page * kv_heads + h) * octets + oct;
}
