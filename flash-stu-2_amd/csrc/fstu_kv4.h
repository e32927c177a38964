// A ring cache of keys and values in 4 bits: where everything lies in its buffer.
//
// Values are e2m1 codes (sign, two bits of exponent, one of mantissa: 0 0.5 1 1.5 2 3 4 6), 32 values of a head's row share a power of
// two as their scale, held as its biased exponent (a byte; 255: the block stands for NaN).  A value is code * 2^(byte - 127), which is
// exact in bf16.  Slots are padded to a multiple of 32; head = sequence * kv_heads + key head.
//   key codes     (head, slot, hd/2)                         a row as it is
//   value codes   (head, slot/8, plane, 16, ...)             a lane of the second product takes hd/16 dims (hd/32 bytes) of eight slots, slot by slot; what
//                                                            is more than 16 bytes of that is cut into planes of 16, so that 16 lanes read 256 beside each other
//   key scales    (head, slot/8, hd/32, slot%8)              eight slots' scales of a block beside each other
//   value scales  the same
#pragma once
#include <stdint.h>

#define KV4_TILE 32       // slots that one step of the attention takes

struct Kv4 {
  unsigned char *kc, *vc, *ks, *vs;
  int slots;              // capacity, padded
};

static inline __host__ __device__ int kv4_slots(int cap) { return (cap + KV4_TILE - 1) / KV4_TILE * KV4_TILE; }

static inline __host__ __device__ Kv4 kv4_at(void* cache, int64_t heads, int hd, int cap) {
  Kv4 c;
  c.slots = kv4_slots(cap);
  const int64_t codes = heads * c.slots * (hd / 2), scales = heads * c.slots * (hd / 32);
  c.kc = (unsigned char*)cache;
  c.vc = c.kc + codes;
  c.ks = c.vc + codes;
  c.vs = c.ks + scales;
  return c;
}
