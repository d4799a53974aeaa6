// Cross attention on gfx950: what the forward and the backward share.
//
//   O = softmax(scale Q K^T over the sample's valid keys) V
//
// q rows are [batch, heads, sq], k / v rows [batch, kv_heads, skv], any strides
// with the channels next to each other and 16-byte aligned rows.  The heads of
// a group (heads / kv_heads) share a key head.  A key is valid if it lies below
// its sample's kv_lens and its key_mask byte is not zero.
//
// Tiles of K and V (or Q and dO) are copied to LDS by direct loads that write
// zeros for the rows of keys that are not valid and for the channels past the
// head dim, so that nothing behind a mask (infinities, NaN, memory past the last
// row) takes part in a product.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "vsa_device.h"
#include "vsa_launch.h"

namespace vsa {

// 32x32 products over 16 elements of the reduced axis, per element type.  fp32
// takes v_mfma_f32_32x32x2_f32: element e of the two operands is the pair of
// reduced elements e and 8 + e of lane halves 0 and 1, the same pairing on both
// sides, so any order of the 16 does.
template <typename T>
struct Mma {
  typedef typename Elem<T>::vec8 V8;
  static __device__ __forceinline__ f32x16 mul(V8 a, V8 b, f32x16 c) {
    return Elem<T>::mfma32(a, b, c);
  }
};
typedef float f32x8 __attribute__((ext_vector_type(8)));
template <>
struct Mma<float> {
  typedef f32x8 V8;
  static __device__ __forceinline__ f32x16 mul(V8 a, V8 b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

template <typename T>
__device__ __forceinline__ typename Mma<T>::V8 pack_op(const float* v) {
  if constexpr (sizeof(T) == 4) {
    f32x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = v[e];
    return r;
  } else {
    return pack8<T>(v);
  }
}

template <typename T>
__device__ __forceinline__ typename Mma<T>::V8 zero8() {
  typename Mma<T>::V8 z = {};
  return z;
}

// Eight values as an operand, and what rounding them to T left over as another.  (The
// pairs are opaque: unpacked by the compiler each value is rounded a second time.)
template <typename T>
__device__ __forceinline__ void pack_both(const float* v, typename Mma<T>::V8& hi,
                                          typename Mma<T>::V8& lo) {
  if constexpr (sizeof(T) == 4) {
    hi = pack_op<T>(v);
    lo = zero8<T>();
  } else {
    u32x4 w = __builtin_bit_cast(u32x4, pack_op<T>(v));
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = opaque(w[i]);
    hi = as_vec8<T>(w);
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) rest[e] = fmaf((float)hi[e], -1.f, v[e]);
    lo = pack_op<T>(rest);
  }
}

// 8 consecutive elements at a 16-byte aligned address
template <typename T>
__device__ __forceinline__ typename Mma<T>::V8 ld8(const T* p) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  } else {
    return as_vec8<T>(*reinterpret_cast<const u32x4*>(p));
  }
}

// Wide rows leave no registers to read many operands ahead: without a fence after
// each step of a product the compiler moves the reads of all of them to the
// front and spills (head dim 256, and 128 in fp32).
template <typename T, int D>
constexpr bool kWide = D * sizeof(T) > 256;
template <typename T, int D>
__device__ __forceinline__ void step_fence() {
  if constexpr (kWide<T, D>) __builtin_amdgcn_sched_barrier(0);
}

// Whether the channels from d on take part in a product.  fp32 products of 16
// channels take 512 cycles, a scalar branch pays for leaving out those past the
// head dim (80 of 128: forward 66 -> 55 us, dQ 96 -> 74); at 16 bits, 32 cycles, it would not.
template <typename T>
__device__ __forceinline__ bool in_dim(int d, int dim) {
  return sizeof(T) == 2 || d < dim;
}

// LDS tile of rows of D elements, 16-byte chunks swizzled by the row: 16-bit
// types as in vsa_device.h, fp32 rows (at least 256 bytes: one pass over the 64
// banks) by the row's low four bits.
template <typename T, int D>
struct Tile {
  static constexpr int CH = D * (int)sizeof(T) / 16;  // chunks of a row
  static constexpr int ROW = D * (int)sizeof(T);      // bytes of a row
  static __device__ __forceinline__ int off(int r, int c) {
    if constexpr (sizeof(T) == 2) return swz<D>(r, c) * 2;
    else return r * ROW + ((c >> 4) << 8) + (((c & 15) ^ (r & 15)) << 4);
  }
  // row and chunk that live at chunk position P
  static __device__ __forceinline__ int unoff(int P, int& c) {
    if constexpr (sizeof(T) == 2) {
      return unswz_row_chunk<D>(P, c);
    } else {
      const int r = P / CH;
      c = (P % CH) ^ (r & 15);   // the upper bits of a chunk stay
      return r;
    }
  }
};

// Row operand: lane (r, h) takes elements 16 ks + 8 h .. + 7 of row `row`.
template <typename T, int D>
__device__ __forceinline__ typename Mma<T>::V8 row_op(const char* X, int row, int ks, int h) {
  typedef Tile<T, D> L;
  if constexpr (sizeof(T) == 2) {
    return as_vec8<T>(*reinterpret_cast<const u32x4*>(X + L::off(row, 2 * ks + h)));
  } else {
    const f32x4 a = *reinterpret_cast<const f32x4*>(X + L::off(row, 4 * ks + 2 * h));
    const f32x4 b = *reinterpret_cast<const f32x4*>(X + L::off(row, 4 * ks + 2 * h + 1));
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
}

// Column operand: lane (r, h) takes channel d0 + r of rows s + 4h .. + 3 and
// s + 8 + 4h .. + 3, the order in which a 32x32 result holds its rows.
template <typename T, int D>
__device__ __forceinline__ typename Mma<T>::V8 col_op(const char* X, int d0, int s) {
  if constexpr (sizeof(T) == 2) {
    return tr_a8<T, D>(reinterpret_cast<const T*>(X), d0, s, s + 8);
  } else {
    typedef Tile<T, D> L;
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    f32x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int row = s + (e >> 2) * 8 + 4 * h + (e & 3);
      // chunk d0 / 4 + r / 4: d0 is a multiple of 32, so its bits above the low
      // three of r / 4 can be split off
      const int lo = ((d0 >> 2) & 8) | (r >> 2);
      v[e] = *reinterpret_cast<const float*>(X + row * L::ROW + ((d0 >> 6) << 8) +
                                             ((lo ^ (row & 15)) << 4) + (r & 3) * 4);
    }
    return v;
  }
}

// What the statistics of query rows past the last one read: P = 2^(s - inf) = 0.
__device__ __attribute__((aligned(16))) static const float kPastStats[2] = {INFINITY, 0.f};

// Direct copies of 16 bytes a lane to LDS through a buffer descriptor: a lane
// whose offset lies past the descriptor's bytes writes zeros, so rows past the
// last one, keys behind a mask and channels past the head dim need no branch
// and no address of their own (dma16 in vsa_device.h explains the asm's form).
typedef u32x4 Srd;
__device__ __forceinline__ Srd srd_of(const void* base, uint32_t bytes) {
  // (uniform values, in scalar registers whatever the compiler knows of them)
  const uint64_t p = (uint64_t)(uintptr_t)base;
  return Srd{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)p),
             (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(p >> 32)) & 0xffffu,
             (uint32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}
__device__ __forceinline__ void dma16_b(uint32_t voff, Srd srd, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff),
               "s"(srd), "s"(__builtin_amdgcn_readfirstlane(lds))
               : "memory");
}
constexpr uint32_t kPastEnd = 0x80000000u;  // descriptors hold less than 2^31 bytes

// Copies ROWS rows of D elements into a tile, as threads 0 .. NT - 1 (whole waves
// of a workgroup).  A thread keeps the
// byte offsets of up to eight of its 16-byte pieces; the swizzle repeats every
// 16 rows, so the pieces of later rows take the same offsets from a descriptor
// that starts 16 rows on.
template <typename T, int D, int ROWS, int NT>
struct TileCopy {
  typedef Tile<T, D> L;
  static constexpr int N = ROWS * L::CH / NT;                   // pieces of a thread
  static constexpr int K = N <= 8 ? N : 16 * L::CH / NT;        // of them kept
  static constexpr int G = N / K;                               // descriptors
  static constexpr bool KEEP = D * sizeof(T) <= 512;            // else worked out again
  static_assert(ROWS * L::CH % NT == 0 && ROWS % 32 == 0 && N % K == 0 && K <= 8, "");
  uint32_t voff[KEEP ? K : 1];   // byte offset of the piece from the descriptor's first row
  uint32_t stride;               // bytes between rows
  int dim;                       // bytes of a row
  uint32_t wave;                 // of this thread's wave, bytes into each piece
  int tid;
  struct Src {
    Srd s[G];
  };

  __device__ __forceinline__ void init(int64_t row_stride, int channels, int thread) {
    stride = (uint32_t)(row_stride * (int)sizeof(T));
    dim = channels * (int)sizeof(T);
    tid = thread;
    wave = (uint32_t)__builtin_amdgcn_readfirstlane(thread >> 6) * 1024u;
    if constexpr (KEEP) {
#pragma unroll
      for (int i = 0; i < K; ++i) voff[i] = opaque(offset(i, tid));
    }
  }
  __device__ __forceinline__ uint32_t offset(int i, int t) const {
    int c;
    const int row = L::unoff(i * NT + t, c);
    return c * 16 < dim ? (uint32_t)row * stride + (uint32_t)c * 16u : kPastEnd;
  }
  __device__ __forceinline__ uint32_t at(int i) const {
    return KEEP ? voff[KEEP ? i % K : 0] : offset(i % K, opaque(tid));
  }
  // the rows from src on, `left` (>= 1) of which exist
  __device__ __forceinline__ Src rows(const T* src, int left) const {
    Src r;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int n = min(left, ROWS) - 16 * g;
      r.s[g] = srd_of(reinterpret_cast<const char*>(src) + (uint64_t)(16 * g) * stride,
                      n > 0 ? (uint32_t)(n - 1) * stride + (uint32_t)dim : 0u);
    }
    return r;
  }
  __device__ __forceinline__ void piece(int i, uint32_t lds, const Src& src) const {
    dma16_b(at(i), src.s[i / K], lds + wave + (uint32_t)i * (NT / 64) * 1024u);
  }
  __device__ __forceinline__ void copy(uint32_t lds, const Src& src) const {
#pragma unroll
    for (int i = 0; i < N; ++i) piece(i, lds, src);
  }
  // Rows whose bit of `valid` is clear become zeros.
  __device__ __forceinline__ void copy_valid(uint32_t lds, const Src& src,
                                             const uint32_t (&valid)[ROWS / 32]) const {
    const int t = opaque(tid);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int c;
      const int row = L::unoff(i * NT + t, c);
      uint32_t w = valid[0];
#pragma unroll
      for (int x = 1; x < ROWS / 32; ++x) w = row >= 32 * x ? valid[x] : w;
      dma16_b((w >> (row & 31)) & 1u ? at(i) : kPastEnd, src.s[i / K],
              lds + wave + (uint32_t)i * (NT / 64) * 1024u);
    }
  }
};

// Operand reads of tiles in LDS.  For 16-bit types the per-lane byte offsets
// are set once (the swizzle repeats every 16 rows, so other rows and stages
// differ by constants); left to the compiler the swizzle was worked out again
// for every chunk.  `at` is a tile's byte offset from the workgroup's LDS.
template <typename T, int D>
struct Operands {
  typedef typename Mma<T>::V8 V8;
  const char* lds;
  int r, h;
  __device__ __forceinline__ void init(const char* base, int r_, int h_) {
    lds = base, r = r_, h = h_;
  }
  __device__ __forceinline__ V8 row(int at, int tile32, int ks) const {
    return row_op<T, D>(lds + at, 32 * tile32 + r, ks, h);
  }
  __device__ __forceinline__ V8 col(int at, int d0, int mt, int kk) const {
    return col_op<T, D>(lds + at, d0 + 32 * mt, 16 * kk);
  }
};
template <typename T, int D>
struct Operands16 {
  typedef typename Mma<T>::V8 V8;
  const char* lds;
  uint32_t row_off[D / 16], col_off[D / 32][2];
  __device__ __forceinline__ void init(const char* base, int r, int h) {
    lds = base;
    const int lane = threadIdx.x & 63, grp = lane >> 4, j = lane & 15, q = grp & 1, hh = grp >> 1;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
      row_off[ks] = opaque((uint32_t)(swz<D>(r, 2 * ks + h) * 2));
#pragma unroll
    for (int mt = 0; mt < D / 32; ++mt)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        col_off[mt][x] = opaque(
            (uint32_t)(swz_elem<D>(8 * x + 4 * hh + (j >> 2), mt * 32 + 16 * q + 4 * (j & 3)) * 2));
  }
  __device__ __forceinline__ V8 row(int at, int tile32, int ks) const {
    return as_vec8<T>(*reinterpret_cast<const u32x4*>(lds + row_off[ks] + at + tile32 * 64 * D));
  }
  // channels 32 mt .. of a tile; a constant first channel of 0 or 128
  __device__ __forceinline__ V8 col(int at, int d0, int mt, int kk) const {
    const char* p = lds + at + kk * 32 * D + (d0 >> 7) * 256;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + col_off[mt][0]));
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + col_off[mt][1]));
    const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
    return as_vec8<T>(u32x4{a[0], a[1], b[0], b[1]});
  }
};
template <int D>
struct Operands<__bf16, D> : Operands16<__bf16, D> {};
template <int D>
struct Operands<_Float16, D> : Operands16<_Float16, D> {};

struct Rows {          // a [batch, head, token] view
  const void* p;
  int64_t b, h, s;     // strides in elements
};

struct CrossArgs {
  Rows q, k, v, o, dout;
  void *out, *dq, *dk, *dv;
  uint8_t* lo;                 // what rounding the output left over, [batch, heads, sq, dim], or null
  int64_t out_s[3], dq_s[3], dk_s[3], dv_s[3];
  float *lse, *delta;          // [batch, heads, sq]
  float *part_a, *part_b;      // fp32 partial results of the splits
  const int32_t* lens;
  const uint32_t* words;       // [batch, nwords] of 32 keys, or null
  int nwords;
  int sq, skv, heads, kv_heads, group, dim;
  int batch, splits, tiles;    // tiles of a split
  int per_head;                // tiles of a (batch, key head)
  int spread;                  // order of the tiles: see tile_of
  float c2, scale;
  uint32_t qsign;
};

// The tile of a workgroup.  An XCD takes a contiguous range (xcd_tile), so that
// the K and V of a head stay in its L2.  Where samples may differ in their keys
// and one head's K and V are small, tiles go round the XCDs instead: by ranges
// the XCDs of the samples with few keys end early (2 samples of 10 heads, 3001
// queries in fp32 on 333 keys and on none: forward 115 -> 66 us, dQ 165 -> 96).
// Pairs of alternating samples within a range were no better than the ranges: an
// XCD hands its workgroups round its shader engines, and half of them got the
// empty ones.
__device__ __forceinline__ int tile_of(const CrossArgs& a) {
  return a.spread ? (int)blockIdx.x : xcd_tile(blockIdx.x, a.tiles * a.splits);
}

typedef const __attribute__((address_space(4))) uint32_t* const_words;

// Whether a sample's first n keys hold a single valid one.  Its weight is 1 whatever
// the scores and dS is 0, where P (dP - delta) would leave the rounding of two sums
// over the channels: gradients of q and k that are nothing but noise.
__device__ __forceinline__ bool single_key(const CrossArgs& a, int b, int n) {
  if (!a.words) return n == 1;
  const const_words words = (const_words)(uintptr_t)(a.words + (int64_t)b * a.nwords);
  int count = 0;
  for (int x = 0; x < (n + 31) / 32 && count < 2; ++x) count += __builtin_popcount(words[x]);
  return count == 1;
}

// The chunks of KC keys of one sample that hold a valid key, in order.  The
// words are read through the constant address space: scalar loads, which the
// direct copies' vmcnt waits never include.
template <int KC>
struct KeyWalk {
  const_words words;
  int n, last;               // valid prefix; chunk past the last one
  int j;
  uint32_t w[KC / 32];

  __device__ __forceinline__ void init(const CrossArgs& a, int b, int first, int chunks) {
    n = a.skv;
    if (a.lens) n = min(max(a.lens[b], 0), a.skv);
    n = __builtin_amdgcn_readfirstlane(n);
    words = a.words ? (const_words)(uintptr_t)(a.words + (int64_t)b * a.nwords) : nullptr;
    j = first;
    last = min(first + chunks, (n + KC - 1) / KC);
  }
  // The next chunk with a valid key among j, j + STEP, ..; false if there is none.
  template <int STEP = 1>
  __device__ __forceinline__ bool find() {
    for (; j < last; j += STEP) {
      uint32_t any = 0;
#pragma unroll
      for (int x = 0; x < KC / 32; ++x) {
        const int left = n - j * KC - 32 * x;
        w[x] = left >= 32 ? ~0u : left > 0 ? (1u << left) - 1u : 0u;
        if (words) w[x] &= words[j * (KC / 32) + x];
        any |= w[x];
      }
      if (any) return true;
    }
    return false;
  }
  // a key below the valid prefix is masked: zeros must come from the copy
  __device__ __forceinline__ bool holes() const { return words && !whole(); }
  __device__ __forceinline__ bool whole() const {
    uint32_t all = ~0u;
#pragma unroll
    for (int x = 0; x < KC / 32; ++x) all &= w[x];
    return all == ~0u;
  }
};

// Whether the key that accumulator element i holds is valid: key 8 (i / 4) + i % 4
// in the lanes of half 0, four on in half 1.  The two bits of the (uniform) word
// become a lane mask on the scalar unit.
__device__ __forceinline__ bool acc_valid(uint32_t w, int i) {
  const int k = 8 * (i >> 2) + (i & 3);
  const uint32_t lo = (uint32_t)((int32_t)(w << (31 - k)) >> 31);
  const uint32_t hi = (uint32_t)((int32_t)(w << (27 - k)) >> 31);
  return __builtin_amdgcn_inverse_ballot_w64((uint64_t)hi << 32 | lo);
}

// Eight consecutive channels of a row, as T.
template <typename T>
__device__ __forceinline__ void st8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    T o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = Elem<T>::from_f(v[e]);
    *reinterpret_cast<u32x4*>(p) = *reinterpret_cast<const u32x4*>(o);
  }
}

// What rounding an output value o to 16 bits left over, as a byte: in units of
// 1/254 of o's unit in the last place, 128 for nothing.  kLeast keeps the unit of
// fp16's subnormals, and bf16's inverse finite.
template <typename T>
struct RestOf {
  static constexpr bool kHalf = std::is_same<T, _Float16>::value;
  static constexpr uint32_t kLeast = (127u - (kHalf ? 14u : 100u)) << 23;
  static constexpr float kUnits = 127.f * (float)(1 << (kHalf ? 11 : 8));
  static __device__ __forceinline__ uint32_t power(float o) {   // 2^exponent of o, as bits
    return max(__float_as_uint(o) & 0x7f800000u, kLeast);
  }
};

// Eight channels of the output, and what rounding them to T left over: delta is
// sum dO O, and where the weights are spread over many keys dS = P (dP - delta)
// is so much smaller than dP that the rounding of O shows in dQ (bf16, 4000
// keys: 6.6e-3 of its norm, 1e-5 with the rest; the roundings that stay, of dS
// and of dQ, make 2.4e-3).  A byte holds it to 2^-8 of itself, as 16 bits would.
template <typename T>
__device__ __forceinline__ void st8_out(T* out, uint8_t* lo, const float (&v)[8]) {
  st8<T>(out, v);
  if constexpr (sizeof(T) == 2) {
    if (lo) {
      typedef RestOf<T> R;
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float o = round_t<T>(v[e]);
        const float per = __uint_as_float(0x7f000000u - R::power(o)) * R::kUnits;
        w[e >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(rintf(fmaf(v[e] - o, per, 128.f)), e & 3, w[e >> 2]);
      }
      *reinterpret_cast<u32x2*>(lo) = u32x2{w[0], w[1]};
    }
  }
}

// The sum of eight channels' g o with the rests of o.
template <typename T>
__device__ __forceinline__ float dot_rest(typename Mma<T>::V8 g, typename Mma<T>::V8 o, u32x2 rest,
                                          float sum) {
  typedef RestOf<T> R;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float n = (float)((rest[e >> 2] >> (8 * (e & 3))) & 255u), x = (float)o[e];
    const float units = fmaf(n, 1.f / R::kUnits, -128.f / R::kUnits);
    sum = fmaf((float)g[e], fmaf(units, __uint_as_float(R::power(x)), x), sum);
  }
  return sum;
}

// Splits of a walk over the keys.  With `fit` workgroups that do not slow each other
// (one a CU, of four waves), s splits take ceil(tiles s / fit) rounds of their
// chunks, and their parts are written, read again and joined: 4.5 us and 0.4 us a
// MB.  A chunk takes `us`; MB is one split's part.  Forward and join of 16-bit 128
// channels, us, for the splits that fill the chip's LDS / by this rule: 12 heads,
// 2000 queries on 512 keys 39.6 (4) / 20.7 (1), 5000 queries 54.8 (2) / 29.6 (1);
// 8 heads, 256 queries on 10000 keys 44.4 (60) / 32.3 (16).
inline int64_t split_keys(int64_t tiles, int64_t fit, int64_t chunks, double us, double mb) {
  int64_t best = 1;
  double least = 1e300;
  auto look = [&](int64_t s) {
    s = std::max<int64_t>(1, std::min(s, chunks));
    const int64_t per = (chunks + s - 1) / s;
    s = (chunks + per - 1) / per;
    const double rounds = (double)((tiles * s + fit - 1) / fit);
    const double cost = rounds * ((double)per * us + 1.5) + (s > 1 ? 4.5 + 0.4 * mb * (double)s : 0);
    if (cost < least) least = cost, best = s;
  };
  for (int64_t s = 1; s <= 8; ++s) look(s);
  for (int64_t k = 1; k <= 3; ++k) look(k * fit / tiles);       // k whole rounds
  look((int64_t)std::sqrt((double)chunks * us / (0.4 * mb)));   // where both sides are equal
  return best;
}

}  // namespace vsa
