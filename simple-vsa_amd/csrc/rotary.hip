// Rotary positions on gfx950: tables of a latent grid, and the rotation of q and k.
//
// A pair of channels (x1, x2) at angle a becomes (x1 cos a - x2 sin a,
// x2 cos a + x1 sin a); the gradient is the same rotation by -a.  Pairs are
// channels (2i, 2i + 1) or (i, i + R/2) of the first R channels of a head.
//
// Both are bound by memory.  The rotation reads and writes q and k once (the
// table adds 4 R bytes a token and block of heads, from L2): 40 heads x 41k tokens
// x 128 channels in 0.28 ms, 6.0 TB/s, where the best copy of this card reaches
// 6.25.  The table is written once: 92160 positions x 64 pairs in 13 us, 3.6 TB/s
// (runs of 8 / 16 / 32 positions: 17.9 / 14.1 / 13.0 us, and 9.6 / 8.3 / 9.5 for
// 32760 x 64).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/vsa_capi.h"
#include "vsa_device.h"
#include "vsa_launch.h"

namespace vsa {

constexpr int kMaxPairs = 128;  // head dims up to 256

// ---------------------------------------------------------------------------
// Table
// ---------------------------------------------------------------------------

// Frequencies in 64 bits, made on the host and passed by value: no copy to the
// device, so a table can be made inside a graph capture.
struct TableArgs {
  double freq[kMaxPairs];
  double start[3];
  double size[3];      // the factor of an axis' cosines and sines
  int32_t n[3];        // positions of each axis
  int32_t pairs[3];
};

// One thread walks kTableRun consecutive tokens for one pair of channels.  The
// angle of a far position needs 64 bits (1e6 rad in 32 bits is off by 0.03),
// and a 64-bit sine costs about a hundred operations, so a thread takes two of
// them (its first angle and the step) and turns (cos, sin) by the step from one
// position to the next: four multiply-adds a token, each turn off by 2^-52 at
// most, a run of 16 by 1e-14 of the circle, far below the fp32 result's 2^-24.
constexpr int kTableRun = 16;

__global__ __launch_bounds__(256) void rotary_table_kernel(TableArgs a, int pairs, int64_t tokens,
                                                           float* __restrict__ co,
                                                           float* __restrict__ si) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int i = (int)(id % pairs);
  const int64_t t0 = id / pairs * kTableRun;
  if (t0 >= tokens) return;
  const int axis = i < a.pairs[0] ? 0 : i < a.pairs[0] + a.pairs[1] ? 1 : 2;
  // tokens between two positions of this axis, and how many positions it has
  const int64_t inner = axis == 0 ? (int64_t)a.n[1] * a.n[2] : axis == 1 ? a.n[2] : 1;
  const int n = a.n[axis];
  const double f = a.freq[i], start = a.start[axis], size = a.size[axis];
  int64_t in = t0 % inner;              // tokens since the last step
  int pos = (int)(t0 / inner % n);
  double c, s, c1, s1;
  sincos((start + pos) * f, &s, &c);
  sincos(f, &s1, &c1);
  const int64_t t1 = t0 + kTableRun < tokens ? t0 + kTableRun : tokens;
  for (int64_t t = t0; t < t1; ++t) {
    co[t * pairs + i] = (float)(c * size);
    si[t * pairs + i] = (float)(s * size);
    if (++in < inner) continue;
    in = 0;
    if (++pos < n) {
      const double c2 = c * c1 - s * s1;
      s = fma(s, c1, c * s1);
      c = c2;
    } else {
      pos = 0;
      sincos(start * f, &s, &c);
    }
  }
}

// ---------------------------------------------------------------------------
// Rotation
// ---------------------------------------------------------------------------

struct RotaryArgs {
  const void* x[2];     // q, k
  void* y[2];
  int64_t xs[2][3];     // strides of batch, head, token, in elements
  int64_t ys[2][3];
  const float *co, *si;
  const void* positions;
  int64_t pos_batch;    // elements between two samples' positions
  int64_t rows;         // of the table
  int64_t tokens;
  int32_t pos64, heads_q, heads, dim, pairs, units, turns, per_block, head_blocks, heads_fastest;
  float sign;
};

template <typename T, int V>
struct alignas(V * sizeof(T)) Piece {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ Piece<T, V> ld_piece(const T* p) {
  if constexpr (V * sizeof(T) == 16)
    return __builtin_bit_cast(Piece<T, V>, ld_stream(reinterpret_cast<const u32x4*>(p)));
  else
    return *reinterpret_cast<const Piece<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void st_piece(T* p, const Piece<T, V>& v) {
  if constexpr (V * sizeof(T) == 16)
    st_stream(reinterpret_cast<u32x4*>(p), __builtin_bit_cast(u32x4, v));
  else
    *reinterpret_cast<Piece<T, V>*>(p) = v;
}

// A thread owns a unit of one token's channels, the same in up to per_block heads
// of q and k, which it walks with its cosines and sines in registers.  A unit is
//  * kInter: a piece of V channels, V / 2 pairs;
//  * kSwap: a piece of V channels of which each is one of a pair; the other one's
//    piece comes from the lane that has it (the units of a row divide a wave);
//  * kTwo: V pairs, as a piece of either half (rows of other lengths; two loads of
//    half a row each: 24 heads x 41k tokens of 64 channels 112 us, kSwap 85);
//  * behind the turned channels, a piece that is copied.
// LOOSE: no alignment but the element's (kInter with an odd start or end).
enum RotaryMode { kTwo, kInter, kSwap };

template <typename T, int V, int MODE, bool LOOSE>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  constexpr int P = MODE == kInter ? V / 2 : V;   // cosines of a unit
  const int per = 256 / a.units;                  // tokens of a workgroup
  const int unit = threadIdx.x % a.units;
  if ((int)threadIdx.x >= per * a.units) return;
  // Head-major memory: the blocks of heads follow each other slowest, so that the
  // workgroups at work read and write neighbouring rows of a few heads; token-major:
  // fastest, so that they cover whole tokens (40 heads x 41k tokens, all heads in
  // a workgroup / blocks of four or eight in that order: 309 -> 289 and 322 -> 291
  // us, interleaved 321 -> 285 and 321 -> 273).
  const int64_t blocks = (a.tokens + per - 1) / per;
  int64_t g = blockIdx.x;
  int hb;
  if (a.heads_fastest) {
    hb = (int)(g % a.head_blocks);
    g /= a.head_blocks;
  }
  const int64_t t = g % blocks * per + threadIdx.x / a.units;
  g /= blocks;
  if (!a.heads_fastest) {
    hb = (int)(g % a.head_blocks);
    g /= a.head_blocks;
  }
  const int64_t b = g;
  if (t >= a.tokens) return;
  const bool turn = unit < a.turns;
  const int o1 = turn ? unit * V : 2 * a.pairs + (unit - a.turns) * V;
  const int o2 = a.pairs + o1;                    // kTwo: the second piece
  const int half = a.pairs / V;                   // kSwap: units of half a row
  const bool second = MODE == kSwap && unit >= half;

  float c[P], s[P];
#pragma unroll
  for (int e = 0; e < P; ++e) c[e] = 1.f, s[e] = 0.f;
  if (turn) {
    int64_t p = t;
    if (a.positions) {
      const int64_t at = b * a.pos_batch + t;
      p = a.pos64 ? ((const int64_t*)a.positions)[at] : ((const int32_t*)a.positions)[at];
    }
    if (p >= a.rows) {
#pragma unroll
      for (int e = 0; e < P; ++e) c[e] = s[e] = NAN;
    } else if (p >= 0) {
      const int64_t at = p * a.pairs + (second ? unit - half : unit) * P;
      const float sign = second ? -a.sign : a.sign;
#pragma unroll
      for (int e = 0; e < P; ++e) c[e] = a.co[at + e], s[e] = a.si[at + e] * sign;
    }
  }
  auto load = [&](const T* x) {
    if constexpr (!LOOSE) return ld_piece<T, V>(x);
    Piece<T, V> r;
    const int64_t left = a.dim - o1;
#pragma unroll
    for (int e = 0; e < V; ++e) r.e[e] = x[e < left ? e : 0];
    return r;
  };
  auto store = [&](T* y, const Piece<T, V>& v) {
    if constexpr (!LOOSE) return st_piece<T, V>(y, v);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < a.dim - o1) y[e] = v.e[e];
  };
  const int h0 = hb * a.per_block, h1 = min(h0 + a.per_block, a.heads);
  constexpr int UR = 4;
  for (int h = h0; h < h1; h += UR) {
    Piece<T, V> x1[UR], x2[UR];
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      const int hh = min(h + u, h1 - 1);
      const int w = hh >= a.heads_q;
      const T* x = (const T*)a.x[w] + b * a.xs[w][0] + (hh - w * a.heads_q) * a.xs[w][1] +
                   t * a.xs[w][2];
      x1[u] = load(x + o1);
      if (MODE == kTwo && turn) x2[u] = load(x + o2);
    }
    if constexpr (MODE == kSwap) {
      typedef uint32_t Words __attribute__((ext_vector_type(V * sizeof(T) / 4)));
      const int other = (int)(threadIdx.x & 63) + (turn ? second ? -half : half : 0);
#pragma unroll
      for (int u = 0; u < UR; ++u) {
        Words w = __builtin_bit_cast(Words, x1[u]);
#pragma unroll
        for (int i = 0; i < (int)(V * sizeof(T) / 4); ++i) w[i] = __shfl(w[i], other, 64);
        x2[u] = __builtin_bit_cast(Piece<T, V>, w);
      }
    }
#pragma unroll
    for (int u = 0; u < UR; ++u) {
      if (h + u >= h1) break;
      const int w = h + u >= a.heads_q;
      T* y = (T*)a.y[w] + b * a.ys[w][0] + (h + u - w * a.heads_q) * a.ys[w][1] + t * a.ys[w][2];
      if (turn) {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          T& lo = MODE == kInter ? x1[u].e[2 * e] : x1[u].e[e];
          T& hi = MODE == kInter ? x1[u].e[2 * e + 1] : x2[u].e[e];
          const float p = Elem<T>::to_f(lo), q = Elem<T>::to_f(hi);
          // (kSwap: the second of a pair has the sine's sign turned)
          lo = Elem<T>::from_f(p * c[e] - q * s[e]);
          if (MODE != kSwap) hi = Elem<T>::from_f(q * c[e] + p * s[e]);
        }
        if (MODE == kTwo) store(y + o2, x2[u]);
      }
      store(y + o1, x1[u]);
    }
  }
}

template <typename T, int V, int MODE, bool LOOSE = false>
static int launch_rotary(const RotaryArgs& a, int64_t batch, hipStream_t s) {
  const int per = 256 / a.units;
  const int64_t grid = (a.tokens + per - 1) / per * batch * a.head_blocks;
  if (grid > (1LL << 31) - 1) return VSA_ERR_SHAPE;
  hipLaunchKernelGGL((rotary_kernel<T, V, MODE, LOOSE>), dim3((unsigned)grid), dim3(256), 0, s, a);
  return vsa_check_launch();
}

// v: channels of a piece that every start and length allows
template <typename T>
static int rotary_of(const RotaryArgs& a, int64_t batch, int v, int mode, hipStream_t s) {
  constexpr int W = 16 / sizeof(T);
  if (mode == kSwap) return launch_rotary<T, W, kSwap>(a, batch, s);   // (v is W)
  const bool inter = mode == kInter;
  if constexpr (sizeof(T) == 2) {
    if (v == 8)
      return inter ? launch_rotary<T, 8, kInter>(a, batch, s) : launch_rotary<T, 8, kTwo>(a, batch, s);
  }
  if (v == 4)
    return inter ? launch_rotary<T, 4, kInter>(a, batch, s) : launch_rotary<T, 4, kTwo>(a, batch, s);
  if (v == 2)
    return inter ? launch_rotary<T, 2, kInter>(a, batch, s) : launch_rotary<T, 2, kTwo>(a, batch, s);
  return inter ? launch_rotary<T, 2, kInter, true>(a, batch, s) : launch_rotary<T, 1, kTwo>(a, batch, s);
}

}  // namespace vsa

using namespace vsa;

extern "C" int vsa_rotary_table(const vsa_rotary_axis* axes, float* cos_out, float* sin_out,
                                void* stream) {
  if (!axes || !cos_out || !sin_out) return VSA_ERR_NULL;
  if (!vsa_aligned<4>(cos_out, sin_out)) return VSA_ERR_ALIGN;
  TableArgs a;
  int pairs = 0;
  int64_t tokens = 1;
  for (int x = 0; x < 3; ++x) {
    const vsa_rotary_axis& ax = axes[x];
    if (ax.positions <= 0 || ax.channels < 0 || ax.channels % 2 ||
        pairs + ax.channels / 2 > kMaxPairs || !(ax.theta > 0) || !(ax.factor > 0) ||
        !isfinite(ax.theta) || !isfinite(ax.factor) || !(fabs(ax.start) <= 4503599627370496.0))
      return VSA_ERR_SHAPE;
    const int n = ax.channels / 2;
    double theta = ax.theta;
    a.n[x] = ax.positions;
    a.pairs[x] = n;
    a.start[x] = ax.start;
    a.size[x] = 1.0;
    if (ax.method == VSA_ROTARY_NTK) {
      // the lowest frequency falls by the factor, the highest stays
      if (ax.channels > 2) theta *= pow(ax.factor, ax.channels / (ax.channels - 2.0));
    } else if (ax.method == VSA_ROTARY_YARN) {
      if (!(ax.original > 0) || !isfinite(ax.original)) return VSA_ERR_SHAPE;
      a.size[x] = 0.1 * log(ax.factor) + 1.0;
    } else if (ax.method != VSA_ROTARY_LINEAR) {
      return VSA_ERR_SHAPE;
    }
    for (int i = 0; i < n; ++i) {
      double f = pow(theta, -2.0 * i / ax.channels);
      if (ax.method == VSA_ROTARY_LINEAR) f /= ax.factor;
      if (ax.method == VSA_ROTARY_YARN) {
        // channels that turn 32 times or more in the trained length keep their
        // frequency, those that turn once or less are interpolated
        const double turns = ax.original * f / (2.0 * M_PI);
        const double keep = fmin(1.0, fmax(0.0, (turns - 1.0) / 31.0));
        f = f * keep + f / ax.factor * (1.0 - keep);
      }
      a.freq[pairs + i] = f;
    }
    pairs += n;
    if (tokens > (1LL << 31) / ax.positions) return VSA_ERR_SHAPE;
    tokens *= ax.positions;
  }
  if (pairs == 0) return VSA_ERR_SHAPE;
  const int64_t threads = (tokens + kTableRun - 1) / kTableRun * pairs;
  if ((threads + 255) / 256 > (1LL << 31) - 1) return VSA_ERR_SHAPE;
  hipLaunchKernelGGL(rotary_table_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0,
                     (hipStream_t)stream, a, pairs, tokens, cos_out, sin_out);
  return vsa_check_launch();
}

extern "C" int vsa_rotary(const vsa_rotary_op* op, void* stream) {
  if (!op || !op->q || !op->q_out || !op->cos_table || !op->sin_table ||
      (op->k_heads > 0 && (!op->k || !op->k_out)))
    return VSA_ERR_NULL;
  if (op->dtype != VSA_BF16 && op->dtype != VSA_F16 && op->dtype != VSA_F32) return VSA_ERR_DTYPE;
  const int es = op->dtype == VSA_F32 ? 4 : 2;
  if (op->batch <= 0 || op->tokens <= 0 || op->q_heads <= 0 || op->k_heads < 0 ||
      op->q_heads > (1 << 20) || op->k_heads > (1 << 20) || op->head_dim <= 0 ||
      op->head_dim > 256 || op->channels <= 0 || op->channels % 2 ||
      op->channels > op->head_dim || op->rows <= 0 || (!op->positions && op->rows < op->tokens))
    return VSA_ERR_SHAPE;
  if (!vsa_aligned<4>(op->cos_table, op->sin_table) ||
      (uintptr_t)op->positions % (op->positions64 ? 8 : 4))
    return VSA_ERR_ALIGN;
  RotaryArgs a;
  a.x[0] = op->q, a.x[1] = op->k, a.y[0] = op->q_out, a.y[1] = op->k_out;
  // the widest pieces that every row's start and every piece of a row allow
  const bool inter = op->interleaved != 0;
  uint64_t low = (uint64_t)(inter ? op->channels : op->channels / 2) |
                 (uint64_t)(op->head_dim - op->channels) | 8;
  for (int w = 0; w < (op->k_heads ? 2 : 1); ++w) {
    low |= ((uint64_t)a.x[w] | (uint64_t)a.y[w]) / es;
    if (((uintptr_t)a.x[w] | (uintptr_t)a.y[w]) % es) return VSA_ERR_ALIGN;
  }
  for (int x = 0; x < 3; ++x) {
    a.xs[0][x] = op->q_stride[x], a.ys[0][x] = op->q_out_stride[x];
    a.xs[1][x] = op->k_stride[x], a.ys[1][x] = op->k_out_stride[x];
    low |= (uint64_t)(a.xs[0][x] | a.ys[0][x]);
    if (op->k_heads) low |= (uint64_t)(a.xs[1][x] | a.ys[1][x]);
  }
  int v = (int)(low & -low);
  if (v * es > 16) v = 16 / es;
  a.co = op->cos_table, a.si = op->sin_table;
  a.positions = op->positions;
  a.pos_batch = op->positions_stride;
  a.pos64 = op->positions64;
  a.rows = op->rows, a.tokens = op->tokens;
  a.heads_q = op->q_heads, a.heads = op->q_heads + op->k_heads;
  a.dim = op->head_dim, a.pairs = op->channels / 2;
  const int unit = inter && v == 1 ? 2 : v;
  const int rest = (op->head_dim - op->channels + unit - 1) / unit;
  int mode = inter ? kInter : kTwo;
  if (!inter && v * es == 16 && 64 % (op->channels / v + rest) == 0) mode = kSwap;
  a.turns = (mode == kTwo ? a.pairs : op->channels) / unit;
  a.units = a.turns + rest;
  a.sign = op->inverse ? -1.f : 1.f;
  // token-major memory, by q's strides
  a.heads_fastest = op->q_heads > 1 && op->tokens > 1 && a.xs[0][1] < a.xs[0][2];
  a.per_block = a.heads_fastest ? 8 : 4;
  a.head_blocks = (a.heads + a.per_block - 1) / a.per_block;
  hipStream_t s = (hipStream_t)stream;
  VSA_DISPATCH_ALL(op->dtype, T, return rotary_of<T>(a, op->batch, v, mode, s));
}
