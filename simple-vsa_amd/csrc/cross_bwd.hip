// Cross attention, backward (the mathematics and the copies: cross.h).
//
//   P = 2^(c2 Q K^T - lse)        delta = sum over channels of dO (O + lo)
//   dS = P (dO V^T - delta)
//   dQ = scale dS K      dK = scale dS^T Q      dV = P^T dO
//
// dQ's pass is bound by reading q, dO, O and its rest and writing dQ up to a few
// hundred keys (24 heads x 16k queries of 128 channels: 0.12 ms on 32 keys, 0.26 on
// 512), then by its products and exponentials (0.30 us a key); the other pass by
// the latter (0.36 us a key).
//
// Two passes, each sum owned by one workgroup (no atomics, a fixed order):
//  * dQ: a wave owns 32 query rows, as in the forward, and walks the keys; it
//    also makes delta, which the second pass reads;
//  * dK / dV: a wave owns 32 keys with K and V in registers and walks the
//    query rows of its group's heads, 32 at a time.
// Either pass is split over its long axis where its tiles do not fill the chip
// (a prompt of 512 keys has four key tiles a head): fp32 parts, then a sum in
// the order of the splits.
#include <algorithm>
#include <type_traits>

#include "cross.h"

namespace vsa {

template <typename T, int D, int NW>
struct CrossDqCfg {
  static constexpr int NT = NW * 64;
  static constexpr int KC = 32;
  static constexpr int NSM = KC / 32;
  static constexpr int TILE = KC * D * (int)sizeof(T);
  static constexpr int STAGE = 2 * TILE;
  static constexpr int WPE = D * (int)sizeof(T) > 256 ? 1 : D == 64 && sizeof(T) == 2 ? 3 : 2;
};

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(CrossDqCfg<T, D, NW>::WPE)))
void cross_dq_kernel(CrossArgs a) {
  using C = CrossDqCfg<T, D, NW>;
  using M = Mma<T>;
  typedef typename M::V8 V8;
  constexpr int KC = C::KC;
  __shared__ __attribute__((aligned(16))) char smem[2 * C::STAGE];

  const int tile = tile_of(a);
  if (tile >= a.tiles * a.splits) return;
  const int split = tile % a.splits, own = tile / a.splits;
  const int hk = own / a.per_head;                  // batch * kv_heads + key head
  const int b = hk / a.kv_heads, kh = hk % a.kv_heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 31, h = lane >> 5;
  const int row = own % a.per_head * (32 * NW) + wave * 32 + r;
  const int rows = a.group * a.sq;
  const int at = min(row, rows - 1);
  const int head = kh * a.group + at / a.sq, sq_i = at % a.sq;
  const int64_t stat = ((int64_t)b * a.heads + head) * a.sq + sq_i;

  const T* kbase = (const T*)a.k.p + b * a.k.b + kh * a.k.h;
  const T* vbase = (const T*)a.v.p + b * a.v.b + kh * a.v.h;
  TileCopy<T, D, KC, C::NT> kcopy, vcopy;
  kcopy.init(a.k.s, a.dim, threadIdx.x);
  vcopy.init(a.v.s, a.dim, threadIdx.x);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem));
  Operands<T, D> ops;
  ops.init(smem, r, h);
  const int chunks = (a.skv + KC - 1) / KC;
  const int per_split = (chunks + a.splits - 1) / a.splits;
  KeyWalk<KC> walk;
  walk.init(a, b, split * per_split, per_split);
  const float some = single_key(a, b, walk.n) ? 0.f : 1.f;
  auto copy = [&](int stage) __attribute__((always_inline)) {
    const int left = walk.n - walk.j * KC;
    const auto ks = kcopy.rows(kbase + (int64_t)walk.j * KC * a.k.s, left);
    const auto vs = vcopy.rows(vbase + (int64_t)walk.j * KC * a.v.s, left);
    const uint32_t to = lds0 + stage * C::STAGE;
    if (!walk.holes()) {
      kcopy.copy(to, ks);
      vcopy.copy(to + C::TILE, vs);
    } else {
      kcopy.copy_valid(to, ks, walk.w);
      vcopy.copy_valid(to + C::TILE, vs, walk.w);
    }
  };

  bool have = walk.find();
  if (have) copy(0);   // in flight with the rows' loads

  V8 qf[D / 16], gf[D / 16];
  float delta = 0.f;
  {
    const T* qrow = (const T*)a.q.p + b * a.q.b + head * a.q.h + sq_i * a.q.s;
    const T* grow = (const T*)a.dout.p + b * a.dout.b + head * a.dout.h + sq_i * a.dout.s;
    const T* orow = (const T*)a.o.p + b * a.o.b + head * a.o.h + sq_i * a.o.s;
    // tensor by tensor: the loads of a row's 128-byte lines follow each other (16k
    // queries on 32 keys, head dim 128: 0.160 -> 0.133 ms; 0.122 with the rests as bytes)
    auto load = [&](V8 (&f)[D / 16], const T* p) __attribute__((always_inline)) {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int d = 16 * ks + 8 * h;
        f[ks] = zero8<T>();
        if (d < a.dim) f[ks] = ld8<T>(p + d);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    const bool rest = sizeof(T) == 2 && a.lo;
    const uint8_t* lrow = a.lo + stat * a.dim;
    auto rests = [&](int d) __attribute__((always_inline)) {
      return *reinterpret_cast<const u32x2*>(lrow + d);
    };
    auto dot = [&](V8 g, V8 o) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf((float)g[e], (float)o[e], delta);
    };
    if constexpr (kWide<T, D>) {   // (no registers for O as a whole)
      load(gf, grow);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int d = 16 * ks + 8 * h;
        if (d < a.dim) {
          const V8 o = ld8<T>(orow + d);
          if constexpr (sizeof(T) == 2) {
            if (rest) {
              delta = dot_rest<T>(gf[ks], o, rests(d), delta);
              continue;
            }
          }
          dot(gf[ks], o);
        }
      }
      load(qf, qrow);
    } else {
      V8 of[D / 16];
      u32x2 lf[D / 16];
      load(gf, grow);
      load(of, orow);
      if (rest) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          lf[ks] = 16 * ks + 8 * h < a.dim ? rests(16 * ks + 8 * h) : u32x2{0, 0};
        __builtin_amdgcn_sched_barrier(0);
      }
      load(qf, qrow);
      // (channels past the head dim: g is 0, and o and its rest are finite)
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        if constexpr (sizeof(T) == 2) {
          if (rest) {
            delta = dot_rest<T>(gf[ks], of[ks], lf[ks], delta);
            continue;
          }
        }
        dot(gf[ks], of[ks]);
      }
    }
    delta = pair_sum32(delta);
  }
  const bool store = row < rows;
  if (store && h == 0 && split == 0) a.delta[stat] = delta;
  const float lse = a.lse[stat];

  f32x16 dq[D / 32];
#pragma unroll
  for (int mt = 0; mt < D / 32; ++mt) dq[mt] = f32x16{};
  dma_wait();
  __syncthreads();
  auto chunk = [&](auto stage_c) __attribute__((always_inline)) {
    const int stage = stage_c;
    const int Ks = stage * C::STAGE, Vs = Ks + C::TILE;
    uint32_t w[C::NSM];
#pragma unroll
    for (int x = 0; x < C::NSM; ++x) w[x] = walk.w[x];
    const bool whole = walk.whole();
    ++walk.j;
    have = walk.find();
    if (have) copy(stage ^ 1);
    f32x16 s[C::NSM], dp[C::NSM];
#pragma unroll
    for (int x = 0; x < C::NSM; ++x) s[x] = dp[x] = f32x16{};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      if (!in_dim<T>(16 * ks, a.dim)) break;
#pragma unroll
      for (int x = 0; x < C::NSM; ++x) {
        s[x] = M::mul(ops.row(Ks, x, ks), qf[ks], s[x]);
        dp[x] = M::mul(ops.row(Vs, x, ks), gf[ks], dp[x]);
      }
      step_fence<T, D>();
    }
    float ds[C::NSM][16];
#pragma unroll
    for (int x = 0; x < C::NSM; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        ds[x][i] = fast_exp2(fmaf(s[x][i], a.c2, -lse)) * (dp[x][i] - delta);
    if (!whole) {   // (a masked key's P may be infinite; a single key's chunk is never whole)
      keep_branch();
#pragma unroll
      for (int x = 0; x < C::NSM; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[x][i] = acc_valid(w[x], i) ? ds[x][i] * some : 0.f;
    }
#pragma unroll
    for (int kk = 0; kk < 2 * C::NSM; ++kk) {
      // dS as T and what that leaves over: rounded once, a third more of this
      // pass' products less, dQ is further off than its own rounding makes it
      // (bf16, 512 keys: 2.5e-3 of its norm against 1.7e-3)
      V8 hi, lo;
      pack_both<T>(&ds[kk >> 1][8 * (kk & 1)], hi, lo);
#pragma unroll
      for (int mt = 0; mt < D / 32; ++mt) {
        if (!in_dim<T>(32 * mt, a.dim)) break;
        const V8 k = ops.col(Ks, 0, mt, kk);
        dq[mt] = M::mul(k, hi, dq[mt]);
        if constexpr (sizeof(T) == 2) dq[mt] = M::mul(k, lo, dq[mt]);
        step_fence<T, D>();
      }
    }
    dma_wait();
    __syncthreads();
  };
  if constexpr (kWide<T, D>) {   // two copies of the body do not fit its registers
    for (int stage = 0; have; stage ^= 1) chunk(stage);
  } else {
    while (have) {
      chunk(std::integral_constant<int, 0>{});
      if (!have) break;
      chunk(std::integral_constant<int, 1>{});
    }
  }
  float w8[2][8];
  T* out = (T*)a.dq + b * a.dq_s[0] + head * a.dq_s[1] + sq_i * a.dq_s[2];
  float* part = a.part_a + ((int64_t)split * a.batch * a.kv_heads * rows + (int64_t)hk * rows + row) * D;
#pragma unroll
  for (int mt = 0; mt < D / 32; ++mt) {
    swap_rows16(dq[mt], a.scale, w8);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int d = mt * 32 + 16 * x + 8 * h;
      if (!store || d >= a.dim) continue;
      if (a.splits > 1) st8<float>(part + d, w8[x]);
      else st8<T>(out + d, w8[x]);
    }
  }
}

// The pass over the queries.  A wave owns 32 KT keys (K and V in registers), a
// workgroup NW waves; an item is 32 query rows of one head: their Q and dO tiles
// and their lse and delta, in a ring of NS stages in LDS.
//   S = Q K^T, dP = dO V^T     A = Q / dO rows,    B = K / V
//   dV^T += dO^T P, dK^T += Q^T dS   A = dO / Q columns, B = P / dS from S and dP
// DA: channels of dK and dV that a workgroup sums (half of them at head dim 256, a
// quarter in fp32: K, V and all sums would not fit a wave's registers).
//
// At 16 bits a SIMD holds one wave (K, V, the sums and two items' S and dP fill
// its registers), so the wave itself overlaps the matrix core with the rest:
// step i multiplies S and dP of item i + 1 while it works out P and dS of item
// i, then dV and dK of item i; operands are read from LDS AHEAD products before
// their use, and the copy of item i + 3 is spread over the second half.
// 2 x 12 heads, 16k queries on 512 and 256 keys, head dim 128: 0.23 ms (0.45 without
// the overlap); on 2048 keys 1.1 PFLOP/s.
template <typename T, int D, int NW>
struct CrossDkvCfg {
  static constexpr int NT = NW * 64;
  static constexpr bool PIPE = sizeof(T) == 2;
  static constexpr int DA = D <= 128 ? D : PIPE ? 128 : 64;
  static constexpr int KT = PIPE && D == 64 ? 2 : 1;     // 32-key tiles of a wave
  static constexpr int KEYS = 32 * KT * NW;              // keys of a workgroup
  static constexpr int TILE = 32 * D * (int)sizeof(T);
  static constexpr int STAGE = 2 * TILE + 256;           // Q, dO, 32 lse, 32 delta
  static constexpr int NS = PIPE ? 4 : 2;
  typedef TileCopy<T, D, 32, NT> Copy;
  static constexpr int PER = 2 * Copy::N + 1;            // copies of a thread per item
  // loads in flight that leave up to `items` items of copies (the counter has 6 bits)
  static constexpr int wait(int items) { return items * PER < 63 ? items * PER : 63; }
  static constexpr int NA = 2 * (D / 16);                // Q and dO rows
  static constexpr int NC = 4 * (DA / 32);               // dO and Q columns
  static constexpr int NV = 16 * KT;                     // P values of a lane per item
  // Up to 64 keys (128 at head dim 64) the pass reads Q and dO for longer than it
  // multiplies, and dK takes what rounding dS leaves over as well: 24 heads x 16k
  // queries on 32 keys 42 us, 3 of them for it, on 64 keys at head dim 64 32 us, 4 of
  // them; dK is off 1.7e-3 of its norm instead of 2.4e-3.  For more keys it stays out (512: 241 -> 288 us).
  static constexpr bool BOTH = PIPE && NW <= 2;
  static constexpr int AHEAD = D > 128 || (KT > 1 && BOTH) ? 4 : KT > 1 ? 6 : 12;
};

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(1, 1)))
void cross_dkv_kernel(CrossArgs a) {
  using C = CrossDkvCfg<T, D, NW>;
  using M = Mma<T>;
  typedef typename M::V8 V8;
  constexpr int DA = C::DA, HALVES = D / DA, KT = C::KT;
  __shared__ __attribute__((aligned(16))) char smem[C::NS * C::STAGE];

  const int tile = tile_of(a);
  if (tile >= a.tiles * a.splits) return;
  const int split = tile % a.splits;
  int own = tile / a.splits;
  const int d0 = own % HALVES * DA;
  own /= HALVES;
  const int hk = own / a.per_head;                  // batch * kv_heads + key head
  const int b = hk / a.kv_heads, kh = hk % a.kv_heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 31, h = lane >> 5;
  const int key0 = own % a.per_head * C::KEYS + wave * 32 * KT + r;
  int n = a.skv;
  if (a.lens) n = min(max(a.lens[b], 0), a.skv);
  bool valid[KT], some = false;
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    const int key = key0 + 32 * t;
    valid[t] = key < n;
    if (valid[t] && a.words)
      valid[t] = (a.words[(int64_t)b * a.nwords + (key >> 5)] >> (key & 31)) & 1u;
    some |= valid[t];
  }
  // a workgroup without a valid key only writes zeros
  const bool live = __syncthreads_or(some);

  V8 kf[KT][D / 16], vf[KT][D / 16];
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    const int at = min(key0 + 32 * t, a.skv - 1);
    const T* krow = (const T*)a.k.p + b * a.k.b + kh * a.k.h + (int64_t)at * a.k.s;
    const T* vrow = (const T*)a.v.p + b * a.v.b + kh * a.v.h + (int64_t)at * a.v.s;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int d = 16 * ks + 8 * h;
      kf[t][ks] = vf[t][ks] = zero8<T>();
      if (valid[t] && d < a.dim) {
        kf[t][ks] = ld8<T>(krow + d);
        vf[t][ks] = ld8<T>(vrow + d);
      }
    }
  }
  // Each sum leaves its zero through an asm of its own: with one zero shared by
  // all of them the compiler moves sums aside in every step.
  f32x16 dk[DA / 32][KT], dv[DA / 32][KT];
#pragma unroll
  for (int mt = 0; mt < DA / 32; ++mt)
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      dk[mt][t] = dv[mt][t] = f32x16{};
      if constexpr (C::PIPE) asm volatile("" : "+a"(dk[mt][t]), "+a"(dv[mt][t]));
    }

  const int qt = (a.sq + 31) / 32, all = a.group * qt;
  const int per_split = (all + a.splits - 1) / a.splits;
  const int first = split * per_split;
  const int items = live ? min(per_split, all - first) : 0;
  typename C::Copy qcopy, gcopy;
  qcopy.init(a.q.s, a.dim, threadIdx.x);
  gcopy.init(a.dout.s, a.dim, threadIdx.x);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem));
  Operands<T, D> ops;
  ops.init(smem, r, h);

  // An item's copy: descriptors of its rows, and this lane's statistic (lanes of
  // half 0 the lse, of half 1 the delta; every wave copies them, so that all
  // wait for the same number of loads).  Addresses go from item to item by
  // additions: a wave issues an instruction at a time, and products of 64 bits
  // for every item took a fifth of its step.
  struct Item {
    typename C::Copy::Src q, g;
    const float* stat;
  };
  const int head_f = first / qt, row_f = first % qt;
  const int head0 = kh * a.group + head_f;
  const T* qhead = (const T*)a.q.p + b * a.q.b + head0 * a.q.h;
  const T* ghead = (const T*)a.dout.p + b * a.dout.b + head0 * a.dout.h;
  const float* shead = (h ? a.delta : a.lse) + ((int64_t)b * a.heads + head0) * a.sq + r;
  // of the next item to copy
  const T* qrows = qhead + (int64_t)row_f * 32 * a.q.s;
  const T* grows = ghead + (int64_t)row_f * 32 * a.dout.s;
  const float* stat = shead + row_f * 32;
  int left = a.sq - row_f * 32;
  const int64_t qstep = 32 * a.q.s, gstep = 32 * a.dout.s;
  auto next_item = [&]() __attribute__((always_inline)) {
    Item it;
    it.q = qcopy.rows(qrows, left);
    it.g = gcopy.rows(grows, left);
    it.stat = r < left ? stat : kPastStats + h;
    return it;
  };
  // (past the last item its copy is made again, into a stage that no one reads)
  auto advance = [&](int i) __attribute__((always_inline)) {
    if (i >= items) return;
    left -= 32, qrows += qstep, grows += gstep, stat += 32;
    if (left <= 0) {
      keep_branch();
      left = a.sq;
      qrows = qhead += a.q.h;
      grows = ghead += a.dout.h;
      stat = shead += a.sq;
    }
  };
  auto piece = [&](const Item& it, int stage, int p) __attribute__((always_inline)) {
    const uint32_t to = lds0 + stage * C::STAGE;
    if (p < C::Copy::N) qcopy.piece(p, to, it.q);
    else if (p < 2 * C::Copy::N) gcopy.piece(p - C::Copy::N, to + C::TILE, it.g);
    else dma4(it.stat, __builtin_amdgcn_readfirstlane(lds0 + stage * C::STAGE + 2 * C::TILE));
  };
  auto stats = [&](int stage, int g, f32x4& lse, f32x4& del) __attribute__((always_inline)) {
    const char* st = smem + stage * C::STAGE + 2 * C::TILE + h * 16;
    lse = *reinterpret_cast<const f32x4*>(st + 32 * g);
    del = *reinterpret_cast<const f32x4*>(st + 128 + 32 * g);
  };

  if constexpr (!C::PIPE) {
    auto copy = [&](int stage) __attribute__((always_inline)) {
      const Item it = next_item();
#pragma unroll
      for (int p = 0; p < C::PER; ++p) piece(it, stage, p);
    };
    if (items > 0) copy(0);
    dma_wait();
    __syncthreads();
    auto step = [&](auto stage_c, int i) __attribute__((always_inline)) {
      const int S = stage_c, Qs = S * C::STAGE, Gs = Qs + C::TILE;
      advance(i + 1);
      if (i + 1 < items) copy(S ^ 1);
      f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        if (!in_dim<T>(16 * ks, a.dim)) break;
        s = M::mul(ops.row(Qs, 0, ks), kf[0][ks], s);
        dp = M::mul(ops.row(Gs, 0, ks), vf[0][ks], dp);
        step_fence<T, D>();
      }
      float p[16], ds[16];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 lse, del;
        stats(S, g, lse, del);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[4 * g + e] = fast_exp2(fmaf(s[4 * g + e], a.c2, -lse[e]));
          ds[4 * g + e] = p[4 * g + e] * (dp[4 * g + e] - del[e]);
        }
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const V8 pb = pack_op<T>(&p[8 * kk]), sb = pack_op<T>(&ds[8 * kk]);
#pragma unroll
        for (int mt = 0; mt < DA / 32; ++mt) {
          if (!in_dim<T>(d0 + 32 * mt, a.dim)) break;
          dv[mt][0] = M::mul(ops.col(Gs, d0, mt, kk), pb, dv[mt][0]);
          dk[mt][0] = M::mul(ops.col(Qs, d0, mt, kk), sb, dk[mt][0]);
          step_fence<T, D>();
        }
      }
      dma_wait();
      __syncthreads();
    };
    if constexpr (kWide<T, D>) {
      for (int i = 0; i < items; ++i) step(i & 1, i);
    } else {
      for (int i = 0; i < items; i += 2) {
        step(std::integral_constant<int, 0>{}, i);
        if (i + 1 < items) step(std::integral_constant<int, 1>{}, i + 1);
      }
    }
  } else if (items > 0) {
    constexpr int NS = C::NS, NA = C::NA, NC = C::NC, L = C::AHEAD;
    // stages 0 .. 2 get items 0 .. 2
    Item cp = next_item();
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) {
#pragma unroll
      for (int p = 0; p < C::PER; ++p) piece(cp, i, p);
      advance(i + 1);
      cp = next_item();
    }
    f32x16 sA[KT], pA[KT], sB[KT], pB[KT];
    f32x4 lA[4], eA[4], lB[4], eB[4];
    wait_vmcnt<C::wait(NS - 2)>();   // item 0 has landed
    __syncthreads();
#pragma unroll
    for (int t = 0; t < KT; ++t) sA[t] = pA[t] = f32x16{};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const V8 qa = ops.row(0, 0, ks), ga = ops.row(C::TILE, 0, ks);
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        sA[t] = M::mul(qa, kf[t][ks], sA[t]);
        pA[t] = M::mul(ga, vf[t][ks], pA[t]);
      }
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) stats(0, g, lA[g], eA[g]);
    // Step i (item i in stage S = i % 4): its barrier publishes item i + 1 and
    // ends every wave's reads of item i - 1, whose stage the copy of item i + 3
    // takes; at most one item of copies is left in flight by its wait.
    auto step = [&](auto stage_c, int i, f32x16 (&sc)[KT], f32x16 (&pc)[KT], f32x16 (&sn)[KT],
                    f32x16 (&pn)[KT], f32x4 (&lc)[4], f32x4 (&ec)[4], f32x4 (&ln)[4],
                    f32x4 (&en)[4]) __attribute__((always_inline)) {
      constexpr int S = decltype(stage_c)::value, SN = (S + 1) % NS, SP = (S + NS - 1) % NS;
      constexpr int Qn = SN * C::STAGE, Qc = S * C::STAGE;
      wait_vmcnt<C::wait(NS - 3)>();
      __syncthreads();
      V8 op[NA + NC];
      auto issue = [&](int x) __attribute__((always_inline)) {
        if (x < NA) {
          op[x] = ops.row(Qn + (x & 1) * C::TILE, 0, x >> 1);
        } else if (x < NA + NC) {
          const int y = x - NA;
          op[x] = ops.col(Qc + (y & 1 ? 0 : C::TILE), d0, (y >> 1) % (DA / 32), y / (2 * (DA / 32)));
        } else if (x < NA + NC + 4) {
          stats(SN, x - NA - NC, ln[x - NA - NC], en[x - NA - NC]);
        }
      };
#pragma unroll
      for (int x = 0; x < L; ++x) issue(x);
#pragma unroll
      for (int t = 0; t < KT; ++t) sn[t] = pn[t] = f32x16{};
      // P and dS of item i, spread over the products of item i + 1 and the first
      // half of its own: value x belongs to key tile (x / 8) % KT, element
      // 8 (x / 8 KT) + x % 8, the order in which the halves below take them
      float pv[KT][16], ds[KT][16];
      auto value = [&](int pos) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < C::NV; ++x) {
          if (x * (NA + NC / 2) / C::NV != pos) continue;
          const int t = x / 8 % KT, e = 8 * (x / (8 * KT)) + x % 8;
          pv[t][e] = fast_exp2(fmaf(sc[t][e], a.c2, -lc[e >> 2][e & 3]));
          ds[t][e] = pv[t][e] * (pc[t][e] - ec[e >> 2][e & 3]);
        }
      };
      static_assert(8 * KT * (NA + NC / 2) / C::NV <= NA, "the first half of dS ends before its use");
#pragma unroll
      for (int u = 0; u < NA; ++u) {
        issue(u + L);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          if (u & 1) pn[t] = M::mul(op[u], vf[t][u >> 1], pn[t]);
          else sn[t] = M::mul(op[u], kf[t][u >> 1], sn[t]);
        }
        value(u);
        __builtin_amdgcn_sched_barrier(0);
      }
      V8 bp[KT][2], bs[KT][2], bl[KT][2];
      auto pack = [&](int j) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          bp[t][j] = pack_op<T>(pv[t] + 8 * j);
          if constexpr (C::BOTH) pack_both<T>(ds[t] + 8 * j, bs[t][j], bl[t][j]);
          else bs[t][j] = pack_op<T>(ds[t] + 8 * j);
        }
      };
      pack(0);
#pragma unroll
      for (int y = 0; y < NC; ++y) {
        issue(NA + y + L);
        const int j = y / (2 * (DA / 32)), mt = (y >> 1) % (DA / 32);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          if (y & 1) dk[mt][t] = M::mul(op[NA + y], bs[t][j], dk[mt][t]);
          else dv[mt][t] = M::mul(op[NA + y], bp[t][j], dv[mt][t]);
          if (C::BOTH && (y & 1)) dk[mt][t] = M::mul(op[NA + y], bl[t][j], dk[mt][t]);
        }
#pragma unroll
        for (int p = 0; p < C::PER; ++p)
          if (NC / 2 + p * (NC / 2) / C::PER == y) piece(cp, SP, p);
        if (y < NC / 2) value(NA + y);
        if (y == NC / 2 - 1) pack(1);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int x = NA + NC + L; x < NA + NC + 4; ++x) issue(x);
      advance(i + NS);
      cp = next_item();
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    int i = 0;
    for (; i + 4 <= items; i += 4) {
      step(I0{}, i, sA, pA, sB, pB, lA, eA, lB, eB);
      step(I1{}, i + 1, sB, pB, sA, pA, lB, eB, lA, eA);
      step(I2{}, i + 2, sA, pA, sB, pB, lA, eA, lB, eB);
      step(I3{}, i + 3, sB, pB, sA, pA, lB, eB, lA, eA);
    }
    if (i < items) step(I0{}, i, sA, pA, sB, pB, lA, eA, lB, eB);
    if (i + 1 < items) step(I1{}, i + 1, sB, pB, sA, pA, lB, eB, lA, eA);
    if (i + 2 < items) step(I2{}, i + 2, sA, pA, sB, pB, lA, eA, lB, eB);
    dma_wait();   // the copies ahead of the last item land before the LDS is given up
  }

  // keys that are not valid get zeros
  const float dk_scale = single_key(a, b, __builtin_amdgcn_readfirstlane(n)) ? 0.f : a.scale;
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    const int key = key0 + 32 * t;
    const int64_t prow = ((int64_t)split * a.batch * a.kv_heads + hk) * a.skv + key;
    T* krow = (T*)a.dk + b * a.dk_s[0] + kh * a.dk_s[1] + (int64_t)key * a.dk_s[2];
    T* vrow = (T*)a.dv + b * a.dv_s[0] + kh * a.dv_s[1] + (int64_t)key * a.dv_s[2];
    float wk[2][8], wv[2][8];
#pragma unroll
    for (int mt = 0; mt < DA / 32; ++mt) {
      swap_rows16(dk[mt][t], dk_scale, wk);
      swap_rows16(dv[mt][t], 1.f, wv);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int d = d0 + mt * 32 + 16 * x + 8 * h;
        if (key >= a.skv || d >= a.dim) continue;
        if (!valid[t])
#pragma unroll
          for (int e = 0; e < 8; ++e) wk[x][e] = wv[x][e] = 0.f;
        if (a.splits > 1) {
          st8<float>(a.part_a + prow * D + d, wk[x]);
          st8<float>(a.part_b + prow * D + d, wv[x]);
        } else {
          st8<T>(krow + d, wk[x]);
          st8<T>(vrow + d, wv[x]);
        }
      }
    }
  }
}

// out = sum of the splits' parts, in a fixed order; blockIdx.y picks one of two
// results.  A row has D / 8 threads of eight channels, times `lanes` that sum every
// lanes-th split each and meet in LDS (256 splits of 128 rows by one thread a
// piece: 66 us, longer than the pass).
struct SumArgs {
  const float* part[2];
  void* out[2];
  int64_t s[2][3];
  int64_t rows;        // batch * heads * tokens
  int splits, heads, tokens, dim, lanes;
};
template <typename T, int D>
__global__ __launch_bounds__(256) void cross_sum_kernel(SumArgs a) {
  constexpr int W = D / 8;
  __shared__ float acc_s[256][9];
  const int y = blockIdx.y;
  const int d = threadIdx.x % W * 8, lane = threadIdx.x / W % a.lanes;
  const int64_t row = (int64_t)blockIdx.x * (256 / W / a.lanes) + threadIdx.x / W / a.lanes;
  const bool on = row < a.rows && d < a.dim;
  float acc[8] = {};
  if (on) {
#pragma unroll 4   // (loads ahead of the sums)
    for (int s = lane; s < a.splits; s += a.lanes) {
      const float* p = a.part[y] + (s * a.rows + row) * D + d;
      const f32x4 u = *reinterpret_cast<const f32x4*>(p), v = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += u[e], acc[4 + e] += v[e];
    }
  }
  if (a.lanes > 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc_s[threadIdx.x][e] = acc[e];
    __syncthreads();
    if (lane) return;
    for (int x = 1; x < a.lanes; ++x)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += acc_s[threadIdx.x + x * W][e];
  }
  if (!on) return;
  const int64_t bh = row / a.tokens, t = row % a.tokens;
  st8<T>((T*)a.out[y] + bh / a.heads * a.s[y][0] + bh % a.heads * a.s[y][1] + t * a.s[y][2] + d, acc);
}

namespace {

struct Plan {
  int kd;
  int q_nw, q_splits, q_per_head;      // dQ
  int k_nw, k_splits, k_per_head;      // dK / dV
  int64_t q_tiles, k_tiles;
};

// Splits of the pass over the queries.  With `fit` workgroups at once, s splits
// take ceil(tiles s / fit) rounds of steps / s items and a workgroup's own cost
// (about eight items: K and V in, the sums out), and their parts are written and
// read again.  Where samples may have fewer keys (`some`), a quarter and a half of
// the tiles having no valid one count as much as all of them at work.
int64_t dkv_splits(int64_t tiles, int64_t fit, int64_t steps, int nw, int es, bool some) {
  int64_t best = 1;
  double least = 1e300;
  // writing and reading a part takes 0.01 items' time for each wave's keys; an
  // fp32 item takes eight times a 16-bit one's time
  const double item = es == 2 ? 1 : 8, part = 0.01 * nw * (double)tiles / item;
  for (int64_t s = 1; s <= 64 && s <= steps; ++s) {
    const int64_t per = (steps + s - 1) / s;
    if ((steps + per - 1) / per != s) continue;
    double rounds = 0;
    for (int live = 4; live >= (some ? 2 : 4); --live)
      rounds += (double)(((tiles * live + 3) / 4 * s + fit - 1) / fit);
    if (some) rounds /= 3;
    const double cost = rounds * ((double)per + 8 / item) + (s > 1 ? 8 / item + part * (double)s : 0);
    if (cost < least) least = cost, best = s;
  }
  return best;
}

Plan bwd_plan(const vsa_cross* c) {
  Plan p = {};
  const int64_t group = c->heads / c->kv_heads, rows = group * c->sq;
  const int es = c->dtype == VSA_F32 ? 4 : 2;
  p.kd = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256;
  // (at head dim 256 in fp32 one wave has too many pieces to copy, and four spill in
  // the second pass; at 16 bits fewer than four spill there)
  const bool wide = p.kd * es > 512;
  p.q_nw = rows <= 32 && !wide ? 1 : rows <= 64 ? 2 : 4;
  p.q_per_head = (int)((rows + 32 * p.q_nw - 1) / (32 * p.q_nw));
  p.q_tiles = (int64_t)c->batch * c->kv_heads * p.q_per_head;
  const double us = es == 4 ? 0.048 * c->head_dim : 0.35 + 0.0055 * p.kd;
  p.q_splits = (int)split_keys(p.q_tiles, (int64_t)cu_count() * (4 / p.q_nw), (c->skv + 31) / 32, us,
                               (double)c->batch * c->kv_heads * rows * p.kd * 4e-6);
  const int wave_keys = es == 2 && p.kd == 64 ? 64 : 32;
  p.k_nw = wide ? 2 : p.kd == 256 ? 4 : c->skv <= wave_keys ? 1 : c->skv <= 2 * wave_keys ? 2 : 4;
  p.k_per_head = (int)((c->skv + wave_keys * p.k_nw - 1) / (wave_keys * p.k_nw));
  p.k_tiles = (int64_t)c->batch * c->kv_heads * p.k_per_head * (p.kd <= 128 ? 1 : es == 2 ? 2 : 4);
  const int stage = 2 * 32 * p.kd * es + 256;
  const int64_t kfit =
      (int64_t)cu_count() * std::max(1, std::min(160 * 1024 / (stage * (es == 2 ? 4 : 2)), 4 / p.k_nw));
  p.k_splits = (int)dkv_splits(p.k_tiles, kfit, group * ((c->sq + 31) / 32), p.k_nw, es,
                               c->batch > 1 && (c->kv_lens || c->key_mask));
  return p;
}

int64_t bytes_dq(const vsa_cross* c, const Plan& p) {
  return p.q_splits == 1 ? 0 : (int64_t)c->batch * c->heads * c->sq * p.q_splits * p.kd * 4;
}
int64_t bytes_dkv(const vsa_cross* c, const Plan& p) {
  return p.k_splits == 1 ? 0 : 2LL * c->batch * c->kv_heads * c->skv * p.k_splits * p.kd * 4;
}

}  // namespace

// the two passes use one scratch after the other
int64_t cross_bwd_parts(const vsa_cross* c) {
  const Plan p = bwd_plan(c);
  return std::max(bytes_dq(c, p), bytes_dkv(c, p));
}

template <typename T, int D>
static int launch_sum(SumArgs a, int results, hipStream_t s) {
  a.lanes = 1;   // a power of two, four splits or more each
  while (8 * a.lanes <= a.splits && a.lanes < 256 / (D / 8)) a.lanes *= 2;
  const int64_t per = 256 / (D / 8) / a.lanes, grid = (a.rows + per - 1) / per;
  if (grid > (1LL << 31) - 1) return VSA_ERR_SHAPE;
  hipLaunchKernelGGL((cross_sum_kernel<T, D>), dim3((unsigned)grid, results), dim3(256), 0, s, a);
  return vsa_check_launch();
}

template <typename T, int D>
static int launch_bwd(const Plan& p, CrossArgs a, char* scratch, hipStream_t s) {
  a.tiles = (int)p.q_tiles, a.per_head = p.q_per_head, a.splits = p.q_splits;
  a.part_a = (float*)scratch;
  const unsigned qgrid = (unsigned)((p.q_tiles * p.q_splits + 7) / 8 * 8);
  constexpr bool kWidest = D * sizeof(T) > 512;
  if (p.q_nw == 4)
    hipLaunchKernelGGL((cross_dq_kernel<T, D, 4>), dim3(qgrid), dim3(256), 0, s, a);
  else if (kWidest || p.q_nw == 2)
    hipLaunchKernelGGL((cross_dq_kernel<T, D, 2>), dim3(qgrid), dim3(128), 0, s, a);
  else if constexpr (!kWidest)
    hipLaunchKernelGGL((cross_dq_kernel<T, D, 1>), dim3(qgrid), dim3(64), 0, s, a);
  int rc = vsa_check_launch();
  if (rc) return rc;
  if (p.q_splits > 1) {
    SumArgs u = {};
    u.part[0] = a.part_a, u.out[0] = a.dq;
    for (int x = 0; x < 3; ++x) u.s[0][x] = a.dq_s[x];
    u.rows = (int64_t)a.batch * a.heads * a.sq;
    u.splits = p.q_splits, u.heads = a.heads, u.tokens = a.sq, u.dim = a.dim;
    if ((rc = launch_sum<T, D>(u, 1, s))) return rc;
  }
  a.tiles = (int)p.k_tiles, a.per_head = p.k_per_head, a.splits = p.k_splits;
  a.part_b = a.part_a + (int64_t)a.batch * a.kv_heads * a.skv * p.k_splits * D;
  const unsigned kgrid = (unsigned)((p.k_tiles * p.k_splits + 7) / 8 * 8);
  if constexpr (kWidest) {
    hipLaunchKernelGGL((cross_dkv_kernel<T, D, 2>), dim3(kgrid), dim3(128), 0, s, a);
  } else if (D == 256 || p.k_nw == 4) {
    hipLaunchKernelGGL((cross_dkv_kernel<T, D, 4>), dim3(kgrid), dim3(256), 0, s, a);
  } else if constexpr (D < 256) {
    if (p.k_nw == 2)
      hipLaunchKernelGGL((cross_dkv_kernel<T, D, 2>), dim3(kgrid), dim3(128), 0, s, a);
    else
      hipLaunchKernelGGL((cross_dkv_kernel<T, D, 1>), dim3(kgrid), dim3(64), 0, s, a);
  }
  if ((rc = vsa_check_launch()) || p.k_splits == 1) return rc;
  SumArgs u = {};
  u.part[0] = a.part_a, u.part[1] = a.part_b, u.out[0] = a.dk, u.out[1] = a.dv;
  for (int x = 0; x < 3; ++x) u.s[0][x] = a.dk_s[x], u.s[1][x] = a.dv_s[x];
  u.rows = (int64_t)a.batch * a.kv_heads * a.skv;
  u.splits = p.k_splits, u.heads = a.kv_heads, u.tokens = a.skv, u.dim = a.dim;
  return launch_sum<T, D>(u, 2, s);
}

template <typename T>
static int bwd_of(const Plan& p, const CrossArgs& a, char* scratch, hipStream_t s) {
  if (p.kd == 64) return launch_bwd<T, 64>(p, a, scratch, s);
  if (p.kd == 128) return launch_bwd<T, 128>(p, a, scratch, s);
  return launch_bwd<T, 256>(p, a, scratch, s);
}

int cross_bwd(const vsa_cross* c, const CrossArgs& a, char* scratch, hipStream_t s) {
  const Plan p = bwd_plan(c);
  if (p.q_tiles * p.q_splits > (1LL << 31) - 16 || p.k_tiles * p.k_splits > (1LL << 31) - 16)
    return VSA_ERR_SHAPE;
  VSA_DISPATCH_ALL(c->dtype, T, return bwd_of<T>(p, a, scratch, s));
}

}  // namespace vsa
