// Cross attention, forward (the mathematics and the copies: cross.h).
//
// One wave owns 32 query rows, a workgroup NW waves; the rows of a (sample, key
// head) are those of its group's heads one after the other, so that a few
// queries of a shared key head fill one tile.  The workgroup walks the key
// chunks of its split (a chunk without a valid key is skipped); the copy of the
// next chunk is in flight while this one is multiplied.
//   S^T (KC x 32) = K Q^T      A = K rows from LDS, B = Q in registers
//   online softmax, a lane per query: the running max moves only where a chunk
//   passes it by more than 2^8, so O is seldom rescaled
//   O^T (D x 32) += V^T P^T    A = V columns from LDS, B = P from the S result
// With splits the parts (O normalised, base-2 LSE) go to fp32 scratch and a
// second kernel joins them by their LSE.  Up to 64 rows (16 bits) run
// cross_few_kernel instead, whose waves share the keys.
//
// P is rounded to T for its product, once, at most 2^8 (a moved maximum's slack);
// the sum of the weights is of the fp32 ones.
//
// Bound by the products and exponentials a tile takes, with the reading of q and
// the writing of O at its start and end on top where it has few chunks: 40 heads x
// 41k queries of 128 channels on 512 keys 0.50 ms, 860 TFLOP/s (matrix core busy
// for 45 % of the cycles, at the 1.7 GHz that the chip's power allows; q and O alone
// 0.17 ms); on 2048 keys of 24 heads x 16k queries 0.42 ms, 980.
#include <algorithm>
#include <type_traits>

#include "cross.h"

namespace vsa {

constexpr float kSlack = 8.0f;  // log2 units

template <typename T, int D, int NW>
struct CrossFwdCfg {
  static constexpr int NT = NW * 64;
  // 128 channels: 32 keys leave registers for three waves a SIMD, 64 for two (40 heads
  // x 41k queries on 512 keys 0.508 / 0.540 ms).  64 channels: 64 keys 582 us, 32 598
  // (24 heads x 41k queries on 2048), 13.1 / 15.2 (12 heads x 2000 on 512).
  static constexpr int KC = sizeof(T) == 2 && D < 128 && NW == 4 ? 64 : 32;
  static constexpr int NSM = KC / 32;
  static constexpr int TILE = KC * D * (int)sizeof(T);   // bytes of a K (or V) chunk
  static constexpr int STAGE = 2 * TILE;
  static constexpr int WPE = D * (int)sizeof(T) > 256 ? 1 : sizeof(T) == 2 ? 3 : 2;
};

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(CrossFwdCfg<T, D, NW>::WPE)))
void cross_fwd_kernel(CrossArgs a) {
  using C = CrossFwdCfg<T, D, NW>;
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
  const int row = own % a.per_head * (32 * NW) + wave * 32 + r;  // of group * sq
  const int rows = a.group * a.sq;
  const int at = min(row, rows - 1);
  const int head = kh * a.group + at / a.sq, sq_i = at % a.sq;

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
  const bool any = have;
  if (have) copy(0);   // in flight with the rows' loads

  V8 qf[D / 16];
  {
    const T* qrow = (const T*)a.q.p + b * a.q.b + head * a.q.h + sq_i * a.q.s;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int d = 16 * ks + 8 * h;
      V8 x = zero8<T>();
      if (d < a.dim) x = ld8<T>(qrow + d);
      // a negative softmax scale is folded into q (the sign bit of each element)
      if constexpr (sizeof(T) == 2) {
        u32x4 raw = __builtin_bit_cast(u32x4, x);
        raw ^= a.qsign;
        qf[ks] = as_vec8<T>(raw);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(__float_as_uint(x[e]) ^ a.qsign);
        qf[ks] = x;
      }
    }
  }
  float m = -INFINITY, lsum = 0.f;
  f32x16 oacc[D / 32];
#pragma unroll
  for (int mt = 0; mt < D / 32; ++mt) oacc[mt] = f32x16{};

  dma_wait();
  __syncthreads();
  // one chunk, of stage `stage` (a constant: every LDS address is a lane offset
  // plus an immediate)
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

    f32x16 sacc[C::NSM];
#pragma unroll
    for (int x = 0; x < C::NSM; ++x) sacc[x] = f32x16{};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      if (!in_dim<T>(16 * ks, a.dim)) break;
#pragma unroll
      for (int x = 0; x < C::NSM; ++x) sacc[x] = M::mul(ops.row(Ks, x, ks), qf[ks], sacc[x]);
      step_fence<T, D>();
    }
    if (!whole) {
      keep_branch();
#pragma unroll
      for (int x = 0; x < C::NSM; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) sacc[x][i] = acc_valid(w[x], i) ? sacc[x][i] : -INFINITY;
    }
    float m4[4] = {sacc[0][0], sacc[0][1], sacc[0][2], sacc[0][3]};
#pragma unroll
    for (int x = 0; x < C::NSM; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) m4[i & 3] = vmax(m4[i & 3], sacc[x][i]);
    const float smax = pair_max32(vmax(vmax(m4[0], m4[1]), vmax(m4[2], m4[3]))) * a.c2;
    const bool grow = smax > m + kSlack;
    if (__any(grow)) {
      const float mnew = grow ? smax : m;
      const float alpha = m == mnew ? 1.f : fast_exp2(m - mnew);
      lsum *= alpha;
#pragma unroll
      for (int mt = 0; mt < D / 32; ++mt) oacc[mt] *= alpha;
      m = mnew;
    }
    const float negm = m == -INFINITY ? 0.f : -m;
    float p[C::NSM][16];
#pragma unroll
    for (int x = 0; x < C::NSM; ++x)
#pragma unroll
      for (int i = 0; i < 16; ++i) p[x][i] = fast_exp2(fmaf(sacc[x][i], a.c2, negm));
    float l4[4] = {p[0][0], p[0][1], p[0][2], p[0][3]};
#pragma unroll
    for (int x = 4; x < 16 * C::NSM; ++x) l4[x & 3] += p[x >> 4][x & 15];
    lsum += (l4[0] + l4[1]) + (l4[2] + l4[3]);
#pragma unroll
    for (int kk = 0; kk < 2 * C::NSM; ++kk) {
      const V8 bop = pack_op<T>(&p[kk >> 1][8 * (kk & 1)]);
#pragma unroll
      for (int mt = 0; mt < D / 32; ++mt) {
        if (!in_dim<T>(32 * mt, a.dim)) break;
        oacc[mt] = M::mul(ops.col(Vs, 0, mt, kk), bop, oacc[mt]);
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

  const float total = pair_sum32(lsum);
  const float inv = any ? 1.0f / total : 0.f;   // no valid key: zeros
  const bool store = row < rows;
  float w8[2][8];
  if (a.splits > 1) {
    const int64_t prow = ((int64_t)split * a.batch * a.kv_heads + hk) * rows + row;
#pragma unroll
    for (int mt = 0; mt < D / 32; ++mt) {
      swap_rows16(oacc[mt], inv, w8);
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (store) st8<float>(a.part_a + prow * D + mt * 32 + 16 * x + 8 * h, w8[x]);
    }
    if (store && h == 0) a.part_b[prow] = any ? m + log2f(total) : -INFINITY;
    return;
  }
  T* orow = (T*)a.out + b * a.out_s[0] + head * a.out_s[1] + sq_i * a.out_s[2];
  const int64_t stat = ((int64_t)b * a.heads + head) * a.sq + sq_i;
  uint8_t* lrow = a.lo ? a.lo + stat * a.dim : nullptr;
#pragma unroll
  for (int mt = 0; mt < D / 32; ++mt) {
    swap_rows16(oacc[mt], inv, w8);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int d = mt * 32 + 16 * x + 8 * h;
      if (store && d < a.dim) st8_out<T>(orow + d, lrow ? lrow + d : nullptr, w8[x]);
    }
  }
  if (store && h == 0 && a.lse) a.lse[stat] = any ? m + log2f(total) : -INFINITY;
}

// 32 NQ query rows of a (sample, key head) on its keys, for up to 64 of them: bound by reading K
// and V, so the waves of a workgroup share the keys, not the rows.  Each walks
// every NW-th chunk of 32 keys through a ring of its own in LDS (no barrier: a
// wave waits for its own copies), and the parts meet in LDS at the end.
// Splits over workgroups are for long keys alone.
template <typename T, int D>
struct CrossFewCfg {
  static constexpr int TILE = 32 * D * (int)sizeof(T);
  static constexpr int RING = 4 * TILE;                    // two chunks of K and V
  static constexpr int NW = D == 64 ? 8 : D == 128 ? 4 : 2;
  static constexpr int LDS = NW * RING;                    // 128 KiB
  typedef TileCopy<T, D, 32, 64> Copy;
};

template <typename T, int D, int NQ>
__global__ __launch_bounds__((CrossFewCfg<T, D>::NW * 64)) void cross_few_kernel(CrossArgs a) {
  using C = CrossFewCfg<T, D>;
  using M = Mma<T>;
  typedef typename M::V8 V8;
  constexpr int NW = C::NW, TT = NQ * (D / 32);
  __shared__ __attribute__((aligned(16))) char smem[C::LDS];
  __shared__ float stat_s[NW][NQ][2][64];
  static_assert(NW * TT * 16 * 256 <= C::LDS, "the parts fit the rings");

  const int own = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const int hk = own / a.per_head, row0 = own % a.per_head * 32 * NQ;
  const int b = hk / a.kv_heads, kh = hk % a.kv_heads;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5;
  const int rows = a.group * a.sq;
  const char* ring = smem + wave * C::RING;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem)) + wave * C::RING;

  const T* kbase = (const T*)a.k.p + b * a.k.b + kh * a.k.h;
  const T* vbase = (const T*)a.v.p + b * a.v.b + kh * a.v.h;
  typename C::Copy kcopy, vcopy;
  kcopy.init(a.k.s, a.dim, lane);
  vcopy.init(a.v.s, a.dim, lane);
  const int chunks = (a.skv + 31) / 32;
  const int per_split = (chunks + a.splits - 1) / a.splits;
  KeyWalk<32> walk;
  walk.init(a, b, split * per_split, per_split);
  walk.j += wave;
  uint32_t next_w = 0;
  auto copy = [&](int stage) __attribute__((always_inline)) {
    const int left = walk.n - walk.j * 32;
    const auto ks = kcopy.rows(kbase + (int64_t)walk.j * 32 * a.k.s, left);
    const auto vs = vcopy.rows(vbase + (int64_t)walk.j * 32 * a.v.s, left);
    const uint32_t to = lds0 + stage * 2 * C::TILE;
    if (!walk.holes()) {
      kcopy.copy(to, ks);
      vcopy.copy(to + C::TILE, vs);
    } else {
      kcopy.copy_valid(to, ks, walk.w);
      vcopy.copy_valid(to + C::TILE, vs, walk.w);
    }
    next_w = walk.w[0];
  };
  uint32_t w = 0;
  bool have = walk.template find<NW>();
  if (have) {
    copy(0);
    w = next_w;
    walk.j += NW;
  }
  bool ahead = have && walk.template find<NW>();
  if (ahead) copy(1);
  const bool any = have;

  V8 qf[NQ][D / 16];
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    const int at = min(row0 + 32 * t + r, rows - 1);
    const T* qrow = (const T*)a.q.p + b * a.q.b + (kh * a.group + at / a.sq) * a.q.h + at % a.sq * a.q.s;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int d = 16 * ks + 8 * h;
      V8 x = zero8<T>();
      if (d < a.dim) x = ld8<T>(qrow + d);
      u32x4 raw = __builtin_bit_cast(u32x4, x);
      raw ^= a.qsign;   // a negative softmax scale
      qf[t][ks] = as_vec8<T>(raw);
    }
  }
  Operands<T, D> ops;
  ops.init(ring, r, h);
  float m[NQ], lsum[NQ];
  f32x16 oacc[NQ][D / 32];
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    m[t] = -INFINITY, lsum[t] = 0.f;
#pragma unroll
    for (int mt = 0; mt < D / 32; ++mt) oacc[t][mt] = f32x16{};
  }
  int stage = 0;
  while (have) {
    // this chunk has landed (the loads of the one ahead may be in flight)
    if (ahead) wait_vmcnt<2 * C::Copy::N>();
    else dma_wait();
    asm volatile("" ::: "memory");   // no read of the stage moves before its wait
    __builtin_amdgcn_sched_barrier(0);
    const int Ks = stage * 2 * C::TILE, Vs = Ks + C::TILE;
    f32x16 s[NQ];
#pragma unroll
    for (int t = 0; t < NQ; ++t) s[t] = f32x16{};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const V8 k = ops.row(Ks, 0, ks);
#pragma unroll
      for (int t = 0; t < NQ; ++t) s[t] = M::mul(k, qf[t][ks], s[t]);
    }
    V8 bop[NQ][2];
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
      if (w != ~0u) {
        keep_branch();
#pragma unroll
        for (int i = 0; i < 16; ++i) s[t][i] = acc_valid(w, i) ? s[t][i] : -INFINITY;
      }
      float m4[4] = {s[t][0], s[t][1], s[t][2], s[t][3]};
#pragma unroll
      for (int i = 4; i < 16; ++i) m4[i & 3] = vmax(m4[i & 3], s[t][i]);
      const float smax = pair_max32(vmax(vmax(m4[0], m4[1]), vmax(m4[2], m4[3]))) * a.c2;
      const bool grow = smax > m[t] + kSlack;
      if (__any(grow)) {
        const float mnew = grow ? smax : m[t];
        const float alpha = m[t] == mnew ? 1.f : fast_exp2(m[t] - mnew);
        lsum[t] *= alpha;
#pragma unroll
        for (int mt = 0; mt < D / 32; ++mt) oacc[t][mt] *= alpha;
        m[t] = mnew;
      }
      const float negm = m[t] == -INFINITY ? 0.f : -m[t];
      float p[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = fast_exp2(fmaf(s[t][i], a.c2, negm));
      float l4[4] = {p[0], p[1], p[2], p[3]};
#pragma unroll
      for (int i = 4; i < 16; ++i) l4[i & 3] += p[i];
      lsum[t] += (l4[0] + l4[1]) + (l4[2] + l4[3]);
      bop[t][0] = pack_op<T>(p);
      bop[t][1] = pack_op<T>(p + 8);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int mt = 0; mt < D / 32; ++mt) {
        const V8 v = ops.col(Vs, 0, mt, kk);
#pragma unroll
        for (int t = 0; t < NQ; ++t) oacc[t][mt] = M::mul(v, bop[t][kk], oacc[t][mt]);
      }
    // every read of this stage has returned (its product has been issued)
    __builtin_amdgcn_sched_barrier(0);
    have = ahead;
    w = next_w;
    if (have) {
      walk.j += NW;
      ahead = walk.template find<NW>();
      if (ahead) copy(stage);
    }
    stage ^= 1;
  }

  // the waves' parts: their sums as registers of 64 lanes, their m and l
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    stat_s[wave][t][0][lane] = m[t];
    stat_s[wave][t][1][lane] = pair_sum32(lsum[t]);
  }
  const bool some = __syncthreads_or(any);   // and every ring is done with
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int t = 0; t < NQ; ++t)
#pragma unroll
    for (int mt = 0; mt < D / 32; ++mt)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        part[((wave * TT + t * (D / 32) + mt) * 16 + i) * 64 + lane] = oacc[t][mt][i];
  __syncthreads();
  for (int x = wave; x < TT; x += NW) {
    const int t = x / (D / 32), mt = x % (D / 32);
    float top = -INFINITY, total = 0.f, weight[NW];
#pragma unroll
    for (int y = 0; y < NW; ++y) top = vmax(top, stat_s[y][t][0][lane]);
#pragma unroll
    for (int y = 0; y < NW; ++y) {
      const float own = stat_s[y][t][0][lane];
      // (a wave without a chunk has -inf and sums of 0; so has a row whose scores
      // are all -inf, and then 0 / 0 below)
      weight[y] = own == -INFINITY ? 0.f : fast_exp2(own - top);
      total = fmaf(weight[y], stat_s[y][t][1][lane], total);
    }
    f32x16 o = f32x16{};
#pragma unroll
    for (int y = 0; y < NW; ++y)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        o[i] = fmaf(weight[y], part[((y * TT + x) * 16 + i) * 64 + lane], o[i]);
    const float inv = some ? 1.0f / total : 0.f;
    float w8[2][8];
    swap_rows16(o, inv, w8);
    const int row = row0 + 32 * t + r;
    if (row >= rows) continue;
    const int head = kh * a.group + row / a.sq, sq_i = row % a.sq;
    const int64_t stat = ((int64_t)b * a.heads + head) * a.sq + sq_i;
    const float lse = some ? top + log2f(total) : -INFINITY;
#pragma unroll
    for (int z = 0; z < 2; ++z) {
      const int d = mt * 32 + 16 * z + 8 * h;
      if (a.splits > 1) {
        st8<float>(a.part_a + (((int64_t)split * a.batch * a.kv_heads + hk) * rows + row) * D + d, w8[z]);
      } else if (d < a.dim) {
        st8_out<T>((T*)a.out + b * a.out_s[0] + head * a.out_s[1] + sq_i * a.out_s[2] + d,
                   a.lo ? a.lo + stat * a.dim + d : nullptr, w8[z]);
      }
    }
    if (h == 0 && mt == 0) {
      if (a.splits > 1) a.part_b[((int64_t)split * a.batch * a.kv_heads + hk) * rows + row] = lse;
      else if (a.lse) a.lse[stat] = lse;
    }
  }
}

// Joins the splits' parts: out = sum_s 2^(lse_s - L) O_s / sum_s 2^(lse_s - L).  A
// row has D / 8 threads of eight channels, times `lanes` that take every
// lanes-th split each and meet in LDS (one thread a row's piece walked a hundred
// splits alone: 52 us for 64 queries on 40960 keys, as long as the attention).
template <typename T, int D>
__global__ __launch_bounds__(256) void cross_join_kernel(CrossArgs a, int lanes) {
  constexpr int W = D / 8;
  __shared__ float acc_s[256][9];
  __shared__ float top_s[256];
  const int rows = a.group * a.sq;
  const int64_t all = (int64_t)a.batch * a.kv_heads * rows;
  const int piece = threadIdx.x % W, lane = threadIdx.x / W % lanes;
  const int64_t prow = (int64_t)blockIdx.x * (256 / W / lanes) + threadIdx.x / W / lanes;
  const int d = piece * 8;
  float top = -INFINITY, sum = 0.f, acc[8] = {};
  if (prow < all) {
    for (int s = lane; s < a.splits; s += lanes) {
      const float* p = a.part_a + (s * all + prow) * D + d;
      const f32x4 x = *reinterpret_cast<const f32x4*>(p), y = *reinterpret_cast<const f32x4*>(p + 4);
      const float l = a.part_b[s * all + prow];
      if (l == -INFINITY) continue;
      const float next = fmaxf(top, l), scale = fast_exp2(top - next), w = fast_exp2(l - next);
      top = next;
      sum = fmaf(sum, scale, w);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[e] = fmaf(acc[e], scale, w * x[e]);
        acc[4 + e] = fmaf(acc[4 + e], scale, w * y[e]);
      }
    }
  }
  if (lanes > 1) {
    top_s[threadIdx.x] = top;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc_s[threadIdx.x][e] = acc[e];
    acc_s[threadIdx.x][8] = sum;
    __syncthreads();
    if (lane) return;
    float t = top;
    for (int x = 1; x < lanes; ++x) t = fmaxf(t, top_s[threadIdx.x + x * W]);
    const float own = top == -INFINITY ? 0.f : fast_exp2(top - t);
    sum *= own;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= own;
    for (int x = 1; x < lanes; ++x) {
      const int at = threadIdx.x + x * W;
      const float w = top_s[at] == -INFINITY ? 0.f : fast_exp2(top_s[at] - t);
      sum = fmaf(w, acc_s[at][8], sum);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, acc_s[at][e], acc[e]);
    }
    top = t;
  }
  if (prow >= all) return;
  const float inv = top == -INFINITY ? 0.f : 1.0f / sum;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] *= inv;
  const int hk = (int)(prow / rows), i = (int)(prow % rows);
  const int b = hk / a.kv_heads, head = hk % a.kv_heads * a.group + i / a.sq;
  const int64_t stat = ((int64_t)b * a.heads + head) * a.sq + i % a.sq;
  if (d < a.dim)
    st8_out<T>((T*)a.out + b * a.out_s[0] + head * a.out_s[1] + (i % a.sq) * a.out_s[2] + d,
               a.lo ? a.lo + stat * a.dim + d : nullptr, acc);
  if (d == 0 && a.lse) a.lse[stat] = top == -INFINITY ? top : top + log2f(sum);
}

// 32 keys of a sample to a word: its key_mask and its kv_lens.
__global__ __launch_bounds__(256) void cross_words_kernel(const uint8_t* __restrict__ mask,
                                                          int64_t stride,
                                                          const int32_t* __restrict__ lens,
                                                          uint32_t* __restrict__ words, int nwords,
                                                          int skv) {
  const int b = blockIdx.y, key = blockIdx.x * 256 + threadIdx.x;
  const int n = lens ? min(max(lens[b], 0), skv) : skv;
  const uint64_t bits = __ballot(key < n && mask[b * stride + key] != 0);
  const int word = key >> 5;
  if ((threadIdx.x & 31) == 0 && word < nwords)
    words[(int64_t)b * nwords + word] = (uint32_t)(threadIdx.x & 32 ? bits >> 32 : bits);
}

namespace {

struct Plan {
  int kd, nw, nq;      // nq: 32-row tiles of the few-row kernel, 0 for the other
  int splits, per_head;
  int64_t tiles;
};

int fwd_kc(const vsa_cross* c, int kd, int nw) {
  return c->dtype != VSA_F32 && kd < 128 && nw == 4 ? 64 : 32;
}

Plan fwd_plan(const vsa_cross* c) {
  Plan p = {};
  const int64_t rows = c->heads / c->kv_heads * c->sq, heads = (int64_t)c->batch * c->kv_heads;
  p.kd = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256;
  if (c->dtype != VSA_F32 && rows <= 64) {
    p.nq = rows <= 32 || p.kd == 256 ? 1 : 2;   // (two at head dim 256 spill)
    p.nw = p.kd == 64 ? 8 : p.kd == 128 ? 4 : 2;
    p.per_head = (int)((rows + 32 * p.nq - 1) / (32 * p.nq));
    p.tiles = heads * p.per_head;
    // a workgroup a CU; splits only where a wave has more than eight chunks
    const int64_t chunks = (c->skv + 31) / 32;
    int64_t splits = std::max<int64_t>(1, cu_count() / p.tiles);
    splits = std::max<int64_t>(1, std::min(splits, chunks / (8 * p.nw)));
    const int64_t per = (chunks + splits - 1) / splits;
    p.splits = (int)((chunks + per - 1) / per);
    return p;
  }
  // (two waves at least for fp32 at head dim 256: one has too many pieces to copy)
  const bool wide = c->dtype == VSA_F32 && p.kd == 256;
  p.nw = rows <= 32 && !wide ? 1 : rows <= 64 ? 2 : 4;
  p.per_head = (int)((rows + 32 * p.nw - 1) / (32 * p.nw));
  p.tiles = heads * p.per_head;
  // (measured with 4 waves on an idle chip; fp32 leaves out channels past the head dim)
  const int kc = fwd_kc(c, p.kd, p.nw);
  const double us = c->dtype == VSA_F32 ? 0.036 * c->head_dim : (0.1 + 0.0052 * p.kd) * kc / 32;
  p.splits = (int)split_keys(p.tiles, (int64_t)cu_count() * (4 / p.nw), (c->skv + kc - 1) / kc, us,
                             (double)heads * rows * p.kd * 4e-6);
  return p;
}

}  // namespace

int64_t cross_fwd_parts(const vsa_cross* c) {
  const Plan p = fwd_plan(c);
  if (p.splits == 1) return 0;
  const int64_t rows = (int64_t)c->batch * c->heads * c->sq * p.splits;
  return rows * (p.kd + 1) * 4;
}

int cross_words(const vsa_cross* c, uint32_t* words, int nwords, hipStream_t s) {
  hipLaunchKernelGGL(cross_words_kernel, dim3((unsigned)((nwords + 7) / 8), (unsigned)c->batch),
                     dim3(256), 0, s, (const uint8_t*)c->key_mask, c->mask_stride, c->kv_lens, words,
                     nwords, (int)c->skv);
  return vsa_check_launch();
}

template <typename T, int D>
static int launch_fwd(const Plan& p, const CrossArgs& a, hipStream_t s) {
  const unsigned grid = (unsigned)((p.tiles * p.splits + 7) / 8 * 8);
  if constexpr (sizeof(T) == 2) {
    const dim3 few((unsigned)(p.tiles * p.splits)), nt(CrossFewCfg<T, D>::NW * 64);
    if (p.nq == 1) hipLaunchKernelGGL((cross_few_kernel<T, D, 1>), few, nt, 0, s, a);
    else if (p.nq == 0) hipLaunchKernelGGL((cross_fwd_kernel<T, D, 4>), dim3(grid), dim3(256), 0, s, a);
    else if constexpr (D < 256) hipLaunchKernelGGL((cross_few_kernel<T, D, 2>), few, nt, 0, s, a);
  } else {
    if (p.nw == 4) hipLaunchKernelGGL((cross_fwd_kernel<T, D, 4>), dim3(grid), dim3(256), 0, s, a);
    else if (D == 256 || p.nw == 2)
      hipLaunchKernelGGL((cross_fwd_kernel<T, D, 2>), dim3(grid), dim3(128), 0, s, a);
    else if constexpr (D < 256)
      hipLaunchKernelGGL((cross_fwd_kernel<T, D, 1>), dim3(grid), dim3(64), 0, s, a);
  }
  const int rc = vsa_check_launch();
  if (rc || p.splits == 1) return rc;
  int lanes = 1;   // a power of two up to the threads that a row can have
  while (lanes < a.splits && lanes < 256 / (D / 8)) lanes *= 2;
  const int64_t n = (int64_t)a.batch * a.heads * a.sq, per = 256 / (D / 8) / lanes;
  hipLaunchKernelGGL((cross_join_kernel<T, D>), dim3((unsigned)((n + per - 1) / per)), dim3(256), 0,
                     s, a, lanes);
  return vsa_check_launch();
}

template <typename T>
static int fwd_of(const Plan& p, const CrossArgs& a, hipStream_t s) {
  if (p.kd == 64) return launch_fwd<T, 64>(p, a, s);
  if (p.kd == 128) return launch_fwd<T, 128>(p, a, s);
  return launch_fwd<T, 256>(p, a, s);
}

int cross_fwd(const vsa_cross* c, CrossArgs a, char* scratch, hipStream_t s) {
  const Plan p = fwd_plan(c);
  a.splits = p.splits;
  a.per_head = p.per_head;
  if (p.tiles * p.splits > (1LL << 31) - 16) return VSA_ERR_SHAPE;
  a.tiles = (int)p.tiles;
  if (p.splits > 1) {
    a.part_a = (float*)scratch;
    a.part_b = a.part_a + (int64_t)c->batch * c->heads * c->sq * p.splits * p.kd;
  }
  VSA_DISPATCH_ALL(c->dtype, T, return fwd_of<T>(p, a, s));
}

}  // namespace vsa
