// Cross attention, backward (the mathematics and the copies: cross.h).
//
//   P = 2^(c2 Q K^T - lse)        delta = sum over channels of dO (O + lo)
//   dS = P (dO V^T - delta)
//   dQ = scale dS K      dK = scale dS^T Q      dV = P^T dO
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

#include "cross.h"

namespace vsa {

template <typename T, int D, int NW>
struct CrossDqCfg {
  static constexpr int NT = NW * 64;
  static constexpr int KC = 32;
  static constexpr int TILE = KC * D * (int)sizeof(T);
  static constexpr int STAGE = 2 * TILE;
  static constexpr int WPE = D * (int)sizeof(T) > 256 ? 1 : 2;
};

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(CrossDqCfg<T, D, NW>::WPE)))
void cross_dq_kernel(CrossArgs a) {
  using C = CrossDqCfg<T, D, NW>;
  using M = Mma<T>;
  typedef typename M::V8 V8;
  constexpr int KC = C::KC;
  __shared__ __attribute__((aligned(16))) char smem[2 * C::STAGE];

  const int tile = xcd_tile(blockIdx.x, a.tiles * a.splits);
  if (tile >= a.tiles * a.splits) return;
  const int split = tile % a.splits, own = tile / a.splits;
  const int hk = own / a.per_head;
  const int b = hk / a.kv_heads, kh = hk % a.kv_heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 31, h = lane >> 5;
  const int row = (own % a.per_head) * (32 * NW) + wave * 32 + r;
  const int rows = a.group * a.sq;
  const int at = min(row, rows - 1);
  const int head = kh * a.group + at / a.sq, sq_i = at % a.sq;
  const int64_t stat = ((int64_t)b * a.heads + head) * a.sq + sq_i;

  V8 qf[D / 16], gf[D / 16];
  float delta = 0.f;
  {
    const T* qrow = (const T*)a.q.p + b * a.q.b + head * a.q.h + sq_i * a.q.s;
    const T* grow = (const T*)a.dout.p + b * a.dout.b + head * a.dout.h + sq_i * a.dout.s;
    const T* orow = (const T*)a.o.p + b * a.o.b + head * a.o.h + sq_i * a.o.s;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int d = 16 * ks + 8 * h;
      qf[ks] = gf[ks] = zero8<T>();
      if (d < a.dim) {
        qf[ks] = ld8<T>(qrow + d);
        gf[ks] = ld8<T>(grow + d);
        const V8 o = ld8<T>(orow + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)gf[ks][e], (float)o[e], delta);
        if (sizeof(T) == 2 && a.lo) {
          const V8 l = ld8<T>((const T*)a.lo + stat * a.dim + d);
#pragma unroll
          for (int e = 0; e < 8; ++e) delta = fmaf((float)gf[ks][e], (float)l[e], delta);
        }
      }
    }
    delta = pair_sum32(delta);
  }
  const bool store = row < rows;
  if (store && h == 0 && split == 0) a.delta[stat] = delta;
  const float lse = a.lse[stat];

  const T* kbase = (const T*)a.k.p + b * a.k.b + kh * a.k.h;
  const T* vbase = (const T*)a.v.p + b * a.v.b + kh * a.v.h;
  TileCopy<T, D, KC, C::NT> kcopy, vcopy;
  kcopy.init(a.k.s, a.dim);
  vcopy.init(a.v.s, a.dim);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem));
  const bool dim_full = a.dim == D;
  const int chunks = (a.skv + KC - 1) / KC;
  const int per_split = (chunks + a.splits - 1) / a.splits;
  KeyWalk<KC> walk;
  walk.init(a, b, split * per_split, per_split);
  auto copy = [&](int stage) {
    const T* ks = kbase + (int64_t)walk.j * KC * a.k.s;
    const T* vs = vbase + (int64_t)walk.j * KC * a.v.s;
    const uint32_t to = lds0 + stage * C::STAGE;
    if (dim_full && walk.whole()) {
      kcopy.whole(to, ks);
      vcopy.whole(to + C::TILE, vs);
    } else {
      kcopy.part(to, ks, walk.w);
      vcopy.part(to + C::TILE, vs, walk.w);
    }
  };

  f32x16 dq[D / 32];
#pragma unroll
  for (int mt = 0; mt < D / 32; ++mt) dq[mt] = f32x16{};
  bool have = walk.find();
  if (have) copy(0);
  dma_wait();
  __syncthreads();
  int stage = 0;
  while (have) {
    const uint32_t w = walk.w[0];
    const bool whole = walk.whole();
    ++walk.j;
    have = walk.find();
    if (have) copy(stage ^ 1);
    const char* Ks = smem + stage * C::STAGE;
    const char* Vs = Ks + C::TILE;
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      s = M::mul(row_op<T, D>(Ks, r, ks, h), qf[ks], s);
      dp = M::mul(row_op<T, D>(Vs, r, ks, h), gf[ks], dp);
      step_fence<T, D>();
    }
    float ds[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) ds[i] = fast_exp2(fmaf(s[i], a.c2, -lse)) * (dp[i] - delta);
    if (!whole) {
      keep_branch();
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (!acc_valid(w, i, h)) ds[i] = 0.f;
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      // dS is rounded to T for the product, as P is for O
      const V8 bop = pack_op<T>(&ds[8 * kk]);
#pragma unroll
      for (int mt = 0; mt < D / 32; ++mt)
        dq[mt] = M::mul(col_op<T, D>(Ks, mt * 32, 16 * kk), bop, dq[mt]), step_fence<T, D>();
    }
    dma_wait();
    __syncthreads();
    stage ^= 1;
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

// DA: channels of dK and dV that a workgroup sums (half of them at head dim 256,
// where K, V and all sums would not fit a wave's registers).
template <typename T, int D, int NW>
struct CrossDkvCfg {
  static constexpr int NT = NW * 64;
  static constexpr int DA = D > 128 ? 128 : D;
  static constexpr int TILE = 32 * D * (int)sizeof(T);
  static constexpr int STAGE = 2 * TILE + 256;   // Q, dO, 32 lse, 32 delta
  static constexpr int WPE = D * (int)sizeof(T) > 128 ? 1 : 2;
};

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(CrossDkvCfg<T, D, NW>::WPE)))
void cross_dkv_kernel(CrossArgs a) {
  using C = CrossDkvCfg<T, D, NW>;
  using M = Mma<T>;
  typedef typename M::V8 V8;
  constexpr int DA = C::DA, HALVES = D / DA;
  __shared__ __attribute__((aligned(16))) char smem[2 * C::STAGE];

  const int tile = xcd_tile(blockIdx.x, a.tiles * a.splits);
  if (tile >= a.tiles * a.splits) return;
  const int split = tile % a.splits;
  int own = tile / a.splits;
  const int d0 = own % HALVES * DA;
  own /= HALVES;
  const int hk = own / a.per_head;
  const int b = hk / a.kv_heads, kh = hk % a.kv_heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 31, h = lane >> 5;
  const int first_key = own % a.per_head * (32 * NW);
  const int key = first_key + wave * 32 + r;
  int n = a.skv;
  if (a.lens) n = min(max(a.lens[b], 0), a.skv);
  bool valid = key < n;
  if (valid && a.words) valid = (a.words[(int64_t)b * a.nwords + (key >> 5)] >> (key & 31)) & 1u;
  // (for a tile without a valid key this workgroup only writes zeros)
  const bool live = __syncthreads_or(valid);

  V8 kf[D / 16], vf[D / 16];
  {
    const int at = min(key, a.skv - 1);
    const T* krow = (const T*)a.k.p + b * a.k.b + kh * a.k.h + (int64_t)at * a.k.s;
    const T* vrow = (const T*)a.v.p + b * a.v.b + kh * a.v.h + (int64_t)at * a.v.s;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int d = 16 * ks + 8 * h;
      kf[ks] = vf[ks] = zero8<T>();
      if (valid && d < a.dim) {
        kf[ks] = ld8<T>(krow + d);
        vf[ks] = ld8<T>(vrow + d);
      }
    }
  }
  f32x16 dk[DA / 32], dv[DA / 32];
#pragma unroll
  for (int mt = 0; mt < DA / 32; ++mt) dk[mt] = dv[mt] = f32x16{};

  const int qt = (a.sq + 31) / 32, items = a.group * qt;
  const int per_split = (items + a.splits - 1) / a.splits;
  int item = split * per_split;
  const int last = live ? min(item + per_split, items) : item;
  TileCopy<T, D, 32, C::NT> qcopy, gcopy;
  qcopy.init(a.q.s, a.dim);
  gcopy.init(a.dout.s, a.dim);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem));
  const bool dim_full = a.dim == D;
  auto copy = [&](int stage, int it) {
    const int head = kh * a.group + it / qt, s0 = it % qt * 32;
    const T* qs = (const T*)a.q.p + b * a.q.b + head * a.q.h + (int64_t)s0 * a.q.s;
    const T* gs = (const T*)a.dout.p + b * a.dout.b + head * a.dout.h + (int64_t)s0 * a.dout.s;
    const uint32_t to = lds0 + stage * C::STAGE;
    const int left = a.sq - s0;
    if (dim_full && left >= 32) {
      qcopy.whole(to, qs);
      gcopy.whole(to + C::TILE, gs);
    } else {
      const uint32_t w[1] = {left >= 32 ? ~0u : (1u << left) - 1u};
      qcopy.part(to, qs, w);
      gcopy.part(to + C::TILE, gs, w);
    }
    if (wave == 0) {
      const int64_t st = ((int64_t)b * a.heads + head) * a.sq + s0 + r;
      const float* g = (h ? a.delta : a.lse) + st;
      if (r >= left) g = kPastStats + h;
      dma4(g, to + 2 * C::TILE);
    }
  };

  if (item < last) copy(0, item);
  dma_wait();
  __syncthreads();
  int stage = 0;
  for (; item < last; ++item) {
    if (item + 1 < last) copy(stage ^ 1, item + 1);
    const char* Qs = smem + stage * C::STAGE;
    const char* Gs = Qs + C::TILE;
    const float* st = reinterpret_cast<const float*>(Gs + C::TILE);
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      s = M::mul(row_op<T, D>(Qs, r, ks, h), kf[ks], s);
      dp = M::mul(row_op<T, D>(Gs, r, ks, h), vf[ks], dp);
      step_fence<T, D>();
    }
    float p[16], ds[16];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 lse = *reinterpret_cast<const f32x4*>(st + 8 * g + 4 * h);
      const f32x4 del = *reinterpret_cast<const f32x4*>(st + 32 + 8 * g + 4 * h);
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
        dv[mt] = M::mul(col_op<T, D>(Gs, d0 + mt * 32, 16 * kk), pb, dv[mt]);
        dk[mt] = M::mul(col_op<T, D>(Qs, d0 + mt * 32, 16 * kk), sb, dk[mt]);
        step_fence<T, D>();
      }
    }
    dma_wait();
    __syncthreads();
    stage ^= 1;
  }

  // keys that are not valid get zeros
  const bool store = key < a.skv;
  const int64_t prow = ((int64_t)split * a.batch * a.kv_heads + hk) * a.skv + key;
  T* krow = (T*)a.dk + b * a.dk_s[0] + kh * a.dk_s[1] + (int64_t)key * a.dk_s[2];
  T* vrow = (T*)a.dv + b * a.dv_s[0] + kh * a.dv_s[1] + (int64_t)key * a.dv_s[2];
  float wk[2][8], wv[2][8];
#pragma unroll
  for (int mt = 0; mt < DA / 32; ++mt) {
    swap_rows16(dk[mt], a.scale, wk);
    swap_rows16(dv[mt], 1.f, wv);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int d = d0 + mt * 32 + 16 * x + 8 * h;
      if (!store || d >= a.dim) continue;
      if (!valid)
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

// out = sum of the splits' parts, in their order; one thread per eight channels
// of a row.  blockIdx.y picks one of two results.
struct SumArgs {
  const float* part[2];
  void* out[2];
  int64_t s[2][3];
  int64_t rows;        // batch * heads * tokens
  int splits, heads, tokens, dim;
};
template <typename T, int D>
__global__ __launch_bounds__(256) void cross_sum_kernel(SumArgs a) {
  const int y = blockIdx.y;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = id / (D / 8);
  const int d = (int)(id % (D / 8)) * 8;
  if (row >= a.rows || d >= a.dim) return;
  float acc[8] = {};
  for (int s = 0; s < a.splits; ++s) {
    const float* p = a.part[y] + (s * a.rows + row) * D + d;
    const f32x4 u = *reinterpret_cast<const f32x4*>(p), v = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += u[e], acc[4 + e] += v[e];
  }
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

int64_t splits_for(int64_t tiles, int64_t fit, int64_t steps, int64_t least) {
  int64_t s = tiles >= fit ? 1 : fit / tiles;
  s = std::max<int64_t>(1, std::min(s, steps / least));
  const int64_t per = (steps + s - 1) / s;
  return (steps + per - 1) / per;
}

Plan bwd_plan(const vsa_cross* c) {
  Plan p;
  const int64_t group = c->heads / c->kv_heads, rows = group * c->sq;
  const int es = c->dtype == VSA_F32 ? 4 : 2;
  p.kd = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256;
  p.q_nw = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  p.q_per_head = (int)((rows + 32 * p.q_nw - 1) / (32 * p.q_nw));
  p.q_tiles = (int64_t)c->batch * c->kv_heads * p.q_per_head;
  const int lds = 4 * 32 * p.kd * es;
  int64_t fit = (int64_t)cu_count() * std::max(1, std::min(160 * 1024 / lds, 8 / p.q_nw));
  p.q_splits = (int)splits_for(p.q_tiles, fit, (c->skv + 31) / 32, 4);
  // two waves for fp32 at head dim 256 (four spill)
  p.k_nw = c->skv <= 32 ? 1 : c->skv <= 64 || p.kd * es > 512 ? 2 : 4;
  p.k_per_head = (int)((c->skv + 32 * p.k_nw - 1) / (32 * p.k_nw));
  p.k_tiles = (int64_t)c->batch * c->kv_heads * p.k_per_head * (p.kd > 128 ? 2 : 1);
  fit = (int64_t)cu_count() *
        std::max(1, std::min(160 * 1024 / (lds + 512), (p.kd * es > 128 ? 4 : 8) / p.k_nw));
  p.k_splits = (int)splits_for(p.k_tiles, fit, group * ((c->sq + 31) / 32), 4);
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
static int launch_sum(const SumArgs& a, int results, hipStream_t s) {
  const int64_t grid = (a.rows * (D / 8) + 255) / 256;
  if (grid > (1LL << 31) - 1) return VSA_ERR_SHAPE;
  hipLaunchKernelGGL((cross_sum_kernel<T, D>), dim3((unsigned)grid, results), dim3(256), 0, s, a);
  return vsa_check_launch();
}

template <typename T, int D>
static int launch_bwd(const Plan& p, CrossArgs a, char* scratch, hipStream_t s) {
  a.tiles = (int)p.q_tiles, a.per_head = p.q_per_head, a.splits = p.q_splits;
  a.part_a = (float*)scratch;
  const unsigned qgrid = (unsigned)((p.q_tiles * p.q_splits + 7) / 8 * 8);
  if (p.q_nw == 1) hipLaunchKernelGGL((cross_dq_kernel<T, D, 1>), dim3(qgrid), dim3(64), 0, s, a);
  else if (p.q_nw == 2) hipLaunchKernelGGL((cross_dq_kernel<T, D, 2>), dim3(qgrid), dim3(128), 0, s, a);
  else hipLaunchKernelGGL((cross_dq_kernel<T, D, 4>), dim3(qgrid), dim3(256), 0, s, a);
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
  if (p.k_nw == 1) hipLaunchKernelGGL((cross_dkv_kernel<T, D, 1>), dim3(kgrid), dim3(64), 0, s, a);
  else if (p.k_nw == 2) hipLaunchKernelGGL((cross_dkv_kernel<T, D, 2>), dim3(kgrid), dim3(128), 0, s, a);
  else if constexpr (D * sizeof(T) <= 512)
    hipLaunchKernelGGL((cross_dkv_kernel<T, D, 4>), dim3(kgrid), dim3(256), 0, s, a);
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
