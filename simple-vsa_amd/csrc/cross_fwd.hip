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
// second kernel joins them by their LSE.
#include <algorithm>

#include "cross.h"

namespace vsa {

constexpr float kSlack = 8.0f;  // log2 units

template <typename T, int D, int NW>
struct CrossFwdCfg {
  static constexpr int NT = NW * 64;
  static constexpr int KC = sizeof(T) == 2 && D <= 128 && NW == 4 ? 64 : 32;
  static constexpr int NSM = KC / 32;
  static constexpr int TILE = KC * D * (int)sizeof(T);   // bytes of a K (or V) chunk
  static constexpr int STAGE = 2 * TILE;
  static constexpr int WPE = D * (int)sizeof(T) > 256 ? 1 : 2;
};

template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(CrossFwdCfg<T, D, NW>::WPE)))
void cross_fwd_kernel(CrossArgs a) {
  using C = CrossFwdCfg<T, D, NW>;
  using M = Mma<T>;
  typedef typename M::V8 V8;
  constexpr int KC = C::KC;
  __shared__ __attribute__((aligned(16))) char smem[2 * C::STAGE];

  const int tile = xcd_tile(blockIdx.x, a.tiles * a.splits);
  if (tile >= a.tiles * a.splits) return;
  const int split = tile % a.splits, own = tile / a.splits;
  const int hk = own / a.per_head;                  // batch * kv_heads + key head
  const int b = hk / a.kv_heads, kh = hk % a.kv_heads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 31, h = lane >> 5;
  const int row = (own % a.per_head) * (32 * NW) + wave * 32 + r;  // of group * sq
  const int rows = a.group * a.sq;
  const int at = min(row, rows - 1);
  const int head = kh * a.group + at / a.sq, sq_i = at % a.sq;

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

  float m = -INFINITY, lsum = 0.f;
  f32x16 oacc[D / 32];
#pragma unroll
  for (int mt = 0; mt < D / 32; ++mt) oacc[mt] = f32x16{};

  bool have = walk.find();
  const bool any = have;
  if (have) copy(0);
  dma_wait();
  __syncthreads();
  int stage = 0;
  while (have) {
    uint32_t w[C::NSM];
#pragma unroll
    for (int x = 0; x < C::NSM; ++x) w[x] = walk.w[x];
    const bool whole = walk.whole();
    ++walk.j;
    have = walk.find();
    if (have) copy(stage ^ 1);
    const char* Ks = smem + stage * C::STAGE;
    const char* Vs = Ks + C::TILE;

    f32x16 sacc[C::NSM];
#pragma unroll
    for (int x = 0; x < C::NSM; ++x) sacc[x] = f32x16{};
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
      for (int x = 0; x < C::NSM; ++x)
        sacc[x] = M::mul(row_op<T, D>(Ks, 32 * x + r, ks, h), qf[ks], sacc[x]);
      step_fence<T, D>();
    }
    if (!whole) {
      keep_branch();
#pragma unroll
      for (int x = 0; x < C::NSM; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!acc_valid(w[x], i, h)) sacc[x][i] = -INFINITY;
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
    if (!whole) {   // with c2 = 0 the masked scores' -inf is lost
      keep_branch();
#pragma unroll
      for (int x = 0; x < C::NSM; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!acc_valid(w[x], i, h)) p[x][i] = 0.f;
    }
    float l4[4] = {p[0][0], p[0][1], p[0][2], p[0][3]};
#pragma unroll
    for (int x = 4; x < 16 * C::NSM; ++x) l4[x & 3] += p[x >> 4][x & 15];
    lsum += (l4[0] + l4[1]) + (l4[2] + l4[3]);
#pragma unroll
    for (int kk = 0; kk < 2 * C::NSM; ++kk) {
      const V8 bop = pack_op<T>(&p[kk >> 1][8 * (kk & 1)]);
#pragma unroll
      for (int mt = 0; mt < D / 32; ++mt)
        oacc[mt] = M::mul(col_op<T, D>(Vs, mt * 32, 16 * kk), bop, oacc[mt]), step_fence<T, D>();
    }
    dma_wait();
    __syncthreads();
    stage ^= 1;
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
  T* lrow = a.lo ? (T*)a.lo + stat * a.dim : nullptr;
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

// Joins the splits' parts: out = sum_s 2^(lse_s - L) O_s, L the row's LSE.  One
// thread per eight channels of a row.
template <typename T, int D>
__global__ __launch_bounds__(256) void cross_join_kernel(CrossArgs a) {
  const int rows = a.group * a.sq;
  const int64_t all = (int64_t)a.batch * a.kv_heads * rows;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t prow = id / (D / 8);
  const int d = (int)(id % (D / 8)) * 8;
  if (prow >= all) return;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_b[s * all + prow]);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f, acc[8] = {};
  for (int s = 0; s < a.splits; ++s) {
    const float l = a.part_b[s * all + prow];
    const float w = fast_exp2(l - base);
    sum += w;
    const float* p = a.part_a + (s * all + prow) * D + d;
    const f32x4 x = *reinterpret_cast<const f32x4*>(p), y = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[e] = fmaf(w, x[e], acc[e]);
      acc[4 + e] = fmaf(w, y[e], acc[4 + e]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] *= inv;
  const int hk = (int)(prow / rows), i = (int)(prow % rows);
  const int b = hk / a.kv_heads, head = hk % a.kv_heads * a.group + i / a.sq;
  const int64_t stat = ((int64_t)b * a.heads + head) * a.sq + i % a.sq;
  if (d < a.dim)
    st8_out<T>((T*)a.out + b * a.out_s[0] + head * a.out_s[1] + (i % a.sq) * a.out_s[2] + d,
               a.lo ? (T*)a.lo + stat * a.dim + d : nullptr, acc);
  if (d == 0 && a.lse) a.lse[stat] = top == -INFINITY ? top : base + log2f(sum);
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
  int nw, kd, splits, per_head;
  int64_t tiles;
};

int fwd_kc(const vsa_cross* c, int kd, int nw) {
  return c->dtype != VSA_F32 && kd <= 128 && nw == 4 ? 64 : 32;
}

Plan fwd_plan(const vsa_cross* c) {
  Plan p;
  const int64_t rows = c->heads / c->kv_heads * c->sq;
  p.kd = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256;
  p.nw = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  p.per_head = (int)((rows + 32 * p.nw - 1) / (32 * p.nw));
  p.tiles = (int64_t)c->batch * c->kv_heads * p.per_head;
  // workgroups that the chip holds at once, by their LDS
  const int kc = fwd_kc(c, p.kd, p.nw);
  const int lds = 4 * kc * p.kd * (c->dtype == VSA_F32 ? 4 : 2);
  const int64_t fit = (int64_t)cu_count() * std::max(1, std::min(160 * 1024 / lds, 16 / p.nw));
  const int64_t chunks = (c->skv + kc - 1) / kc;
  int64_t splits = p.tiles >= fit ? 1 : fit / p.tiles;
  splits = std::max<int64_t>(1, std::min(splits, chunks / 4));
  const int64_t per = (chunks + splits - 1) / splits;
  p.splits = (int)((chunks + per - 1) / per);
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

template <typename T, int D, int NW>
static int launch_fwd(const CrossArgs& a, hipStream_t s) {
  using C = CrossFwdCfg<T, D, NW>;
  const int grid = (a.tiles * a.splits + 7) / 8 * 8;
  static_assert(2 * C::STAGE <= 160 * 1024, "");
  hipLaunchKernelGGL((cross_fwd_kernel<T, D, NW>), dim3((unsigned)grid), dim3(C::NT), 0, s, a);
  const int rc = vsa_check_launch();
  if (rc || a.splits == 1) return rc;
  const int64_t n = (int64_t)a.batch * a.heads * a.sq * (D / 8);
  hipLaunchKernelGGL((cross_join_kernel<T, D>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s,
                     a);
  return vsa_check_launch();
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
#define VSA_CROSS_NW(T, D)                             \
  do {                                                 \
    if (p.nw == 1) return launch_fwd<T, D, 1>(a, s);   \
    if (p.nw == 2) return launch_fwd<T, D, 2>(a, s);   \
    return launch_fwd<T, D, 4>(a, s);                  \
  } while (0)
  VSA_DISPATCH_ALL(c->dtype, T, {
    if (p.kd == 64) VSA_CROSS_NW(T, 64);
    if (p.kd == 128) VSA_CROSS_NW(T, 128);
    VSA_CROSS_NW(T, 256);
  });
#undef VSA_CROSS_NW
}

}  // namespace vsa
