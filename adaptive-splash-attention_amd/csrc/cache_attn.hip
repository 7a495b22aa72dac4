// alpha-entmax attention of a few query tokens over the 4-bit cache.
//
// Per query row, with z_j = (alpha - 1) clamp(scale q.k_j, -10, 10) over the
// visible keys j and e = 1 / (alpha - 1):
//
//   sum_j max(z_j - tau, 0)^e = 1,  out = sum_j p_j v_j / sum_j p_j.
//
// The keys' bytes are what a row costs: 5 bits per channel, read once.  The
// codes never become keys.  With u = 16 + c (bf16 0x4180 | c << 3, exact),
// group g and its query part q_g,
//
//   q.k = sum_g s_g (q_g.u_g - 16 sum q_g) + sum_g m_g sum q_g:
//
// one v_mfma_f32_16x16x32_bf16 per group gives q_g.u_g for 16 rows x 16 keys
// (a group is the instruction's 32 channels), its accumulator starts at
// -16 sum q_g, the keys' scales multiply the finished group sums (a lane of
// the result holds one key, so G scales), and the offsets' part is one more
// MFMA over the groups.  Queries enter as exact sums of bf16 terms (bf16 1,
// fp16 2, fp32 3 terms), so that scores carry fp32 rounding only, for every
// type.
//
// tau lies in [max z - 1, max z], so only keys with z > max z - 1 can have a
// weight.  A better bound: the sum over any part of the row is at most the
// whole one, so the tau of the row's granule maxima (the largest z of each 64
// keys, which the score pass keeps) is at most tau, and close to it, since a
// long row's support lies in as many granules.  Only granules whose maximum
// is above that bound are looked at again: their keys above it are listed
// (index, z) in LDS, Newton steps over the list find tau, and only the value
// rows of the support are read.  alpha-entmax gives most keys of a long row
// no weight, so the values' bytes are a small part of the keys'.  Lists have
// a fixed order, so results do not depend on timing.
#include <climits>
#include <type_traits>

#include "asa_cache.hpp"
#include "asa_device.hpp"

namespace asa {
namespace {

constexpr float kHidden = -3e38f;     // dot and z of a key that a row does not see
constexpr float kNotNumber = -1e38f;  // a dot that is not a number: the score clamp makes it -10
constexpr int kTile = 16;          // rows and keys of an MFMA tile

// ---------------------------------------------------------------------------
// Scores
// ---------------------------------------------------------------------------

// The visible keys of query token i of sequence b are the first of them.
__device__ __forceinline__ int visible_keys(const CacheAttnParams& p, int b, int i) {
  const int len = max(0, min(p.lengths[b], p.maxlen));
  const int at = p.q_idx ? p.q_idx[size_t(b) * p.NQ + i] : len - p.NQ + i;
  return at < 0 ? 0 : at >= len ? len : at + 1;
}

// The 16-bit format of the codes operand: fp16 for fp16 queries, else bf16.
template <typename T> using CodeType = typename std::conditional<std::is_same<T, h16>::value, h16, u16>::type;
template <typename T> using CodeVec = typename Half<CodeType<T>>::v8;

// 8 codes as 16 + c: channels 0 4 1 5 2 6 3 7, since nibbles j and j + 4 are
// 16 bits apart.  The query operand has the same order.
__device__ __forceinline__ int operand_slot(int j) { return j < 4 ? 2 * j : 2 * j - 7; }
template <typename T> __device__ __forceinline__ CodeVec<T> codes_operand(uint32_t w) {
  uint32_t u[4];
  if constexpr (std::is_same<T, h16>::value) {  // 16.0 = 0x4c00, one = 1 << 6
    const uint32_t mask = 0x03c003c0u, one = 0x4c004c00u;
    u[0] = ((w << 6) & mask) | one;
    u[1] = ((w << 2) & mask) | one;
    u[2] = ((w >> 2) & mask) | one;
    u[3] = ((w >> 6) & mask) | one;
  } else {  // 16.0 = 0x4180, one = 1 << 3
    const uint32_t mask = 0x00780078u, one = 0x41804180u;
    u[0] = ((w << 3) & mask) | one;
    u[1] = ((w >> 1) & mask) | one;
    u[2] = ((w >> 5) & mask) | one;
    u[3] = ((w >> 9) & mask) | one;
  }
  CodeVec<T> r;
  __builtin_memcpy(&r, u, 16);
  return r;
}

// One wave's query operand: rows r0 .. of a key head's R rows (row r: query
// head h * rep + r / NQ, token r % NQ), kR of them, for each of the P key
// tiles that share a result, and the accumulators' starts.  Queries of a
// negative scale are negated, so that larger products are larger scores.
template <typename T, int P, int NG>
struct QueryFrag {
  static constexpr int kR = kTile / P;
  static constexpr int NT = std::is_same<T, float>::value ? 3 : 1;
  CodeVec<T> a[P][NG][NT];
  f32x4 bias[NG];  // -16 sum q_g of rows (4 (lane / 16) + k) % kR
  int vis[4];      // visible keys of those rows
  int most, least; // over the real rows of the tile

  __device__ __forceinline__ void load(const CacheAttnParams& p, int b, int h, int r0, int lane) {
    using S = typename Half<CodeType<T>>::scalar;
    const int o = lane >> 4, ar = lane & 15, r = r0 + ar % kR;
    const bool ok = r < p.R;
    const int rr = ok ? r : 0, head = h * p.rep + rr / p.NQ, i = rr % p.NQ;
    const T* q = static_cast<const T*>(p.q) + size_t(b) * p.lq.sb + size_t(head) * p.lq.sh + size_t(i) * p.lq.sn;
    const float sign = p.scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const int ch = 32 * g + 8 * o, nv = ok ? p.c.hd - ch : 0;
      float x[8];
      if (p.chunks) {
        constexpr int kEpc = 16 / int(sizeof(T));
        T e[8] = {};
        if (nv > 0)
          for (int c = 0; c < 8; c += kEpc) {
            const uint4 u = *reinterpret_cast<const uint4*>(q + ch + c);
            __builtin_memcpy(e + c, &u, 16);
          }
        for (int j = 0; j < 8; ++j) x[j] = Elem<T>::load(e + j);
      } else {
        for (int j = 0; j < 8; ++j) x[j] = j < nv ? Elem<T>::load(q + ch + j) : 0.0f;
      }
      for (int j = 0; j < 8; ++j) x[j] *= sign;
      const float sum = sum_groups(((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7])));
      for (int k = 0; k < 4; ++k) bias[g][k] = -16.0f * __shfl(sum, 4 * o + k, 64);
#pragma unroll
      for (int t = 0; t < NT; ++t)
        for (int j = 0; j < 8; ++j) {
          const S y = static_cast<S>(x[j]);
          x[j] -= static_cast<float>(y);
          for (int u = 0; u < P; ++u) a[u][g][t][operand_slot(j)] = ar / kR == u ? y : static_cast<S>(0.0f);
        }
    }
    int hi = 0, lo = INT_MAX;
    for (int k = 0; k < 4; ++k) {
      const int row = r0 + (4 * o + k) % kR;
      vis[k] = row < p.R ? visible_keys(p, b, row % p.NQ) : 0;
      hi = max(hi, vis[k]);
      lo = row < p.R ? min(lo, vis[k]) : lo;
    }
    most = wave_reduce_minmax<true>(hi);
    least = wave_reduce_minmax<false>(lo);
  }
};

// P tiles of 16 keys: the codes (key order: lane group o has octet o of every
// channel group) of key lane % 16 of each tile, and the params of the lane's
// own key of the result.
template <int P, int NG>
struct KeyPack {
  uint32_t w[P][NG], pr[NG];
  bool seen;  // the lane's own key has a page

  template <int N> static __device__ __forceinline__ void words(uint32_t* d, const uint32_t* s) {
    __builtin_memcpy(d, __builtin_assume_aligned(s, N == 4 ? 16 : N == 2 ? 8 : 4), 4 * N);
  }
  // keys base .. base + 16 P - 1 of [.., key1); pages: of the keys from key0
  __device__ __forceinline__ void load(const CachePool& c, int h, const int* pages, int key0, int base, int key1,
                                       int lane) {
    const int o = lane >> 4, col = lane & 15;
#pragma unroll
    for (int u = 0; u < P; ++u) {
      const int key = base + kTile * u;
      const int pg = key < key1 ? __builtin_amdgcn_readfirstlane(pages[(key - key0) >> c.page_shift]) : -1;
      if (pg >= 0) {
        const int64_t row = (int64_t(pg) * c.heads + h) * c.page + (key & (c.page - 1)) + col;
        words<NG>(w[u], reinterpret_cast<const uint32_t*>(c.k_codes) + row * (4 * NG) + NG * o);
      } else {
        for (int g = 0; g < NG; ++g) w[u][g] = 0u;
      }
    }
    const int key = base + kTile * (o * P / 4);
    const int pg = key < key1 ? pages[(key - key0) >> c.page_shift] : -1;
    seen = pg >= 0;
    for (int g = 0; g < NG; ++g) pr[g] = 0u;
    if (seen) words<NG>(pr, c.k_params + ((int64_t(pg) * c.heads + h) * c.page + (key & (c.page - 1)) + col) * NG);
  }
};

// q.k: element k of a lane is row (4 (lane / 16) + k) % kR, key
// 16 (lane / 16 * P / 4) + lane % 16 of the pack.
template <typename T, int P, int NG>
__device__ __forceinline__ f32x4 dots(const QueryFrag<T, P, NG>& q, const KeyPack<P, NG>& k) {
  f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    f32x4 acc = q.bias[g];
#pragma unroll
    for (int u = 0; u < P; ++u) {
      const CodeVec<T> c = codes_operand<T>(k.w[u][g]);
#pragma unroll
      for (int t = 0; t < QueryFrag<T, P, NG>::NT; ++t) acc = mfma(q.a[u][g][t], c, acc);
    }
    const float sc = __uint_as_float(k.pr[g] << 16);
    const float off = __uint_as_float(k.pr[g] & 0xffff0000u) * -0.0625f;  // m sum q_g = -m / 16 bias
    for (int r = 0; r < 4; ++r) s[r] = fmaf(off, q.bias[g][r], fmaf(sc, acc[r], s[r]));
  }
  return s;
}

// z = (alpha - 1) clamp(|scale| dot), hidden keys apart.
struct ZOf {
  float c, zb;
  __device__ __forceinline__ explicit ZOf(const CacheAttnParams& p) : c(p.zc), zb(p.zb) {}
  __device__ __forceinline__ float operator()(float dot) const {
    return dot <= 2.0f * kNotNumber ? kHidden : __builtin_amdgcn_fmed3f(dot * c, -zb, zb);
  }
};

// Pages of the keys [key0, key0 + n) into LDS (-1: none that the pool has).
__device__ __forceinline__ void stage_pages(const CacheAttnParams& p, int b, int key0, int n,
                                            int* pages, int t, int threads) {
  const int first = key0 >> p.c.page_shift, cnt = (n + p.c.page - 1) >> p.c.page_shift;
  for (int e = t; e < cnt; e += threads) {
    const int col = first + e;
    const int pg = col < p.cols ? p.table[size_t(b) * p.cols + col] : -1;
    pages[e] = pg >= 0 && pg < p.c.pages ? pg : -1;
  }
}

// Dots of the keys [key0, key1) by the block's NW waves, a granule of 64 keys
// per wave and step (4 / P packs; the next step's loads are in flight
// meanwhile), handed to put(key, dots) (dots as from `dots`; hidden where a
// row does not see the key); the granule's maxima of each row to
// most(granule, row of the tile, maximum) by one lane.  key0 is a multiple of
// the page size and of 64.
constexpr int kGranule = 64;
template <int NW, typename T, int P, int NG, typename Put, typename Most>
__device__ __forceinline__ void score_keys(const CacheAttnParams& p, const QueryFrag<T, P, NG>& q, int h,
                                           int key0, int key1, const int* pages, int w, int lane,
                                           Put put, Most most) {
  constexpr int V = 4 / P, kKeys = kTile * P, kR = kTile / P;
  const int own = kTile * ((lane >> 4) * P / 4) + (lane & 15);
  KeyPack<P, NG> next[V];
  int base = key0 + w * kGranule;
  if (base < key1)
#pragma unroll
    for (int v = 0; v < V; ++v) next[v].load(p.c, h, pages, key0, base + v * kKeys, key1, lane);
  for (; base < key1; base += NW * kGranule) {
    KeyPack<P, NG> k[V];
#pragma unroll
    for (int v = 0; v < V; ++v) k[v] = next[v];
    const int ahead = base + NW * kGranule;
    if (ahead < key1)
#pragma unroll
      for (int v = 0; v < V; ++v) next[v].load(p.c, h, pages, key0, ahead + v * kKeys, key1, lane);
    f32x4 m = {kHidden, kHidden, kHidden, kHidden};
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int first = base + v * kKeys, key = first + own;
      if (first < key1) {
        f32x4 d = dots<T, P, NG>(q, k[v]);
        for (int r = 0; r < 4; ++r) d[r] = fmaxf(d[r], kNotNumber);
        if (first + kKeys > q.least)
          for (int r = 0; r < 4; ++r) d[r] = key < q.vis[r] ? d[r] : kHidden;
        for (int r = 0; r < 4; ++r) d[r] = k[v].seen ? d[r] : kHidden;
        put(key, d);
        for (int r = 0; r < 4; ++r) m[r] = fmaxf(m[r], d[r]);
      }
    }
    for (int r = 0; r < 4; ++r) {
      float x = m[r];
      x = fmaxf(x, __uint_as_float(lane_xor<1>(__float_as_uint(x))));
      x = fmaxf(x, __uint_as_float(lane_xor<2>(__float_as_uint(x))));
      x = fmaxf(x, __uint_as_float(lane_xor<7>(__float_as_uint(x))));
      x = fmaxf(x, __uint_as_float(lane_xor<15>(__float_as_uint(x))));
      if constexpr (P >= 2) {
        const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
      }
      if constexpr (P == 4) {
        const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
      }
      const int row = 4 * (lane >> 4) + r;
      if ((lane & 15) == 0 && row < kR) most(base / kGranule, row, x);
    }
  }
}

// ---------------------------------------------------------------------------
// Threshold and values of one row by a team of waves
// ---------------------------------------------------------------------------

template <typename F> __device__ __forceinline__ float wave_reduce(float v, F op) {
  v = op(v, __uint_as_float(lane_xor<1>(__float_as_uint(v))));
  v = op(v, __uint_as_float(lane_xor<2>(__float_as_uint(v))));
  v = op(v, __uint_as_float(lane_xor<7>(__float_as_uint(v))));
  v = op(v, __uint_as_float(lane_xor<15>(__float_as_uint(v))));
  return __uint_as_float(group_reduce_bits(__float_as_uint(v), [op](uint32_t x, uint32_t y) {
    return __float_as_uint(op(__uint_as_float(x), __uint_as_float(y)));
  }));
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_reduce(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v) {
  return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}
// v^e and v^(e-1), v >= 0, both 0 at v = 0.
__device__ __forceinline__ void powers(int pc, float v, float e, float& pa, float& pa1) {
  if (pc == kE2) {
    pa = v * v, pa1 = v;
  } else if (pc == kE1) {
    pa = v, pa1 = v > 0.0f ? 1.0f : 0.0f;
  } else if (pc == kE4) {
    const float v2 = v * v;
    pa1 = v2 * v, pa = v2 * v2;
  } else {
    const float l = __builtin_amdgcn_logf(v);
    pa = v > 0.0f ? __builtin_amdgcn_exp2f(e * l) : 0.0f;
    pa1 = v > 0.0f ? __builtin_amdgcn_exp2f((e - 1.0f) * l) : 0.0f;
  }
}

// The next tau from tau, where F = sum v^e and F1 = sum v^(e-1) over the
// keys with v = z - tau > 0; true when tau is final.  For alpha <= 2 (e >= 1)
// the step is Newton's on the norm F^(1/e) - 1: the norm is convex in tau and
// nearly straight, so the steps from the left end stay left of the root and
// few are needed.  For alpha > 2 a key just above tau makes F1 unbounded, and
// the bracket is halved instead.
__device__ __forceinline__ bool next_tau(float alpha, float F, float F1, float& tau, float& lo, float& hi) {
  const float f = F - 1.0f;
  if (f >= 0.0f) lo = tau;
  else hi = tau;
  float nt = 0.5f * (lo + hi);
  if (alpha <= 2.0f) {
    const float s = tau + (F - __builtin_amdgcn_exp2f((2.0f - alpha) * __builtin_amdgcn_logf(F))) / F1;
    if (s >= lo && s <= hi) nt = s;
  }
  const bool done = nt == tau || nt == lo || fabsf(f) <= (alpha <= 2.0f ? 1e-6f : 1e-7f);
  if (alpha <= 2.0f || !done) tau = nt;
  return done;
}
constexpr int kMaxSteps = 64;

// LDS of the row teams.  A wave collects up to CAP candidates of its row; a
// list of up to kList is gathered for the whole team (8 registers of a wave).
constexpr int kList = 512;
constexpr int kAccStride = 132;
template <int NW, int CAP> struct TeamLds {
  static constexpr int kCap = CAP;
  float cz[NW][CAP];  // a wave's candidates, later its part of the support
  int ci[NW][CAP];
  float gm[NW][kWave];
  float red[2][NW][2];
  float psum[NW];
  int cnt[NW];
  float acc[NW][kAccStride];
};

// Adds p_j v_j of the wave's listed keys to the lane's 8 channels: CL lanes
// have a row's octets, so a step takes 64 / CL entries, four loads deep.
template <int NG>
struct ValueSum {
  static constexpr int kCl = NG == 3 ? 16 : 4 * NG, kPer = kWave / kCl;
  float acc[8] = {};
  float off = 0.0f;
  __device__ __forceinline__ void add(const CacheAttnParams& p, int b, int h, const float* pz, const int* pi,
                                      int n, int lane) {
    const int c = lane & (kCl - 1), slot = lane / kCl, g = c >> 2;
    const int32_t* table = p.table + size_t(b) * p.cols;
    for (int e0 = 0; e0 < n; e0 += 4 * kPer) {
      uint32_t w[4], pr[4];
      float pj[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int e = e0 + u * kPer + slot;
        w[u] = pr[u] = 0u;
        pj[u] = 0.0f;
        if (e < n && g < NG) {
          const int64_t row = cache_row(p.c, table, p.cols, pi[e], h);
          if (row >= 0) {
            pj[u] = pz[e];
            w[u] = reinterpret_cast<const uint32_t*>(p.c.v_codes)[row * (4 * NG) + c];
            pr[u] = p.c.v_params[row * NG + g];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float ps = pj[u] * __uint_as_float(pr[u] << 16);
        off = fmaf(pj[u], __uint_as_float(pr[u] & 0xffff0000u), off);
        const uint32_t even = w[u] & 0x0f0f0f0fu, odd = (w[u] >> 4) & 0x0f0f0f0fu;
        for (int j = 0; j < 4; ++j) {
          acc[2 * j] = fmaf(ps, float((even >> (8 * j)) & 255u), acc[2 * j]);
          acc[2 * j + 1] = fmaf(ps, float((odd >> (8 * j)) & 255u), acc[2 * j + 1]);
        }
      }
    }
  }
  // the wave's sums of channels 8 c + j, in every lane with that c
  __device__ __forceinline__ void reduce() {
    for (int j = 0; j < 8; ++j) {
      acc[j] += off;
      if constexpr (kCl <= 4) acc[j] += __uint_as_float(lane_xor<4>(__float_as_uint(acc[j])));
      if constexpr (kCl <= 8) acc[j] += __uint_as_float(lane_xor<8>(__float_as_uint(acc[j])));
      acc[j] = sum_groups(acc[j]);
    }
  }
};

// tau and the output of row `row` (of the key head's R) from its dots at
// sp[0 .. vis) and their granule maxima gp, by `size` waves of the block from
// wave w0 on; lz, li: kList entries of (z, key) of the team.  Every wave of
// the block calls it together (teams meet at the block's barriers); row = -1,
// vis = 0 for a team without a row.  WHOLE: the team is the block.
template <typename T, int NG, int NW, bool WHOLE, typename Lds>
__device__ __forceinline__ void finish_row(const CacheAttnParams& p, int b, int h, int row, int vis,
                                           const float* gp, const float* sp, Lds& L, float* lz, int* li, int w,
                                           int w0, int size, int lane) {
  constexpr int kCap = Lds::kCap;
  const int member = w - w0, pc = p.pc;
  const float e = p.e;
  const ZOf zof(p);

  // ---- the largest z, and a bound below tau from the granules' ----
  const int ng = (vis + kGranule - 1) / kGranule;
  float g = kHidden;
#pragma unroll 4
  for (int j = member * kWave + lane; j < ng; j += size * kWave) g = fmaxf(g, gp[j]);
  L.gm[w][lane] = zof(g);
  __syncthreads();
  float gz[4] = {kHidden, kHidden, kHidden, kHidden};
  for (int i = 0; i < size; i += 4)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < size) gz[k] = fmaxf(gz[k], L.gm[w0 + i + k][lane]);
  const float zmax = wave_max(fmaxf(fmaxf(gz[0], gz[1]), fmaxf(gz[2], gz[3])));
  const bool empty = !(zmax > 0.5f * kHidden);
  float tau = zmax - 1.0f, lo = tau, hi = zmax;
  if (vis > kList && !empty) {
    // a few steps: any tau left of the root of the maxima will do
    for (int it = 0; it < 12; ++it) {
      float F = 0.0f, F1 = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float pa, pa1;
        powers(pc, fmaxf(gz[k] - tau, 0.0f), e, pa, pa1);
        F += pa;
        F1 += pa1;
      }
      F = wave_sum(F);
      if (F < 1.01f && p.alpha <= 2.0f) break;
      if (next_tau(p.alpha, F, wave_sum(F1), tau, lo, hi)) break;
    }
    // the rounding of the steps, and of F at them
    if (p.alpha <= 2.0f) lo = tau;
    lo = fmaxf(lo - 4e-6f, zmax - 1.0f);
    tau = lo;
    hi = zmax;
  }

  // ---- the keys with z > lo, listed; lo moves up while they do not fit ----
  bool listed = false, big = false, dense = empty;
  int n = 0, mine = 0;
  for (int it = 0;; ++it) {
    if (!listed && !dense) {
      mine = 0;
      auto collect = [&](float d, int key) {
        const float z = key < vis ? zof(d) : kHidden;
        const uint64_t m = __ballot(z > lo);
        const int at = mine + lane_rank(m);
        if (z > lo && at < kCap) {
          L.cz[w][at] = z;
          L.ci[w][at] = key;
        }
        mine += __builtin_popcountll(m);
      };
      // granule i is member i % size's
      for (int i0 = 0; i0 < ng; i0 += size * kWave) {
        const int i = i0 + lane * size + member;
        uint64_t todo = __ballot(i < ng && zof(gp[i < ng ? i : 0]) > lo);
        while (todo) {
          float d[4];
          int key[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int l = todo ? __builtin_ctzll(todo) : -1;
            todo &= todo - 1;
            key[k] = l < 0 ? vis : (i0 + l * size + member) * kGranule + lane;
            d[k] = sp[key[k] < vis ? key[k] : 0];
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) collect(d[k], key[k]);
        }
      }
      if (lane == 0) L.cnt[w] = mine;
    }
    __syncthreads();
    if (!listed && !dense) {
      n = 0;
      int before = 0;
      bool fits = true;
      for (int i = 0; i < size; ++i) {
        const int c = L.cnt[w0 + i];
        if (i == member) before = n;
        n += c;
        fits = fits && c <= kCap;
      }
      listed = fits && (WHOLE || n <= kList);
      big = listed && n > kList;
      if (listed && !big)
        for (int j = lane; j < mine; j += kWave) {
          lz[before + j] = L.cz[w][j];
          li[before + j] = L.ci[w][j];
        }
    }
    if (!__syncthreads_or(!listed && !dense)) break;
    // some team's candidates did not fit: one step of its tau over the whole row
    float F = 0.0f, F1 = 0.0f;
    if (!listed && !dense) {
#pragma unroll 4
      for (int j = member * kWave + lane; j < vis; j += size * kWave) {
        float pa, pa1;
        powers(pc, fmaxf(zof(sp[j]) - tau, 0.0f), e, pa, pa1);
        F += pa;
        F1 += pa1;
      }
      F = wave_sum(F);
      F1 = wave_sum(F1);
      if (lane == 0) {
        L.red[0][w][0] = F;
        L.red[0][w][1] = F1;
      }
    }
    __syncthreads();
    if (!listed && !dense) {
      F = F1 = 0.0f;
      for (int i = 0; i < size; ++i) {
        F += L.red[0][w0 + i][0];
        F1 += L.red[0][w0 + i][1];
      }
      dense = next_tau(p.alpha, F, F1, tau, lo, hi) || it == kMaxSteps;
      if (p.alpha <= 2.0f) lo = tau;  // the steps stay left of the root
    }
  }

  // ---- tau over the list ----
  float total = 0.0f;
  if (listed) {
    tau = lo;
    bool done = false;
    if (!big) {  // in registers, by every wave alike
      constexpr int kRegs = kList / kWave;
      float z[kRegs];
#pragma unroll
      for (int k = 0; k < kRegs; ++k) z[k] = k * kWave + lane < n ? lz[k * kWave + lane] : kHidden;
      for (int it = 0; it <= kMaxSteps; ++it) {
        float F = 0.0f, F1 = 0.0f;
#pragma unroll
        for (int k = 0; k < kRegs; ++k)
          if (k * kWave < n) {
            float pa, pa1;
            powers(pc, fmaxf(z[k] - tau, 0.0f), e, pa, pa1);
            F += pa;
            F1 += pa1;
          }
        total = wave_sum(F);
        if (done || it == kMaxSteps) break;  // the sum at the final tau
        done = next_tau(p.alpha, total, wave_sum(F1), tau, lo, hi);
      }
    } else {  // each wave its candidates; the block's barriers are the team's
      for (int it = 0; it <= kMaxSteps; ++it) {
        float F = 0.0f, F1 = 0.0f;
#pragma unroll 2
        for (int j = lane; j < mine; j += kWave) {
          float pa, pa1;
          powers(pc, fmaxf(L.cz[w][j] - tau, 0.0f), e, pa, pa1);
          F += pa;
          F1 += pa1;
        }
        F = wave_sum(F);
        F1 = wave_sum(F1);
        if (lane == 0) {
          L.red[it & 1][w][0] = F;
          L.red[it & 1][w][1] = F1;
        }
        __syncthreads();
        total = F1 = 0.0f;
        for (int i = 0; i < size; ++i) {
          total += L.red[it & 1][i][0];
          F1 += L.red[it & 1][i][1];
        }
        if (done || it == kMaxSteps) break;
        done = next_tau(p.alpha, total, F1, tau, lo, hi);
      }
    }
  }

  // ---- the support's weights and values ----
  ValueSum<NG> vs;
  float psum = 0.0f;
  if (!empty) {
    // the wave's part of the list, or its candidates, or its keys of the
    // row, kCap at a time
    const bool small = listed && !big;
    const int part = small ? (n + size - 1) / size : big ? mine : kCap;
    const int end = small ? min(n, (member + 1) * part) : big ? mine : vis;
    for (int k0 = big ? 0 : member * part; k0 < end; k0 += size * part) {
      const int cnt = min(part, end - k0);
      int c = 0;
      for (int j0 = 0; j0 < cnt; j0 += kWave) {
        const int j = j0 + lane;
        float zj = kHidden;
        int key = 0;
        if (j < cnt) {
          zj = small ? lz[k0 + j] : big ? L.cz[w][j] : zof(sp[k0 + j]);
          key = small ? li[k0 + j] : big ? L.ci[w][j] : k0 + j;
        }
        float pa, pa1;
        powers(pc, fmaxf(zj - tau, 0.0f), e, pa, pa1);
        const uint64_t msk = __ballot(pa > 0.0f);
        if (pa > 0.0f) {
          const int at = c + lane_rank(msk);  // at most j: already read
          L.cz[w][at] = pa;
          L.ci[w][at] = key;
        }
        c += __builtin_popcountll(msk);
        psum += pa;
      }
      vs.add(p, b, h, L.cz[w], L.ci[w], c, lane);
    }
  }
  vs.reduce();
  if (lane < ValueSum<NG>::kCl && lane < 4 * NG)
    for (int j = 0; j < 8; ++j) L.acc[w][8 * lane + j] = vs.acc[j];
  if (!listed) {
    psum = wave_sum(psum);
    if (lane == 0) L.psum[w] = psum;
  }
  __syncthreads();
  if (row >= 0) {
    if (!listed)
      for (int i = 0; i < size; ++i) total += L.psum[w0 + i];
    const float inv = total > 0.0f ? 1.0f / total : 0.0f;
    const int head = h * p.rep + row / p.NQ, i = row % p.NQ;
    T* out = static_cast<T*>(p.out) + ((size_t(b) * p.H + head) * p.NQ + i) * p.c.hd;
    for (int ch = member * kWave + lane; ch < p.c.hd; ch += size * kWave) {
      float v = 0.0f;
      for (int k = 0; k < size; ++k) v += L.acc[w0 + k][ch];
      Elem<T>::store(out + ch, v * inv);
    }
  }
}

// ---------------------------------------------------------------------------
// Kernels
// ---------------------------------------------------------------------------

constexpr int kOneWaves = 8;    // one-block plan
constexpr int kScoreWaves = 4;  // split plan: score blocks
constexpr int kRowKeys = 8192;  // split plan: rows up to this have 4 waves, else 16

// One block per tile of rows of a key head: dots into LDS, then its rows.
using OneLds = TeamLds<kOneWaves, 128>;
template <typename T, int P, int NG>
__global__ __launch_bounds__(kOneWaves * kWave) void cache_one_kernel(CacheAttnParams p, int stride) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ OneLds L;
  constexpr int kR = kTile / P;
  const int t = threadIdx.x, w = t >> 6, lane = t & 63, o = lane >> 4;
  const int nrt = (p.R + kR - 1) / kR;
  const int rt = blockIdx.x % nrt, bh = blockIdx.x / nrt;
  const int b = bh / p.c.heads, h = bh % p.c.heads;
  const int r0 = rt * kR, rows = min(kR, p.R - r0), most = min(kR, p.R), gs = stride / kGranule;
  int pad = 1;
  while (pad < most && pad < kOneWaves) pad *= 2;
  float* zs = reinterpret_cast<float*>(smem);
  float* gs0 = zs + most * stride;  // granule maxima
  float* lz = gs0 + most * gs;      // a list for each of `pad` teams
  int* li = reinterpret_cast<int*>(lz + pad * kList);
  int* pages = li + pad * kList;
  stage_pages(p, b, 0, p.maxlen, pages, t, kOneWaves * kWave);
  const int len = max(0, min(p.lengths[b], p.maxlen));
  {
    QueryFrag<T, P, NG> q;
    q.load(p, b, h, r0, lane);
    __syncthreads();
    score_keys<kOneWaves>(
        p, q, h, 0, min(len, q.most), pages, w, lane,
        [&](int key, f32x4 d) {
          for (int k = 0; k < 4; ++k) {
            const int r = (4 * o + k) % kR;
            if (r < rows) zs[r * stride + key] = d[k];
          }
        },
        [&](int granule, int r, float m) {
          if (r < rows) gs0[r * gs + granule] = m;
        });
  }
  __syncthreads();
  const int size = kOneWaves / pad, team = w / size, w0 = team * size;
  for (int first = 0; first < rows; first += pad) {
    const int r = first + team;
    const bool has = r < rows;
    finish_row<T, NG, kOneWaves, false>(p, b, h, has ? r0 + r : -1, has ? visible_keys(p, b, (r0 + r) % p.NQ) : 0,
                                        gs0 + (has ? r : 0) * gs, zs + (has ? r : 0) * stride, L, lz + team * kList,
                                        li + team * kList, w, w0, size, lane);
  }
}

// Split plan, first launch: dots of `span` keys with a tile of rows, and
// their granules' maxima.
template <typename T, int P, int NG>
__global__ __launch_bounds__(kScoreWaves * kWave) void cache_score_kernel(CacheAttnParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  constexpr int kR = kTile / P;
  int* pages = reinterpret_cast<int*>(smem);
  const int t = threadIdx.x, w = t >> 6, lane = t & 63, o = lane >> 4;
  const int nrt = (p.R + kR - 1) / kR;
  const int split = blockIdx.x % p.nsplit, rest = blockIdx.x / p.nsplit;
  const int rt = rest % nrt, bh = rest / nrt;
  const int b = bh / p.c.heads, h = bh % p.c.heads;
  const int r0 = rt * kR;
  const int key0 = split * p.span;
  const int len = max(0, min(p.lengths[b], p.maxlen));
  if (key0 >= len) return;
  const int key1 = min(len, key0 + p.span);
  stage_pages(p, b, key0, key1 - key0, pages, t, kScoreWaves * kWave);
  QueryFrag<T, P, NG> q;
  q.load(p, b, h, r0, lane);
  __syncthreads();
  const size_t stride = size_t(p.span) * p.nsplit, gs = stride / kGranule, row0 = size_t(bh) * p.R + r0;
  float* base = p.scores + row0 * stride;
  float* gbase = p.gmax + row0 * gs;
  score_keys<kScoreWaves>(
      p, q, h, key0, min(key1, q.most), pages, w, lane,
      [&](int key, f32x4 d) {
        for (int k = 0; k < 4; ++k) {
          const int r = (4 * o + k) % kR;
          if (key < key1 && r0 + r < p.R) base[size_t(r) * stride + key] = d[k];
        }
      },
      [&](int granule, int r, float m) {
        if (r0 + r < p.R) gbase[size_t(r) * gs + granule] = m;
      });
}

// Split plan, second launch: one block per row.
template <typename T, int NG, int NW>
__global__ __launch_bounds__(NW * kWave) void cache_row_kernel(CacheAttnParams p) {
  __shared__ TeamLds<NW, NW == 16 ? 256 : 512> L;
  __shared__ float lz[kList];
  __shared__ int li[kList];
  const int t = threadIdx.x, w = t >> 6, lane = t & 63;
  const int row = blockIdx.x % p.R, bh = blockIdx.x / p.R;
  const int b = bh / p.c.heads, h = bh % p.c.heads;
  const size_t at = size_t(bh) * p.R + row, stride = size_t(p.span) * p.nsplit;
  finish_row<T, NG, NW, true>(p, b, h, row, visible_keys(p, b, row % p.NQ), p.gmax + at * (stride / kGranule),
                              p.scores + at * stride, L, lz, li, w, 0, NW, lane);
}

template <typename K> hipError_t allow_lds(K kern, size_t lds) {
  if (lds <= 65536) return hipSuccess;
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                             int(lds));
}

// Key tiles that share a result: as many as leave room for the rows.  fp32
// queries (three terms) would need P times their 48 operand registers.
int tiles_shared(const CacheAttnParams& p, int dtype) {
  return dtype == kElemF32 || p.R > 8 ? 1 : p.R > 4 ? 2 : 4;
}

size_t one_lds_bytes(const CacheAttnParams& p, int tile_rows, int* stride) {
  const int rows = p.R < tile_rows ? p.R : tile_rows;
  *stride = (p.maxlen + kGranule - 1) / kGranule * kGranule;
  int pad = 1;
  while (pad < rows && pad < kOneWaves) pad *= 2;
  return size_t(rows) * (*stride + *stride / kGranule) * 4 + size_t(pad) * kList * 8 +
         size_t((p.maxlen + p.c.page - 1) / p.c.page + 1) * 4;
}

template <typename T, int P, int NG>
hipError_t launch_png(const CacheAttnParams& p, hipStream_t s) {
  const int nrt = (p.R + kTile / P - 1) / (kTile / P);
  if (p.plan == kCacheOneBlock) {
    int stride = 0;
    const size_t lds = one_lds_bytes(p, kTile / P, &stride);
    auto kern = cache_one_kernel<T, P, NG>;
    if (hipError_t e = allow_lds(kern, lds)) return e;
    profile_begin("cache_attn", s);
    hipLaunchKernelGGL(kern, dim3(unsigned(p.B) * p.c.heads * nrt), dim3(kOneWaves * kWave), lds, s, p, stride);
    profile_end(s);
    return hipGetLastError();
  }
  profile_begin("cache_score", s);
  hipLaunchKernelGGL((cache_score_kernel<T, P, NG>), dim3(unsigned(p.B) * p.c.heads * nrt * p.nsplit),
                     dim3(kScoreWaves * kWave), size_t(p.span / p.c.page + 1) * 4, s, p);
  profile_end(s);
  return hipGetLastError();
}

template <typename T, int NG>
hipError_t launch_ng(const CacheAttnParams& p, int dtype, hipStream_t s) {
  hipError_t e = hipSuccess;
  if constexpr (std::is_same<T, float>::value) {
    e = launch_png<T, 1, NG>(p, s);
  } else {
    const int P = tiles_shared(p, dtype);
    e = P == 1 ? launch_png<T, 1, NG>(p, s) : P == 2 ? launch_png<T, 2, NG>(p, s) : launch_png<T, 4, NG>(p, s);
  }
  if (e != hipSuccess || p.plan == kCacheOneBlock) return e;
  const dim3 grid(unsigned(p.B) * p.c.heads * p.R);
  profile_begin("cache_row", s);
  if (p.maxlen <= kRowKeys) hipLaunchKernelGGL((cache_row_kernel<T, NG, 4>), grid, dim3(4 * kWave), 0, s, p);
  else hipLaunchKernelGGL((cache_row_kernel<T, NG, 16>), grid, dim3(16 * kWave), 0, s, p);
  profile_end(s);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_t(const CacheAttnParams& p, int dtype, hipStream_t s) {
  switch (p.c.G) {
    case 1: return launch_ng<T, 1>(p, dtype, s);
    case 2: return launch_ng<T, 2>(p, dtype, s);
    case 3: return launch_ng<T, 3>(p, dtype, s);
    default: return launch_ng<T, 4>(p, dtype, s);
  }
}

}  // namespace

size_t cache_attn_plan(CacheAttnParams& p, int dtype, size_t max_lds, int cus) {
  const int tile_rows = kTile / tiles_shared(p, dtype);
  int stride = 0;
  p.span = p.nsplit = 0;
  if (p.maxlen <= 2048 &&
      one_lds_bytes(p, tile_rows, &stride) + sizeof(OneLds) <= max_lds) {
    p.plan = kCacheOneBlock;
    return 0;
  }
  p.plan = kCacheSplit;
  const long long nrt = (p.R + tile_rows - 1) / tile_rows, tiles = (long long)p.B * p.c.heads * nrt;
  // eight score blocks per compute unit, of at least 256 keys (the largest
  // page: a block starts on a page)
  long long span = (p.maxlen * tiles + 8LL * cus - 1) / (8LL * cus);
  span = (span + 255) / 256 * 256;
  if (span > 4096) span = 4096;
  p.span = int(span);
  p.nsplit = int((p.maxlen + span - 1) / span);
  return size_t(p.B) * p.c.heads * p.R * p.nsplit * (size_t(p.span) + p.span / kGranule) * sizeof(float);
}

hipError_t launch_cache_attn(const CacheAttnParams& call, int dtype, hipStream_t s) {
  CacheAttnParams p = call;
  p.e = 1.0f / (p.alpha - 1.0f);
  p.pc = pow_class_of(p.e);
  p.zc = (p.alpha - 1.0f) * (p.scale < 0.0f ? -p.scale : p.scale);
  p.zb = 10.0f * (p.alpha - 1.0f);
  if (dtype == kElemBF16) return launch_t<u16>(p, dtype, s);
  if (dtype == kElemF16) return launch_t<h16>(p, dtype, s);
  return launch_t<float>(p, dtype, s);
}

}  // namespace asa
