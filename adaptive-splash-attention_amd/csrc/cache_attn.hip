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
// weight: they are listed (index, z) in LDS, Newton steps over the list find
// tau, and only the value rows of the support are read, by their entry in
// the list.  alpha-entmax gives most keys of a long row no weight, so the
// values' bytes are a small part of the keys'.
#include <climits>

#include "asa_cache.hpp"
#include "asa_device.hpp"

namespace asa {
namespace {

constexpr float kHidden = -3e38f;  // z of a key that a row does not see
constexpr int kRows = 16;          // query rows of an MFMA tile
constexpr int kSub = 16;           // keys of an MFMA tile

// ---------------------------------------------------------------------------
// Scores
// ---------------------------------------------------------------------------

// The visible keys of query token i of sequence b are the first of them.
__device__ __forceinline__ int visible_keys(const CacheAttnParams& p, int b, int i) {
  const int len = max(0, min(p.lengths[b], p.maxlen));
  const int at = p.q_idx ? p.q_idx[size_t(b) * p.NQ + i] : len - p.NQ + i;
  return at < 0 ? 0 : at >= len ? len : at + 1;
}

// One wave's query operand: rows r0 .. r0 + 15 of a key head's R rows (row
// r: query head h * rep + r / NQ, token r % NQ) as NT bf16 terms per group,
// the accumulators' starts, and the offsets' operand.
template <typename T, int NT, int NG>
struct QueryFrag {
  bf16x8 a[NG][NT];
  f32x4 bias[NG];
  bf16x8 am;
  int vis[4];  // visible keys of rows 4 (lane / 16) + r

  __device__ __forceinline__ void load(const CacheAttnParams& p, int b, int h, int r0, int lane) {
    const int o = lane >> 4, r = r0 + (lane & 15);
    const bool ok = r < p.R;
    const int rr = ok ? r : 0, head = h * p.rep + rr / p.NQ, i = rr % p.NQ;
    const T* q = static_cast<const T*>(p.q) + size_t(b) * p.lq.sb + size_t(head) * p.lq.sh + size_t(i) * p.lq.sn;
    float sum[NG];
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
      float t = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
      sum[g] = sum_groups(t);
#pragma unroll
      for (int k = 0; k < NT; ++k)
        for (int j = 0; j < 8; ++j) {
          const __bf16 y = static_cast<__bf16>(x[j]);
          a[g][k][j < 4 ? 2 * j : 2 * j - 7] = y;  // codes_operand's order
          x[j] -= static_cast<float>(y);
        }
      for (int k = 0; k < 4; ++k) bias[g][k] = -16.0f * __shfl(sum[g], 4 * o + k, 64);
    }
    // sum q_g in three bf16 terms (24 bits) against m_g: slots of lane group
    // 0 hold the first two terms of four groups, those of group 1 the third
    for (int j = 0; j < 8; ++j) am[j] = static_cast<__bf16>(0.0f);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const __bf16 s0 = static_cast<__bf16>(sum[g]);
      const float r1 = sum[g] - static_cast<float>(s0);
      const __bf16 s1 = static_cast<__bf16>(r1);
      const __bf16 s2 = static_cast<__bf16>(r1 - static_cast<float>(s1));
      if (o == 0) am[g] = s0, am[4 + g] = s1;
      if (o == 1) am[g] = s2;
    }
    for (int k = 0; k < 4; ++k) {
      const int row = r0 + 4 * o + k;
      vis[k] = row < p.R ? visible_keys(p, b, row % p.NQ) : 0;
    }
  }
};

// The codes (key order: lane group o has octet o of every group) and params
// of the lane's key.
template <int NG>
struct KeyRow {
  uint32_t w[NG], pr[NG];
  __device__ __forceinline__ void load(const CachePool& c, int64_t row, int o) {
    const uint32_t* cw = reinterpret_cast<const uint32_t*>(c.k_codes) + row * (4 * NG) + NG * o;
    const uint32_t* cp = c.k_params + row * NG;
    __builtin_memcpy(w, __builtin_assume_aligned(cw, NG == 4 ? 16 : NG == 2 ? 8 : 4), 4 * NG);
    __builtin_memcpy(pr, __builtin_assume_aligned(cp, NG == 4 ? 16 : NG == 2 ? 8 : 4), 4 * NG);
  }
};

// 8 codes as bf16 16 + c: channels 0 4 1 5 2 6 3 7, since nibbles j and j + 4
// are 16 bits apart.  The query operand has the same order.
__device__ __forceinline__ bf16x8 codes_operand(uint32_t w) {
  const uint32_t mask = 0x00780078u, one = 0x41804180u;
  uint32_t u[4];
  u[0] = ((w << 3) & mask) | one;
  u[1] = ((w >> 1) & mask) | one;
  u[2] = ((w >> 5) & mask) | one;
  u[3] = ((w >> 9) & mask) | one;
  bf16x8 r;
  __builtin_memcpy(&r, u, 16);
  return r;
}

// q.k of 16 rows x 16 keys: element r of a lane is row 4 (lane / 16) + r,
// key lane % 16.
template <typename T, int NT, int NG>
__device__ __forceinline__ f32x4 dots(const QueryFrag<T, NT, NG>& q, const KeyRow<NG>& k) {
  uint32_t mm[4] = {};
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const uint32_t m = k.pr[g] >> 16;
    mm[g >> 1] |= (g & 1) ? (k.pr[g] & 0xffff0000u) : m;
  }
  mm[2] = mm[0], mm[3] = mm[1];
  bf16x8 bm;
  __builtin_memcpy(&bm, mm, 16);
  f32x4 s = mfma(q.am, bm, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const bf16x8 u = codes_operand(k.w[g]);
    f32x4 acc = q.bias[g];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc = mfma(q.a[g][t], u, acc);
    const float sc = __uint_as_float(k.pr[g] << 16);
    for (int r = 0; r < 4; ++r) s[r] = fmaf(sc, acc[r], s[r]);
  }
  return s;
}

// z = (alpha - 1) clamp(scale dot); a dot that is not a number counts as the
// lower bound, as in the score clamp of the dense path.
__device__ __forceinline__ float z_of(float dot, float c, float zb) {
  return __builtin_amdgcn_fmed3f(dot * c, -zb, zb);
}

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

// z of the keys [key0, key1) x 16 rows by the block's waves, 16 U keys per
// wave and step, handed to put(r, key, z) (row 4 (lane / 16) + r of the
// tile).  key0 is a multiple of the page size; pages: stage_pages of it.
template <int U, int NW, typename T, int NT, int NG, typename Put>
__device__ __forceinline__ void score_keys(const CacheAttnParams& p, const QueryFrag<T, NT, NG>& q, int h,
                                           int key0, int key1, const int* pages, int w, int lane,
                                           Put put) {
  const float zc = (p.alpha - 1.0f) * p.scale, zb = 10.0f * (p.alpha - 1.0f);
  const int o = lane >> 4, kl = lane & 15;
  for (int base = key0 + w * (kSub * U); base < key1; base += NW * (kSub * U)) {
    KeyRow<NG> kr[U];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = base + kSub * u;
      const int pg = key < key1 ? __builtin_amdgcn_readfirstlane(pages[(key - key0) >> p.c.page_shift]) : -1;
      on[u] = pg >= 0;
      if (on[u])
        kr[u].load(p.c, (int64_t(pg) * p.c.heads + h) * p.c.page + (key & (p.c.page - 1)) + kl, o);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = base + kSub * u + kl;
      if (on[u]) {
        const f32x4 d = dots<T, NT, NG>(q, kr[u]);
        for (int r = 0; r < 4; ++r) put(r, key, key < q.vis[r] ? z_of(d[r], zc, zb) : kHidden);
      } else if (base + kSub * u < key1) {
        for (int r = 0; r < 4; ++r) put(r, key, kHidden);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Threshold and values of one row by a team of waves
// ---------------------------------------------------------------------------

__device__ __forceinline__ float wave_sum(float v) {
  v += __uint_as_float(lane_xor<1>(__float_as_uint(v)));
  v += __uint_as_float(lane_xor<2>(__float_as_uint(v)));
  v += __uint_as_float(lane_xor<7>(__float_as_uint(v)));
  v += __uint_as_float(lane_xor<15>(__float_as_uint(v)));
  return sum_groups(v);
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, __uint_as_float(lane_xor<1>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(lane_xor<2>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(lane_xor<7>(__float_as_uint(v))));
  v = fmaxf(v, __uint_as_float(lane_xor<15>(__float_as_uint(v))));
  return __uint_as_float(group_reduce_bits(__float_as_uint(v), [](uint32_t x, uint32_t y) {
    return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y)));
  }));
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

// LDS of the row teams: a candidate list and partial sums for each wave.
struct TeamLds {
  float* lz;   // [NW][cap] z, later p
  int* li;     // [NW][cap] key
  float* red;  // [NW][4]
  int* cnt;    // [NW]
  float* acc;  // [NW][kAccStride]
  int cap;
};
constexpr int kAccStride = 132;
template <int NW> __host__ __device__ inline size_t team_lds_bytes(int cap) {
  return size_t(NW) * (size_t(cap) * 8 + 16 + 4 + kAccStride * 4);
}
template <int NW> __device__ __forceinline__ TeamLds team_lds(void* base, int cap) {
  TeamLds l;
  l.lz = static_cast<float*>(base);
  l.li = reinterpret_cast<int*>(l.lz + NW * cap);
  l.red = reinterpret_cast<float*>(l.li + NW * cap);
  l.cnt = reinterpret_cast<int*>(l.red + NW * 4);
  l.acc = reinterpret_cast<float*>(l.cnt + NW);
  l.cap = cap;
  return l;
}

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
  // the wave's sums of channels 8 c + j, in the lanes of slot 0
  __device__ __forceinline__ void reduce() {
    for (int j = 0; j < 8; ++j) {
      acc[j] += off;
      if constexpr (kCl <= 4) acc[j] += __uint_as_float(lane_xor<4>(__float_as_uint(acc[j])));
      if constexpr (kCl <= 8) acc[j] += __uint_as_float(lane_xor<8>(__float_as_uint(acc[j])));
      acc[j] = sum_groups(acc[j]);
    }
  }
};

// tau and the output of row `row` (of the key head's R) from its z at zp[0 ..
// vis), by `size` waves of the block, of which this is number `member`; its
// waves are w0 .. w0 + size - 1.  Every wave of the block calls it together
// (teams meet at the block's barriers); vis = 0 for a team without a row.
// zpart: the wave's part of the row's maximum.
template <typename T, int NG, int NW>
__device__ __forceinline__ void finish_row(const CacheAttnParams& p, int b, int h, int row, int vis,
                                           const float* zp, float zpart, const TeamLds& L, int w, int w0,
                                           int size, int lane) {
  const int member = w - w0;
  const float e = 1.0f / (p.alpha - 1.0f);
  const int pc = pow_class_of(e);
  const float wm = wave_max(zpart);
  if (lane == 0) L.red[4 * w] = wm;
  __syncthreads();
  float zmax = kHidden;
  for (int i = 0; i < size; ++i) zmax = fmaxf(zmax, L.red[4 * (w0 + i)]);
  const bool empty = !(zmax > 0.5f * kHidden);
  float tau = zmax - 1.0f, lo = tau, hi = zmax;

  // ---- the keys with z > lo, listed per wave; lo moves up while they do not fit ----
  float* lz = L.lz + w * L.cap;
  int* li = L.li + w * L.cap;
  bool listed = false, dense = empty;
  int mine = 0;
  for (int it = 0;; ++it) {
    if (!listed && !dense) {
      mine = 0;
      for (int j0 = member * kWave; j0 < vis; j0 += size * kWave) {
        const float z = j0 + lane < vis ? zp[j0 + lane] : kHidden;
        const uint64_t m = __ballot(z > lo);
        const int at = mine + lane_rank(m);
        if (z > lo && at < L.cap) {
          lz[at] = z;
          li[at] = j0 + lane;
        }
        mine += __builtin_popcountll(m);
      }
      if (lane == 0) L.cnt[w] = mine;
    }
    __syncthreads();
    if (!listed && !dense) {
      listed = true;
      for (int i = 0; i < size; ++i) listed = listed && L.cnt[w0 + i] <= L.cap;
    }
    if (!__syncthreads_or(!listed && !dense)) break;
    // some team's candidates did not fit: one step of its tau over the whole row
    float F = 0.0f, F1 = 0.0f;
    if (!listed && !dense) {
      for (int j0 = member * kWave; j0 < vis; j0 += size * kWave) {
        const float z = j0 + lane < vis ? zp[j0 + lane] : kHidden;
        float pa, pa1;
        powers(pc, fmaxf(z - tau, 0.0f), e, pa, pa1);
        F += pa;
        F1 += pa1;
      }
      F = wave_sum(F);
      F1 = wave_sum(F1);
      if (lane == 0) {
        L.red[4 * w + 1] = F;
        L.red[4 * w + 2] = F1;
      }
    }
    __syncthreads();
    if (!listed && !dense) {
      F = F1 = 0.0f;
      for (int i = 0; i < size; ++i) {
        F += L.red[4 * (w0 + i) + 1];
        F1 += L.red[4 * (w0 + i) + 2];
      }
      dense = next_tau(p.alpha, F, F1, tau, lo, hi) || it == kMaxSteps;
      if (p.alpha <= 2.0f) lo = tau;  // the steps stay left of the root
    }
  }

  // ---- tau over the team's lists; every wave does the same steps ----
  if (listed) {
    tau = lo;
    for (int it = 0; it < kMaxSteps; ++it) {
      float F = 0.0f, F1 = 0.0f;
      for (int i = 0; i < size; ++i) {
        const float* z = L.lz + (w0 + i) * L.cap;
        const int n = L.cnt[w0 + i];
        for (int j = lane; j < n; j += kWave) {
          float pa, pa1;
          powers(pc, fmaxf(z[j] - tau, 0.0f), e, pa, pa1);
          F += pa;
          F1 += pa1;
        }
      }
      if (next_tau(p.alpha, wave_sum(F), wave_sum(F1), tau, lo, hi)) break;
    }
  }
  __syncthreads();  // every wave has read the lists that their owners now reuse

  // ---- the support's weights and values ----
  ValueSum<NG> vs;
  float psum = 0.0f;
  if (!empty) {
    // listed: the wave's own list; else its keys of the row, cap at a time
    const int per = listed ? mine : L.cap;
    const int end = listed ? 1 : vis;
    for (int k0 = listed ? 0 : member * per; k0 < end; k0 += size * per) {
      const int cnt = listed ? mine : min(per, vis - k0);
      int n = 0;
      for (int j0 = 0; j0 < cnt; j0 += kWave) {
        const int j = j0 + lane;
        const float z = j >= cnt ? kHidden : listed ? lz[j] : zp[k0 + j];
        const int key = j >= cnt ? 0 : listed ? li[j] : k0 + j;
        float pa, pa1;
        powers(pc, fmaxf(z - tau, 0.0f), e, pa, pa1);
        const uint64_t m = __ballot(pa > 0.0f);
        if (pa > 0.0f) {
          const int at = n + lane_rank(m);  // at most j: already read
          lz[at] = pa;
          li[at] = key;
        }
        n += __builtin_popcountll(m);
        psum += pa;
      }
      vs.add(p, b, h, lz, li, n, lane);
      if (listed) break;
    }
    psum = wave_sum(psum);
  }
  vs.reduce();
  constexpr int kCl = ValueSum<NG>::kCl;
  if (lane < kCl && lane < 4 * NG)
    for (int j = 0; j < 8; ++j) L.acc[w * kAccStride + 8 * lane + j] = vs.acc[j];
  if (lane == 0) L.red[4 * w + 3] = psum;
  __syncthreads();
  if (row >= 0) {
    float total = 0.0f;
    for (int i = 0; i < size; ++i) total += L.red[4 * (w0 + i) + 3];
    const float inv = total > 0.0f ? 1.0f / total : 0.0f;
    const int head = h * p.rep + row / p.NQ, i = row % p.NQ;
    T* out = static_cast<T*>(p.out) + ((size_t(b) * p.H + head) * p.NQ + i) * p.c.hd;
    for (int ch = member * kWave + lane; ch < p.c.hd; ch += size * kWave) {
      float v = 0.0f;
      for (int k = 0; k < size; ++k) v += L.acc[(w0 + k) * kAccStride + ch];
      Elem<T>::store(out + ch, v * inv);
    }
  }
}

// ---------------------------------------------------------------------------
// Kernels
// ---------------------------------------------------------------------------

constexpr int kOneWaves = 16;   // one-block plan
constexpr int kScoreWaves = 4;  // split plan: score blocks

// One block per 16 rows of a key head: scores into LDS, then its rows.
template <typename T, int NT, int NG>
__global__ __launch_bounds__(kOneWaves * kWave) void cache_one_kernel(CacheAttnParams p, int cap, int stride) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int t = threadIdx.x, w = t >> 6, lane = t & 63;
  const int nrt = (p.R + kRows - 1) / kRows;
  const int rt = blockIdx.x % nrt, bh = blockIdx.x / nrt;
  const int b = bh / p.c.heads, h = bh % p.c.heads;
  const int r0 = rt * kRows, rows = min(kRows, p.R - r0);
  const TeamLds L = team_lds<kOneWaves>(smem, cap);
  float* zs = reinterpret_cast<float*>(smem + team_lds_bytes<kOneWaves>(cap));
  int* pages = reinterpret_cast<int*>(zs + rows * stride);

  const int len = max(0, min(p.lengths[b], p.maxlen));
  stage_pages(p, b, 0, len, pages, t, kOneWaves * kWave);
  QueryFrag<T, NT, NG> q;
  q.load(p, b, h, r0, lane);
  __syncthreads();
  const int o = lane >> 4;
  score_keys<2, kOneWaves>(p, q, h, 0, len, pages, w, lane, [&](int r, int key, float z) {
    if (4 * o + r < rows) zs[(4 * o + r) * stride + key] = z;
  });
  __syncthreads();
  int pad = 1;
  while (pad < rows) pad *= 2;
  const int size = kOneWaves / pad, row = w / size, w0 = row * size;
  const bool has = row < rows;
  const int vis = has ? visible_keys(p, b, (r0 + row) % p.NQ) : 0;
  const float* zp = zs + (has ? row : 0) * stride;
  float zpart = kHidden;
  for (int j = (w - w0) * kWave + lane; j < vis; j += size * kWave) zpart = fmaxf(zpart, zp[j]);
  finish_row<T, NG, kOneWaves>(p, b, h, has ? r0 + row : -1, vis, zp, zpart, L, w, w0, size, lane);
}

// Split plan, first launch: z of `span` keys x 16 rows, and its maxima.
template <typename T, int NT, int NG>
__global__ __launch_bounds__(kScoreWaves * kWave) void cache_score_kernel(CacheAttnParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ float wmax[kScoreWaves][kRows];
  int* pages = reinterpret_cast<int*>(smem);
  const int t = threadIdx.x, w = t >> 6, lane = t & 63, o = lane >> 4;
  const int nrt = (p.R + kRows - 1) / kRows;
  const int split = blockIdx.x % p.nsplit, rest = blockIdx.x / p.nsplit;
  const int rt = rest % nrt, bh = rest / nrt;
  const int b = bh / p.c.heads, h = bh % p.c.heads;
  const int r0 = rt * kRows;
  const int key0 = split * p.span;
  const int len = max(0, min(p.lengths[b], p.maxlen));
  if (key0 >= len) return;
  const int key1 = min(len, key0 + p.span);
  stage_pages(p, b, key0, key1 - key0, pages, t, kScoreWaves * kWave);
  QueryFrag<T, NT, NG> q;
  q.load(p, b, h, r0, lane);
  __syncthreads();
  const size_t zstride = size_t(p.span) * p.nsplit;
  float* zrow = p.scores + (size_t(bh) * p.R + r0 + 4 * o) * zstride;
  float rmax[4] = {kHidden, kHidden, kHidden, kHidden};
  const int nr = p.R - r0 - 4 * o;  // the lane's rows below nr are real
  score_keys<4, kScoreWaves>(p, q, h, key0, key1, pages, w, lane, [&](int r, int key, float z) {
    if (r < nr && key < key1) zrow[size_t(r) * zstride + key] = z;
    rmax[r] = fmaxf(rmax[r], z);
  });
  for (int r = 0; r < 4; ++r) {
    float m = rmax[r];
    m = fmaxf(m, __uint_as_float(lane_xor<1>(__float_as_uint(m))));
    m = fmaxf(m, __uint_as_float(lane_xor<2>(__float_as_uint(m))));
    m = fmaxf(m, __uint_as_float(lane_xor<7>(__float_as_uint(m))));
    m = fmaxf(m, __uint_as_float(lane_xor<15>(__float_as_uint(m))));
    if ((lane & 15) == 0) wmax[w][4 * o + r] = m;
  }
  __syncthreads();
  if (t < kRows && r0 + t < p.R) {
    float m = wmax[0][t];
    for (int i = 1; i < kScoreWaves; ++i) m = fmaxf(m, wmax[i][t]);
    p.smax[(size_t(bh) * p.R + r0 + t) * p.nsplit + split] = m;
  }
}

// Split plan, second launch: one block per row.
template <typename T, int NG, int NW>
__global__ __launch_bounds__(NW * kWave) void cache_row_kernel(CacheAttnParams p, int cap) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int t = threadIdx.x, w = t >> 6, lane = t & 63;
  const int row = blockIdx.x % p.R, bh = blockIdx.x / p.R;
  const int b = bh / p.c.heads, h = bh % p.c.heads;
  const TeamLds L = team_lds<NW>(smem, cap);
  const int vis = visible_keys(p, b, row % p.NQ);
  const size_t at = size_t(bh) * p.R + row;
  const float* zp = p.scores + at * (size_t(p.span) * p.nsplit);
  const int ns = (vis + p.span - 1) / p.span;
  float zpart = kHidden;
  for (int j = t; j < ns; j += NW * kWave) zpart = fmaxf(zpart, p.smax[at * p.nsplit + j]);
  finish_row<T, NG, NW>(p, b, h, row, vis, zp, zpart, L, w, 0, NW, lane);
}

template <typename K> hipError_t allow_lds(K kern, size_t lds) {
  if (lds <= 65536) return hipSuccess;
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                             int(lds));
}

constexpr int kOneCap = 256;   // candidates per wave, one-block plan
constexpr int kRowCap = 512;   // candidates per wave, split plan
constexpr int kRowWaves = 16;

size_t one_lds_bytes(const CacheAttnParams& p, int* stride) {
  const int rows = p.R < kRows ? p.R : kRows;
  *stride = (p.maxlen + 15) / 16 * 16 + 4;
  return team_lds_bytes<kOneWaves>(kOneCap) + size_t(rows) * *stride * 4 +
         size_t((p.maxlen + p.c.page - 1) / p.c.page + 1) * 4;
}

template <typename T, int NT, int NG>
hipError_t launch_ng(const CacheAttnParams& p, hipStream_t s) {
  const int nrt = (p.R + kRows - 1) / kRows;
  if (p.plan == kCacheOneBlock) {
    int stride = 0;
    const size_t lds = one_lds_bytes(p, &stride);
    auto kern = cache_one_kernel<T, NT, NG>;
    if (hipError_t e = allow_lds(kern, lds)) return e;
    profile_begin("cache_attn", s);
    hipLaunchKernelGGL(kern, dim3(unsigned(p.B) * p.c.heads * nrt), dim3(kOneWaves * kWave), lds, s, p, kOneCap,
                       stride);
    profile_end(s);
    return hipGetLastError();
  }
  profile_begin("cache_score", s);
  hipLaunchKernelGGL((cache_score_kernel<T, NT, NG>), dim3(unsigned(p.B) * p.c.heads * nrt * p.nsplit),
                     dim3(kScoreWaves * kWave), size_t(p.span / p.c.page + 1) * 4, s, p);
  profile_end(s);
  if (hipError_t e = hipGetLastError()) return e;
  const size_t lds = team_lds_bytes<kRowWaves>(kRowCap);
  auto kern = cache_row_kernel<T, NG, kRowWaves>;
  if (hipError_t e = allow_lds(kern, lds)) return e;
  profile_begin("cache_row", s);
  hipLaunchKernelGGL(kern, dim3(unsigned(p.B) * p.c.heads * p.R), dim3(kRowWaves * kWave), lds, s, p, kRowCap);
  profile_end(s);
  return hipGetLastError();
}

template <typename T, int NT>
hipError_t launch_t(const CacheAttnParams& p, hipStream_t s) {
  switch (p.c.G) {
    case 1: return launch_ng<T, NT, 1>(p, s);
    case 2: return launch_ng<T, NT, 2>(p, s);
    case 3: return launch_ng<T, NT, 3>(p, s);
    default: return launch_ng<T, NT, 4>(p, s);
  }
}

}  // namespace

size_t cache_attn_plan(CacheAttnParams& p, size_t max_lds, int cus) {
  int stride = 0;
  p.span = p.nsplit = 0;
  if (p.maxlen <= 2048 && one_lds_bytes(p, &stride) <= max_lds) {
    p.plan = kCacheOneBlock;
    return 0;
  }
  p.plan = kCacheSplit;
  const long long nrt = (p.R + kRows - 1) / kRows, tiles = (long long)p.B * p.c.heads * nrt;
  // eight score blocks per compute unit, of at least 256 keys (the largest
  // page: a block starts on a page)
  long long span = (p.maxlen * tiles + 8LL * cus - 1) / (8LL * cus);
  span = (span + 255) / 256 * 256;
  if (span > 4096) span = 4096;
  p.span = int(span);
  p.nsplit = int((p.maxlen + span - 1) / span);
  const size_t rows = size_t(p.B) * p.c.heads * p.R;
  return rows * p.nsplit * (size_t(p.span) + 1) * sizeof(float);
}

hipError_t launch_cache_attn(const CacheAttnParams& p, int dtype, hipStream_t s) {
  if (dtype == kElemBF16) return launch_t<u16, 1>(p, s);
  if (dtype == kElemF16) return launch_t<h16, 2>(p, s);
  return launch_t<float, 3>(p, s);
}

}  // namespace asa
