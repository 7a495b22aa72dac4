// alpha-entmax attention of a few query tokens over the 4-bit cache.
//
// Per query row, with z_j = (alpha - 1) clamp(scale q.k_j, -10, 10) over the
// visible keys j and e = 1 / (alpha - 1):
//
//   sum_j max(z_j - tau, 0)^e = 1,  out = sum_j p_j v_j / sum_j p_j,
//   p_j = max(z_j - tau, 0)^e.
//
// Bytes: the keys', 5 bits per channel, are what a row costs.  They are read
// once and never become keys.  With u = 16 + c (exact in 16 bits: c is shifted
// into the mantissa of 16.0), group g and its query part q_g,
//
//   q.k = sum_g s_g (q_g.u_g - 16 sum q_g) + m_g sum q_g:
//
// one 16x16x32 MFMA per group gives q_g.u_g for 16 rows x 16 keys (a group is
// the instruction's 32 channels), its accumulator starts at -16 sum q_g, and
// the keys' scales multiply the finished group sums.  16-bit queries enter as
// they are, fp32 ones as three bf16 terms (24 bits), so that scores carry
// fp32 rounding only, for every type.
//
// A key head serves few query rows, and what follows an MFMA (scales, maxima,
// stores) costs the same for one row as for 16.  With R <= 16 / P rows, P key
// tiles share the 16 rows of one result: tile u's operand holds the queries
// in rows u (16 / P) .. and zeros elsewhere, so that its products add to
// those of the other tiles without meeting them, and each lane of the result
// has a key of its own to scale (about 250 vector instructions per 64 keys of
// head dimension 128 at P = 4).
//
// tau lies in [max z - 1, max z], so only keys with z > max z - 1 can have a
// weight.  A better bound: the sum over any part of the row is at most the
// whole one, so the tau of the row's granule maxima (the largest z of each 64
// keys, which the score pass keeps) is at most tau, and close to it, since a
// long row's support lies in as many granules.  Only granules whose maximum
// is above that bound are looked at again: their keys above it are listed
// (key, z) in LDS, Newton steps over the list find tau, and only the value
// rows of the list are read.  alpha-entmax gives most keys of a long row no
// weight, so the values' bytes are a small part of the keys'.  A list that
// does not fit raises the bound by Newton steps over the whole row, down to
// rows with more weights than any list, which are summed as they are read.
// Lists and sums have a fixed order: results do not depend on timing.
//
// Two plans (cache_attn_plan).  One block per tile of rows, dots in LDS; or
// keys split over score blocks, dots in the workspace, then one block per
// row.  16 x 32768 keys, 8 key heads, 32 heads of 128, bf16: score pass 75 us
// for 335 MB of keys (the card reads 6.3 TB/s and copies 5.1; 61 MB of dots
// are written), rows 15 us, which are latency: five dependent reads and a
// dozen Newton steps.
#pragma once

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
// mask and one are held in registers (v_and_or_b32 takes no literals).  For
// fp32 queries c - 8 instead, 21 instructions to eight codes rather than 8: the
// sums' roundings are relative to the operand's size, and 16-bit results do
// not show them (60 drawn fp32 calls: mean error 4.6e-7, the plain fp32
// form's 7.4e-7).
template <typename T> struct Codes {
  static constexpr bool kF16 = std::is_same<T, h16>::value;
  static constexpr bool kCentred = std::is_same<T, float>::value;
  uint32_t mask = kF16 ? 0x03c003c0u : 0x00780078u;
  uint32_t one = kF16 ? 0x4c004c00u : 0x41804180u;  // 16.0; the codes' unit is 1 << 6, 1 << 3
  __device__ __forceinline__ Codes() { asm("" : "+s"(mask), "+v"(one)); }
  __device__ __forceinline__ CodeVec<T> operator()(uint32_t w) const {
    uint32_t u[4];
    if constexpr (kCentred) {
      const int x = int(w ^ 0x88888888u);  // nibbles c - 8 in two's complement
      for (int j = 0; j < 4; ++j) {
        const uint32_t lo = __float_as_uint(float((x << (28 - 4 * j)) >> 28));
        const uint32_t hi = __float_as_uint(float((x << (12 - 4 * j)) >> 28));
        u[j] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);  // the bf16 halves: small integers are exact
      }
    } else if constexpr (kF16) {
      u[0] = ((w << 6) & mask) | one;
      u[1] = ((w << 2) & mask) | one;
      u[2] = ((w >> 2) & mask) | one;
      u[3] = ((w >> 6) & mask) | one;
    } else {
      u[0] = ((w << 3) & mask) | one;
      u[1] = ((w >> 1) & mask) | one;
      u[2] = ((w >> 5) & mask) | one;
      u[3] = ((w >> 9) & mask) | one;
    }
    CodeVec<T> r;
    __builtin_memcpy(&r, u, 16);
    return r;
  }
};

// The query operand of a tile of rows r0 .. of a key head's R rows (row r:
// query head h * rep + r / NQ, token r % NQ), kR of them, in LDS: a lane of
// tile u reads its row's 8 channels if its operand row is one of tile u's,
// and the zeros behind each group's entries if not.  In registers the P
// operands would take 64 of them and the occupancy that hides the loads.
template <typename T, int P, int NG>
struct QueryLds {
  static constexpr int kR = kTile / P;
  static constexpr int NT = std::is_same<T, float>::value ? 3 : 1;
  uint4 a[NG][NT][4 * kR + 1];  // [..][octet * kR + row], zeros
  f32x4 bias[NG][kTile / 4];        // -16 sum q_g of each row
};

// 8 channels of a query row from `ch` on, zeros past the head dimension.
template <typename T>
__device__ __forceinline__ void load_query(const CacheAttnParams& p, const T* q, int ch, float* x) {
  const int nv = p.c.hd - ch;
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
}

// Fills ql by the block's `waves` waves, a channel group each; queries of a
// negative scale are negated, so that larger products are larger scores.
template <typename T, int P, int NG>
__device__ __forceinline__ void stage_query(const CacheAttnParams& p, QueryLds<T, P, NG>& ql, int b, int h, int r0,
                                            int w, int waves, int lane) {
  using S = typename Half<CodeType<T>>::scalar;
  using QL = QueryLds<T, P, NG>;
  constexpr int kR = QL::kR;
  const int o = lane >> 4, r = lane & 15;
  const bool ok = r < kR && r0 + r < p.R;
  const int rr = ok ? r0 + r : 0, head = h * p.rep + rr / p.NQ, i = rr % p.NQ;
  const T* q = static_cast<const T*>(p.q) + size_t(b) * p.lq.sb + size_t(head) * p.lq.sh + size_t(i) * p.lq.sn;
  const float sign = p.scale < 0.0f ? -1.0f : 1.0f;
  for (int g = w; g < NG; g += waves) {
    float x[8];
    load_query<T>(p, q, 32 * g + 8 * o, x);
    for (int j = 0; j < 8; ++j) x[j] = ok ? x[j] * sign : 0.0f;
    const float sum = sum_groups(((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7])));
    if (o == 0) reinterpret_cast<float*>(ql.bias[g])[r] = -16.0f * sum;
#pragma unroll
    for (int t = 0; t < QL::NT; ++t) {
      CodeVec<T> v;
      for (int j = 0; j < 8; ++j) {
        const S y = static_cast<S>(x[j]);
        x[j] -= static_cast<float>(y);
        v[operand_slot(j)] = y;
      }
      uint4 u;
      __builtin_memcpy(&u, &v, 16);
      if (r < kR) ql.a[g][t][o * kR + r] = u;
      if (lane == 0) ql.a[g][t][4 * kR] = uint4{0u, 0u, 0u, 0u};
    }
  }
}

// Where a wave reads the operand, and what its rows see.
template <int P>
struct TileRows {
  static constexpr int kR = kTile / P;
  int at[P];       // entry of QueryLds::a for tile u
  int bias;        // and of its bias, for the result's rows
  int vis[4];      // visible keys of rows (4 (lane / 16) + k) % kR
  int most, least; // over the real rows of the tile
  // row whose granule maximum the lane has after granule_maxima
  __device__ __forceinline__ static int max_row(int lane) {
    const int o = lane >> 4;
    return P == 4 ? o : P == 2 ? 4 * (o & 1) + (o & 2) + (lane & 1) : 4 * o + (lane & 3);
  }
  __device__ __forceinline__ void load(const CacheAttnParams& p, int b, int r0, int lane) {
    const int o = lane >> 4, ar = lane & 15, row = r0 + ar % kR;
    for (int u = 0; u < P; ++u) at[u] = ar / kR == u ? o * kR + ar % kR : 4 * kR;
    bias = o % (kR / 4);
    const int v = row < p.R ? visible_keys(p, b, row % p.NQ) : 0;
    most = wave_reduce_minmax<true>(v);
    least = wave_reduce_minmax<false>(row < p.R ? v : INT_MAX);
    for (int k = 0; k < 4; ++k) vis[k] = __shfl(v, (4 * o + k) % kR, 64);
  }
};

// A granule: 64 keys, four tiles of 16 in 4 / P packs of P tiles that share a
// result.  The codes (key order: lane group o has octet o of every channel
// group) of key lane % 16 of each tile, and the params of the lane's own key
// of each pack's result.
constexpr int kGranule = kCacheGranule;
template <int P, int NG>
struct KeyGranule {
  static constexpr int V = 4 / P;
  uint32_t w[4][NG], pr[V][NG];
  bool seen[V];  // the lane's own key has a page
  bool whole;    // every key of the granule has one (wave-uniform)

  // Where one tile holds all rows (P > 1: the plan's rule) the keys are read
  // once in a call, and a large batch's would only push the dots and values
  // out of the caches: 16 x 32768 93 -> 88 us, 4 x 16384 (spread rows) 47 ->
  // 42, 1 x 131072 (84 MB, which do fit) 32 -> 33.
  template <int N> static __device__ __forceinline__ void words(uint32_t* d, const uint32_t* s) {
    if constexpr (P > 1 && (N == 2 || N == 4)) {
      typedef uint32_t vec __attribute__((ext_vector_type(N)));
      const vec x = __builtin_nontemporal_load(reinterpret_cast<const vec*>(s));
      __builtin_memcpy(d, &x, 4 * N);
    } else if constexpr (P > 1) {
      for (int i = 0; i < N; ++i) d[i] = __builtin_nontemporal_load(s + i);
    } else {
      __builtin_memcpy(d, __builtin_assume_aligned(s, N == 4 ? 16 : N == 2 ? 8 : 4), 4 * N);
    }
  }
  // keys base .. base + 63 of [.., key1); pages: of the keys from key0
  __device__ __forceinline__ void load(const CachePool& c, int h, const int* pages, int key0, int base, int key1,
                                       int lane) {
    const int o = lane >> 4, col = lane & 15;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(c.k_codes);
    if (c.page >= kGranule) {  // one page: its address is the wave's, the rest a constant of the lane
      const int pg = __builtin_amdgcn_readfirstlane(pages[(base - key0) >> c.page_shift]);
      const bool on = pg >= 0;
      const size_t row = (size_t(on ? pg : 0) * c.heads + h) * c.page + (base & (c.page - 1));
      const uint32_t* cw = codes + row * (4 * NG);
      const uint32_t* cp = c.k_params + row * NG;
#pragma unroll
      for (int u = 0; u < 4; ++u) words<NG>(w[u], cw + (kTile * u + col) * (4 * NG) + NG * o);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        seen[v] = on;
        words<NG>(pr[v], cp + (kTile * (P * v + o * P / 4) + col) * NG);
      }
      whole = on;
    } else {
      // a page for each tile (read without branches: positions past the last
      // key take its page, and are not seen)
      whole = base + kGranule <= key1;
      int pg[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        pg[u] = __builtin_amdgcn_readfirstlane(pages[(min(base + kTile * u, key1 - 1) - key0) >> c.page_shift]);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        whole = whole && pg[u] >= 0;
        const size_t row = (size_t(pg[u] >= 0 ? pg[u] : 0) * c.heads + h) * c.page + ((base + kTile * u) & (c.page - 1));
        words<NG>(w[u], codes + row * (4 * NG) + (col * (4 * NG) + NG * o));
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        // the lane's own tile is P v + o P / 4
        int mine = pg[P * v];
        for (int u = 1; u < P; ++u) mine = o * P / 4 == u ? pg[P * v + u] : mine;
        const int key = base + kTile * (P * v + o * P / 4);
        seen[v] = mine >= 0 && key < key1;
        const size_t row = (size_t(mine >= 0 ? mine : 0) * c.heads + h) * c.page + (key & (c.page - 1)) + col;
        words<NG>(pr[v], c.k_params + row * NG);
      }
    }
  }
};

// q.k: element k of s[v] is row (4 (lane / 16) + k) % kR, key
// 16 (P v + lane / 16 * P / 4) + lane % 16 of the granule.
template <typename T, int P, int NG>
__device__ __forceinline__ void dots(const QueryLds<T, P, NG>& ql, const TileRows<P>& t, const KeyGranule<P, NG>& k,
                                     const Codes<T>& codes, f32x4* s) {
  constexpr int V = 4 / P, NT = QueryLds<T, P, NG>::NT;
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const f32x4 bias = ql.bias[g][t.bias];
    CodeVec<T> a[P][NT];
#pragma unroll
    for (int u = 0; u < P; ++u)
      for (int i = 0; i < NT; ++i) __builtin_memcpy(&a[u][i], &ql.a[g][i][t.at[u]], 16);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      f32x4 acc = Codes<T>::kCentred ? f32x4{0.0f, 0.0f, 0.0f, 0.0f} : bias;
#pragma unroll
      for (int u = 0; u < P; ++u) {
        const CodeVec<T> c = codes(k.w[P * v + u][g]);
        for (int i = 0; i < NT; ++i) acc = mfma(a[u][i], c, acc);
      }
      const float sc = __uint_as_float(k.pr[v][g] << 16);
      // m sum q_g = -m / 16 bias; with c - 8 the offset is that of code 8
      float off = __uint_as_float(k.pr[v][g] & 0xffff0000u);
      if constexpr (Codes<T>::kCentred) off = fmaf(8.0f, sc, off);
      off *= -0.0625f;
      for (int r = 0; r < 4; ++r) s[v][r] = fmaf(off, bias[r], fmaf(sc, acc[r], s[v][r]));
    }
  }
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

// The granule's maximum of the row TileRows::max_row(lane), from the maxima m
// over the lane's own keys: halves and rows are exchanged first, so that
// later steps work on one register, then lanes of a 16-lane row that share
// the query row are reduced by rotations.
template <int R> __device__ __forceinline__ float max_ror(float x) {  // with the lane R further in its 16
  return fmaxf(x, __uint_as_float(dpp_mov<0x120 + R>(__float_as_uint(x))));
}
__device__ __forceinline__ float max_swap32(float x, float y) {  // lanes 0-31: x, 32-63: y, over both halves
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float max_swap16(float x, float y) {  // even 16-lane rows: x, odd: y, over pairs
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
template <int P> __device__ __forceinline__ float granule_maxima(const f32x4& m, int lane) {
  if constexpr (P == 4) {
    float x = max_swap16(max_swap32(m[0], m[2]), max_swap32(m[1], m[3]));
    x = max_ror<1>(x);
    x = max_ror<2>(x);
    x = max_ror<4>(x);
    return max_ror<8>(x);
  } else {
    // lanes with bit k of their number set take y, the others x, over pairs
    auto merge1 = [lane](float x, float y) {
      const bool odd = lane & 1;
      return fmaxf(odd ? y : x, __uint_as_float(lane_xor<1>(__float_as_uint(odd ? x : y))));
    };
    if constexpr (P == 2) {
      float x = merge1(max_swap32(m[0], m[2]), max_swap32(m[1], m[3]));
      x = max_ror<2>(x);
      x = max_ror<4>(x);
      return max_ror<8>(x);
    } else {
      const float x = merge1(m[0], m[1]), y = merge1(m[2], m[3]);
      const bool two = lane & 2;
      float z = fmaxf(two ? y : x, __uint_as_float(lane_xor<2>(__float_as_uint(two ? x : y))));
      z = max_ror<4>(z);
      return max_ror<8>(z);
    }
  }
}

// Dots of the keys [key0, key1) by the block's NW waves, a granule per wave
// and step (the next step's loads are in flight meanwhile), into
// out[(granule * rows + row) * 64 + key % 64], granule = key / 64, and each
// granule's maxima into gmax[row * gstride + granule].  Rows whose largest z
// in a granule is not above that of the wave's granules so far less one can
// have no weight there: their dots are left out.  ONCE: stores past the
// caches, which the dots (16 bytes to a key's 80 at four rows) would share
// with the keys' stream: 16 x 32768, 86 -> 78 us.  key0 is a multiple of the
// page size and of 64.
template <bool ONCE> __device__ __forceinline__ void store_dot(float* p, float d) {
  if constexpr (ONCE) __builtin_nontemporal_store(d, p);
  else *p = d;
}
template <int NW, bool ONCE, typename T, int P, int NG>
__device__ __forceinline__ void score_keys(const CacheAttnParams& p, const QueryLds<T, P, NG>& ql,
                                           const TileRows<P>& tr, int h, int key0, int key1, const int* pages,
                                           int rows, float* out, float* gmax, size_t gstride, int w, int lane) {
  constexpr int V = 4 / P, kR = kTile / P;
  const int o = lane >> 4, own = kTile * (o * P / 4) + (lane & 15), mrow = tr.max_row(lane);
  const ZOf zof(p);
  const Codes<T> codes;
  // lanes that store their row's maximum
  const bool teller = mrow < rows && (lane & 15) == (P == 4 ? 0 : P == 2 ? (lane & 1) : (lane & 3));
  float* gm = gmax + size_t(mrow < rows ? mrow : 0) * gstride;
  float bound = kHidden;
  auto step = [&](int base, const KeyGranule<P, NG>& k) {
    // the operand is read again for every granule (empty, not volatile asm:
    // the reads stay in the loop, and nothing else is ordered by it)
    TileRows<P> t = tr;
    for (int u = 0; u < P; ++u) asm("" : "+v"(t.at[u]) : "s"(base));
    asm("" : "+v"(t.bias) : "s"(base));
    f32x4 d[V];
    dots<T, P, NG>(ql, t, k, codes, d);
#pragma unroll
    for (int v = 0; v < V; ++v)
      for (int r = 0; r < 4; ++r) d[v][r] = fmaxf(d[v][r], kNotNumber);
    if (!k.whole || base + kGranule > t.least)
#pragma unroll
      for (int v = 0; v < V; ++v)
        for (int r = 0; r < 4; ++r)
          d[v][r] = k.seen[v] && base + kTile * P * v + own < t.vis[r] ? d[v][r] : kHidden;
    f32x4 m = d[0];
    for (int v = 1; v < V; ++v)
      for (int r = 0; r < 4; ++r) m[r] = fmaxf(m[r], d[v][r]);
    const float x = granule_maxima<P>(m, lane);
    if (teller) gm[base / kGranule] = x;
    const float z = zof(x);
    const uint64_t want = __ballot(z > bound && mrow < rows);
    bound = fmaxf(bound, z - 1.0f);
    float* og = out + size_t(base / kGranule) * (rows * kGranule);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      // bits of the lanes that have row (4 o + r) % kR
      if constexpr (P == 4) {
        if ((want >> (16 * r)) & 1) store_dot<ONCE>(&og[r * kGranule + own], d[0][r]);
      } else {
        const int row = (4 * o + r) % kR;
        const int bit = P == 2 ? 16 * (o & 1) + 32 * (r >> 1) + (r & 1) : 16 * o + r;
        if ((want >> bit) & 1)
          for (int v = 0; v < V; ++v) store_dot<ONCE>(&og[row * kGranule + kTile * P * v + own], d[v][r]);
      }
    }
  };
  constexpr int kStep = NW * kGranule;
  KeyGranule<P, NG> ka, kb;
  int base = key0 + w * kGranule;
  if (base < key1) ka.load(p.c, h, pages, key0, base, key1, lane);
  while (base < key1) {
    if (base + kStep < key1) kb.load(p.c, h, pages, key0, base + kStep, key1, lane);
    step(base, ka);
    base += kStep;
    if (base >= key1) break;
    if (base + kStep < key1) ka.load(p.c, h, pages, key0, base + kStep, key1, lane);
    step(base, kb);
    base += kStep;
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
// The sums of x and of y over the wave: lanes 0-31 go on with x, the others
// with y, so that both take the steps of one.
__device__ __forceinline__ void wave_sum2(float& x, float& y) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  float v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  v += __uint_as_float(lane_xor<1>(__float_as_uint(v)));
  v += __uint_as_float(lane_xor<2>(__float_as_uint(v)));
  v += __uint_as_float(lane_xor<7>(__float_as_uint(v)));
  v += __uint_as_float(lane_xor<15>(__float_as_uint(v)));
  const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(t[0]) + __uint_as_float(t[1]);
  x = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 0));
  y = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 32));
}
__device__ __forceinline__ float wave_max(float v) {
  return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}
// v^e and v^(e-1), v >= 0, both 0 at v = 0.  The class is the kernel's (alpha
// 1.5, or any): a choice per value costs more than the powers, which other
// alphas take through the hardware's log2 and exp2 (relative error 2^-22 or
// so times e log2 v).
template <int PC> __device__ __forceinline__ void powers(float v, float e, float& pa, float& pa1) {
  if constexpr (PC == kE2) {
    pa = v * v, pa1 = v;
  } else {
    const float l = __builtin_amdgcn_logf(v);
    pa = v > 0.0f ? __builtin_amdgcn_exp2f(e * l) : 0.0f;
    pa1 = v > 0.0f ? __builtin_amdgcn_exp2f((e - 1.0f) * l) : 0.0f;
  }
}

// The weight itself: fp32 results take the library's power.
template <typename T, int PC> __device__ __forceinline__ float weight(float v, float e) {
  if constexpr (PC == kE2) return v * v;
  else if constexpr (std::is_same<T, float>::value) return v > 0.0f ? powf(v, e) : 0.0f;
  else return v > 0.0f ? __builtin_amdgcn_exp2f(e * __builtin_amdgcn_logf(v)) : 0.0f;
}

// One step from tau, where F = sum v^e and F1 = sum v^(e-1) over the keys with
// v = z - tau > 0; true if tau is final instead.  For alpha <= 2 (e >= 1) the
// step is Newton's on the norm F^(1/e) - 1: the norm is convex in tau and
// nearly straight, so the steps from the left end stay left of the root and
// few are needed (five or six from max z - 1).  For alpha > 2 a key just above
// tau makes F1 unbounded, and the bracket is halved instead.  |F - 1| <= 5e-7
// is a few roundings of the sum; the weights are divided by it anyway.
__device__ __forceinline__ bool next_tau(float alpha, float F, float F1, float& tau, float& lo, float& hi) {
  const float f = F - 1.0f;
  if (fabsf(f) <= 5e-7f) return true;
  if (f >= 0.0f) lo = tau;
  else hi = tau;
  float nt = 0.5f * (lo + hi);
  if (alpha <= 2.0f) {
    const float s = tau + (F - __builtin_amdgcn_exp2f((2.0f - alpha) * __builtin_amdgcn_logf(F))) * __builtin_amdgcn_rcpf(F1);
    if (s >= lo && s <= hi) nt = s;
  }
  if (nt == tau || nt == lo || nt == hi) return true;  // between neighbouring floats
  tau = nt;
  return false;
}
constexpr int kMaxSteps = 64;

// LDS of the row teams.  A wave collects up to CAP candidates of its row.
constexpr int kAccStride = 132;
template <int NW, int CAP> struct TeamLds {
  static constexpr int kCap = CAP;
  float cz[NW][CAP];  // a wave's candidates, later its part of the support
  int ci[NW][CAP];
  float gm[NW][kWave];
  float red[2][NW][2];
  float say[NW][4];   // from a team's first wave: zmax, lo; tau, the sum at tau
  float psum[NW];
  int cnt[NW];
  float acc[NW][kAccStride];
};

// Where a key's rows are: page * page_size + offset in it, or -1.
__device__ __forceinline__ int slot_of(const CacheAttnParams& p, int b, int key) {
  const int col = key >> p.c.page_shift;
  const int pg = col < p.cols ? p.table[size_t(b) * p.cols + col] : -1;
  return pg >= 0 && pg < p.c.pages ? (pg << p.c.page_shift) + (key & (p.c.page - 1)) : -1;
}

// Adds p_j v_j of the wave's listed keys to the lane's 8 channels: kCl lanes
// have a row's octets, so DEEP loads in flight take DEEP * 64 / kCl entries.
template <int NG, int DEEP>
struct ValueSum {
  static constexpr int kCl = NG == 3 ? 16 : 4 * NG, kPer = kWave / kCl, kDeep = DEEP, kStep = kDeep * kPer;
  float acc[8] = {};
  float off = 0.0f;
  uint32_t w[kDeep], pr[kDeep];
  // entries e0 .. of a list of slots (slot_of; -1: no row)
  __device__ __forceinline__ void load(const CacheAttnParams& p, int h, const int* pi, int e0, int n, int lane) {
    const int c = lane & (kCl - 1), slot = lane / kCl, g = c >> 2;
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      const int e = e0 + u * kPer + slot;
      const int at = e < n && g < NG ? pi[e] : -1;
      w[u] = pr[u] = 0u;
      if (at >= 0) {
        const size_t row = (size_t(at >> p.c.page_shift) * p.c.heads + h) * p.c.page + (at & (p.c.page - 1));
        w[u] = reinterpret_cast<const uint32_t*>(p.c.v_codes)[row * (4 * NG) + c];
        pr[u] = p.c.v_params[row * NG + g];
      }
    }
  }
  // weights pz[e] of the entries that load was given
  __device__ __forceinline__ void use(const float* pz, int e0, int n, int lane) {
    const int slot = lane / kCl;
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      const int e = e0 + u * kPer + slot;
      const float pj = e < n ? pz[e] : 0.0f;
      const float ps = pj * __uint_as_float(pr[u] << 16);
      off = fmaf(pj, __uint_as_float(pr[u] & 0xffff0000u), off);
      const uint32_t even = w[u] & 0x0f0f0f0fu, odd = (w[u] >> 4) & 0x0f0f0f0fu;
      for (int j = 0; j < 4; ++j) {
        acc[2 * j] = fmaf(ps, float((even >> (8 * j)) & 255u), acc[2 * j]);
        acc[2 * j + 1] = fmaf(ps, float((odd >> (8 * j)) & 255u), acc[2 * j + 1]);
      }
    }
  }
  __device__ __forceinline__ void add(const CacheAttnParams& p, int h, const float* pz, const int* pi, int n,
                                      int lane) {
    ValueSum next;  // its loads: a step ahead of the sums
    if (n > 0) next.load(p, h, pi, 0, n, lane);
    for (int e0 = 0; e0 < n; e0 += kStep) {
#pragma unroll
      for (int u = 0; u < kDeep; ++u) w[u] = next.w[u], pr[u] = next.pr[u];
      if (e0 + kStep < n) next.load(p, h, pi, e0 + kStep, n, lane);
      use(pz, e0, n, lane);
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

// tau and the output of row `row` (of the key head's R) from its dots (key j at
// sp[j / 64 * gstep + j % 64], where its granule may hold a weight) and its
// granule maxima gp, by `size` waves of the block from wave w0 on.  Every
// wave of the block calls it together (teams meet at the block's barriers);
// row = -1, vis = 0 for a team without a row.  WHOLE: the team is the block.
// The Newton steps are a team's first wave's: the same steps on every wave
// would share the SIMDs with one another.  Meanwhile the others load the
// values of their candidates.
template <typename T, int NG, int PC, int NW, bool WHOLE, typename Lds>
__device__ __forceinline__ void finish_row(const CacheAttnParams& p, int b, int h, int row, int vis,
                                           const float* gp, const float* sp, int gstep, Lds& L, int w, int w0,
                                           int size, int lane) {
  constexpr int kCap = Lds::kCap;
  const int member = w - w0;
  const float e = p.e;
  const ZOf zof(p);

  // ---- the largest z, and a bound below tau from the granules' ----
  // granule i is member i % size's
  const int ng = (vis + kGranule - 1) / kGranule;
  const int g0 = lane * size + member;
  constexpr int kHeld = WHOLE ? 4 : 1;  // granules of a lane whose maxima stay in registers
  constexpr int kDeep = WHOLE ? 8 : 4;  // loads in flight of a wave: global memory, LDS
  float held[kHeld];
#pragma unroll
  for (int c = 0; c < kHeld; ++c) {
    const int i = g0 + c * size * kWave;
    held[c] = i < ng ? gp[i] : kHidden;
  }
#pragma unroll
  for (int c = 0; c < kHeld; ++c) held[c] = zof(held[c]);
  float g = held[0];
#pragma unroll
  for (int c = 1; c < kHeld; ++c) g = fmaxf(g, held[c]);
  for (int i = g0 + kHeld * size * kWave; i < ng; i += size * kWave) g = fmaxf(g, zof(gp[i]));
  L.gm[w][lane] = g;
  __syncthreads();
  if (member == 0) {
    float gz[4] = {kHidden, kHidden, kHidden, kHidden};
    for (int i = 0; i < size; i += 4)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < size) gz[k] = fmaxf(gz[k], L.gm[w + i + k][lane]);
    const float zm = wave_max(fmaxf(fmaxf(gz[0], gz[1]), fmaxf(gz[2], gz[3])));
    float t = zm - 1.0f, lo = t, hi = zm;
    if (ng > 1 && zm > 0.5f * kHidden) {
      // a few steps: any tau left of the root of the maxima will do, and near
      // the root a step drops few candidates
      for (int it = 0; it < 12; ++it) {
        float F = 0.0f, F1 = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float pa, pa1;
          powers<PC>(fmaxf(gz[k] - t, 0.0f), e, pa, pa1);
          F += pa;
          F1 += pa1;
        }
        wave_sum2(F, F1);
        if (F < 1.5f && p.alpha <= 2.0f) break;
        if (next_tau(p.alpha, F, F1, t, lo, hi)) break;
      }
      // less the rounding of the steps, and of F at them
      lo = fmaxf((p.alpha <= 2.0f ? t : lo) - 4e-6f, zm - 1.0f);
    }
    if (lane == 0) {
      L.say[w][0] = zm;
      L.say[w][1] = lo;
    }
  }
  __syncthreads();
  const float zmax = L.say[w0][0];
  const bool empty = !(zmax > 0.5f * kHidden);
  float lo = L.say[w0][1], tau = lo, hi = zmax;

  // ---- the keys with z > lo, listed; lo moves up while they do not fit ----
  bool listed = false, dense = empty;
  int most = 0, mine = 0;  // the longest of the team's lists
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
      for (int i0 = 0; i0 < ng; i0 += kHeld * size * kWave) {
#pragma unroll
        for (int c = 0; c < kHeld; ++c) {
          const int i1 = i0 + c * size * kWave;
          // the granules to look at, as a mask of the lanes that have them
          uint64_t todo = __ballot((i0 ? (i1 + g0 < ng ? zof(gp[i1 + g0]) : kHidden) : held[c]) > lo);
          while (todo) {
            constexpr int kLook = 2 * kDeep;
            const int cnt = __builtin_popcountll(todo);
            float d[kLook];
            int key[kLook];
#pragma unroll
            for (int k = 0; k < kLook; ++k) {
              const int l = todo ? __builtin_ctzll(todo) : -1;
              todo &= todo - 1;
              const int gi = l < 0 ? 0 : i1 + l * size + member;
              key[k] = l < 0 ? vis : gi * kGranule + lane;
              d[k] = kHidden;
              if (l >= 0) d[k] = sp[size_t(gi) * gstep + lane];
            }
#pragma unroll
            for (int k = 0; k < kLook; ++k) {
              if (k >= cnt) break;
              collect(d[k], key[k]);
            }
          }
        }
      }
      if (lane == 0) L.cnt[w] = mine;
    }
    __syncthreads();
    if (!listed && !dense) {
      most = 0;
      for (int i = 0; i < size; ++i) most = max(most, L.cnt[w0 + i]);
      listed = most <= kCap;
    }
    if (!__syncthreads_or(!listed && !dense)) break;
    // some team's candidates did not fit: one step of its tau over the whole row
    float F = 0.0f, F1 = 0.0f;
    if (!listed && !dense) {
#pragma unroll 4
      for (int i = member; i < ng; i += size) {
        const int j = i * kGranule + lane;
        const bool in = j < vis && zof(gp[i]) > lo;  // the others hold no dots
        float pa, pa1;
        powers<PC>(fmaxf(in ? zof(sp[size_t(i) * gstep + lane]) - tau : 0.0f, 0.0f), e, pa, pa1);
        F += pa;
        F1 += pa1;
      }
      wave_sum2(F, F1);
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

  // ---- tau over the lists ----
  using Values = ValueSum<NG, kDeep>;
  Values vs;
  const bool few = listed && mine <= Values::kStep;
  if (few) {
    for (int j = lane; j < mine; j += kWave) L.ci[w][j] = slot_of(p, b, L.ci[w][j]);
    vs.load(p, h, L.ci[w], 0, mine, lane);
  }
  float total = 0.0f;
  if (WHOLE && listed && most > kWave) {  // each wave its own
    tau = lo;
    for (int it = 0; it <= kMaxSteps; ++it) {
      float F = 0.0f, F1 = 0.0f;
#pragma unroll 2
      for (int j = lane; j < mine; j += kWave) {
        float pa, pa1;
        powers<PC>(fmaxf(L.cz[w][j] - tau, 0.0f), e, pa, pa1);
        F += pa;
        F1 += pa1;
      }
      wave_sum2(F, F1);
      if (lane == 0) {
        L.red[it & 1][w][0] = F;
        L.red[it & 1][w][1] = F1;
      }
      __syncthreads();
      F = lane < NW ? L.red[it & 1][lane][0] : 0.0f;
      F1 = lane < NW ? L.red[it & 1][lane][1] : 0.0f;
      wave_sum2(F, F1);
      total = F;
      if (next_tau(p.alpha, F, F1, tau, lo, hi)) break;
    }
    __syncthreads();
  } else {
    if (listed && member == 0) {
      float t = lo;
      auto steps = [&](auto sums) {
        for (int it = 0; it <= kMaxSteps; ++it) {
          float F = 0.0f, F1 = 0.0f;
          sums(t, F, F1);
          wave_sum2(F, F1);
          total = F;
          if (next_tau(p.alpha, F, F1, t, lo, hi)) break;
        }
      };
      if (most <= kWave) {  // a register for each wave's list
        float z[NW];
        int cnt[NW];
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          const int j = i < size ? w + i : w;
          cnt[i] = L.cnt[j];
          z[i] = L.cz[j][lane];
        }
#pragma unroll
        for (int i = 0; i < NW; ++i) z[i] = i < size && lane < cnt[i] ? z[i] : kHidden;
        steps([&](float at, float& F, float& F1) {
#pragma unroll
          for (int i = 0; i < NW; ++i) {
            float pa, pa1;
            powers<PC>(fmaxf(z[i] - at, 0.0f), e, pa, pa1);
            F += pa;
            F1 += pa1;
          }
        });
      } else {
        steps([&](float at, float& F, float& F1) {
          for (int i = 0; i < size; ++i)
            for (int j = lane; j < L.cnt[w + i]; j += kWave) {
              float pa, pa1;
              powers<PC>(fmaxf(L.cz[w + i][j] - at, 0.0f), e, pa, pa1);
              F += pa;
              F1 += pa1;
            }
        });
      }
      if (lane == 0) {
        L.say[w][2] = t;
        L.say[w][3] = total;
      }
    }
    __syncthreads();
    if (listed) {
      tau = L.say[w0][2];
      total = L.say[w0][3];
    }
  }

  // ---- the support's weights and values ----
  float psum = 0.0f;
  if (few) {
    for (int j = lane; j < mine; j += kWave) {
      const float pa = weight<T, PC>(fmaxf(L.cz[w][j] - tau, 0.0f), e);
      L.cz[w][j] = pa;
      psum += pa;
    }
    vs.use(L.cz[w], 0, mine, lane);
  } else if (!empty) {
    // the wave's candidates, or its keys of the row, kCap at a time
    const int part = listed ? mine : kCap, end = listed ? mine : vis;
    for (int k0 = listed ? 0 : member * part; k0 < end; k0 += size * part) {
      const int cnt = min(part, end - k0);
      int c = 0;
#pragma unroll 2
      for (int j0 = 0; j0 < cnt; j0 += kWave) {
        const int j = j0 + lane;
        float zj = kHidden;
        int slot = -1;
        if (j < cnt) {
          const int gi = (k0 + j) / kGranule;
          zj = listed ? L.cz[w][j] : zof(gp[gi]) > lo ? zof(sp[size_t(gi) * gstep + (k0 + j) % kGranule]) : kHidden;
          if (zj > tau) slot = slot_of(p, b, listed ? L.ci[w][j] : k0 + j);
        }
        const float pa = weight<T, PC>(fmaxf(zj - tau, 0.0f), e);
        const uint64_t msk = __ballot(pa > 0.0f);
        if (pa > 0.0f) {
          const int at = c + lane_rank(msk);  // at most j: already read
          L.cz[w][at] = pa;
          L.ci[w][at] = slot;
        }
        c += __builtin_popcountll(msk);
        psum += pa;
      }
      vs.add(p, h, L.cz[w], L.ci[w], c, lane);
    }
  }
  vs.reduce();
  if (lane < Values::kCl && lane < 4 * NG)
    for (int j = 0; j < 8; ++j) L.acc[w][8 * lane + j] = vs.acc[j];
  // the steps' last sum is that of the weights, unless those are the library's
  // or no list was summed
  const bool resum = !listed || (PC != kE2 && std::is_same<T, float>::value);
  if (resum) {
    psum = wave_sum(psum);
    if (lane == 0) L.psum[w] = psum;
  }
  __syncthreads();
  if (row >= 0) {
    if (resum) {
      total = 0.0f;
      for (int i = 0; i < size; ++i) total += L.psum[w0 + i];
    }
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
constexpr int kRowKeys = 8192;  // split plan: rows up to this have 4 waves, else 8 or 16

// One block per tile of rows of a key head: dots into LDS, then its rows.
template <typename T, int P, int NG, int PC>
__global__ __launch_bounds__(kOneWaves * kWave) void cache_one_kernel(CacheAttnParams p, int stride) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  constexpr int NW = kOneWaves;
  __shared__ TeamLds<NW, 128> L;
  constexpr int kR = kTile / P;
  const int t = threadIdx.x, w = t >> 6, lane = t & 63;
  const int nrt = (p.R + kR - 1) / kR;
  const int tile = blockIdx.x % nrt, bh = blockIdx.x / nrt;
  const int b = bh / p.c.heads, h = bh % p.c.heads;
  const int r0 = tile * kR, rows = min(kR, p.R - r0), most = min(kR, p.R), gs = stride / kGranule;
  int pad = 1;
  while (pad < most && pad < NW) pad *= 2;
  float* zs = reinterpret_cast<float*>(smem);
  float* gs0 = zs + most * stride;  // granule maxima
  int* pages = reinterpret_cast<int*>(gs0 + most * gs);
  stage_pages(p, b, 0, p.maxlen, pages, t, NW * kWave);
  __shared__ QueryLds<T, P, NG> ql;
  static_assert(sizeof(L) + sizeof(ql) <= kCacheOneStatic, "the plan's bound");
  stage_query<T, P, NG>(p, ql, b, h, r0, w, NW, lane);
  {
    TileRows<P> rt;
    rt.load(p, b, r0, lane);
    __syncthreads();
    score_keys<NW, false>(p, ql, rt, h, 0, rt.most, pages, most, zs, gs0, gs, w, lane);
  }
  __syncthreads();
  const int size = NW / pad, team = w / size, w0 = team * size;
  for (int first = 0; first < rows; first += pad) {
    const int r = first + team;
    const bool has = r < rows;
    finish_row<T, NG, PC, NW, false>(p, b, h, has ? r0 + r : -1, has ? visible_keys(p, b, (r0 + r) % p.NQ) : 0,
                                        gs0 + (has ? r : 0) * gs, zs + (has ? r : 0) * kGranule, most * kGranule, L, w,
                                        w0, size, lane);
  }
}

// Split plan, first launch: dots of `span` keys with a tile of rows, and
// their granules' maxima.
template <typename T, int P, int NG>
__global__ __launch_bounds__(kScoreWaves * kWave, 4) void cache_score_kernel(CacheAttnParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  constexpr int kR = kTile / P;
  int* pages = reinterpret_cast<int*>(smem);
  __shared__ QueryLds<T, P, NG> ql;
  const int t = threadIdx.x, w = t >> 6, lane = t & 63;
  const int nrt = (p.R + kR - 1) / kR;
  const int split = blockIdx.x % p.nsplit, rest = blockIdx.x / p.nsplit;
  const int tile = rest % nrt, bh = rest / nrt;
  const int b = bh / p.c.heads, h = bh % p.c.heads;
  const int r0 = tile * kR;
  const int key0 = split * p.span;
  stage_pages(p, b, key0, min(p.span, p.maxlen - key0), pages, t, kScoreWaves * kWave);
  stage_query<T, P, NG>(p, ql, b, h, r0, w, kScoreWaves, lane);
  TileRows<P> rt;
  rt.load(p, b, r0, lane);
  if (key0 >= rt.most) return;  // block-uniform
  __syncthreads();
  const int rows = min(kR, p.R);
  const size_t gs = size_t(p.span / kGranule) * p.nsplit, row0 = (size_t(bh) * nrt + tile) * rows;
  score_keys<kScoreWaves, true>(p, ql, rt, h, key0, min(key0 + p.span, rt.most), pages, rows,
                                p.scores + row0 * gs * kGranule, p.gmax + row0 * gs, gs, w, lane);
}

// Split plan, second launch: one block per row.
template <typename T, int NG, int PC, int NW>
__global__ __launch_bounds__(NW * kWave) void cache_row_kernel(CacheAttnParams p) {
  __shared__ TeamLds<NW, 512> L;
  const int t = threadIdx.x, w = t >> 6, lane = t & 63;
  const int row = blockIdx.x % p.R, bh = blockIdx.x / p.R;
  const int b = bh / p.c.heads, h = bh % p.c.heads;
  // the score blocks' tiles of `rows` rows
  const int rows = min(p.tile_rows, p.R), nrt = (p.R + rows - 1) / rows, tile = row / rows, r = row % rows;
  const size_t gs = size_t(p.span / kGranule) * p.nsplit, row0 = (size_t(bh) * nrt + tile) * rows;
  finish_row<T, NG, PC, NW, true>(p, b, h, row, visible_keys(p, b, row % p.NQ), p.gmax + (row0 + r) * gs,
                              p.scores + row0 * gs * kGranule + r * kGranule, rows * kGranule, L, w, 0, NW, lane);
}

template <typename K> hipError_t allow_lds(K kern, size_t lds) {
  if (lds + kCacheOneStatic <= 65536) return hipSuccess;
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                             int(lds));
}

template <typename T, int P, int NG>
hipError_t launch_png(const CacheAttnParams& p, hipStream_t s) {
  const int nrt = (p.R + kTile / P - 1) / (kTile / P);
  if (p.plan == kCacheOneBlock) {
    int stride = 0;
    const size_t lds = cache_one_lds(p, &stride);
    auto kern = p.pc == kE2 ? cache_one_kernel<T, P, NG, kE2> : cache_one_kernel<T, P, NG, kEGen>;
    if (hipError_t e = allow_lds(kern, lds)) return e;
    profile_begin("cache_attn", s);
    hipLaunchKernelGGL(kern, dim3(unsigned(p.B) * p.c.heads * nrt), dim3(kOneWaves * kWave), lds, s, p,
                       stride);
    profile_end(s);
    return hipGetLastError();
  }
  profile_begin("cache_score", s);
  hipLaunchKernelGGL((cache_score_kernel<T, P, NG>), dim3(unsigned(p.B) * p.c.heads * nrt * p.nsplit),
                     dim3(kScoreWaves * kWave), size_t(p.span / p.c.page + 1) * 4, s, p);
  profile_end(s);
  return hipGetLastError();
}

template <typename T, int NG, int PC>
hipError_t launch_rows(const CacheAttnParams& p, hipStream_t s) {
  const dim3 grid(unsigned(p.B) * p.c.heads * p.R);
  profile_begin("cache_row", s);
  if (p.maxlen <= kRowKeys) hipLaunchKernelGGL((cache_row_kernel<T, NG, PC, 4>), grid, dim3(4 * kWave), 0, s, p);
  else if (grid.x > 256) hipLaunchKernelGGL((cache_row_kernel<T, NG, PC, 8>), grid, dim3(8 * kWave), 0, s, p);
  else hipLaunchKernelGGL((cache_row_kernel<T, NG, PC, 16>), grid, dim3(16 * kWave), 0, s, p);
  profile_end(s);
  return hipGetLastError();
}

template <typename T, int NG>
hipError_t launch_ng(const CacheAttnParams& p, hipStream_t s) {
  hipError_t e = hipSuccess;
  if constexpr (std::is_same<T, float>::value) {
    e = p.tile_rows > 8 ? launch_png<T, 1, NG>(p, s) : launch_png<T, 2, NG>(p, s);
  } else {
    const int P = kTile / p.tile_rows;
    e = P == 1 ? launch_png<T, 1, NG>(p, s) : P == 2 ? launch_png<T, 2, NG>(p, s) : launch_png<T, 4, NG>(p, s);
  }
  if (e != hipSuccess || p.plan == kCacheOneBlock) return e;
  return p.pc == kE2 ? launch_rows<T, NG, kE2>(p, s) : launch_rows<T, NG, kEGen>(p, s);
}

template <typename T>
hipError_t launch_cache_attn_t(const CacheAttnParams& p, hipStream_t s) {
  switch (p.c.G) {
    case 1: return launch_ng<T, 1>(p, s);
    case 2: return launch_ng<T, 2>(p, s);
    case 3: return launch_ng<T, 3>(p, s);
    default: return launch_ng<T, 4>(p, s);
  }
}

}  // namespace

}  // namespace asa
