// Writing tokens into the 4-bit key/value cache, and reading rows of it back.
//
// Both are one pass over the data: a thread has 8 channels of one row, the
// four threads of a quad one channel group, so the group's minimum and
// maximum are two DPP exchanges and no data moves through LDS.  Each thread
// takes the key row and the value row of its token (two independent loads in
// flight).
#include <type_traits>

#include "asa_cache.hpp"
#include "asa_device.hpp"

namespace asa {
namespace {

constexpr int kThreads = 256;

// Values at or past this bound are taken as the bound (NaN as 0), so that a
// group's range and scale are finite.
constexpr float kMostCached = 0x1p126f;

// 8 consecutive channels from `src` as floats; channels at or past `nv` give 0.
template <typename T, bool CHUNKS>
__device__ __forceinline__ void load8(const T* src, int nv, float* x) {
  if constexpr (CHUNKS) {
    if constexpr (std::is_same<T, float>::value) {
      const float4 a = *reinterpret_cast<const float4*>(src);
      const float4 b = *reinterpret_cast<const float4*>(src + 4);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
      x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(src);
      T e[8];
      __builtin_memcpy(e, &u, 16);
      for (int j = 0; j < 8; ++j) x[j] = Elem<T>::load(e + j);
    }
  } else {
    for (int j = 0; j < 8; ++j) x[j] = j < nv ? Elem<T>::load(src + j) : 0.0f;
  }
}

// Values read back are stored past the caches: most of a read's bytes are its
// results, and a batch of contexts is larger than the caches (8 x 8191, 268 MB
// of results: 59.6 -> 44.9 us, 7.0 TB/s with the reads; a 16k prompt written
// and read 39.7 -> 32.7; 17 MB unchanged).
template <typename T, bool CHUNKS>
__device__ __forceinline__ void store8(T* dst, int nv, const float* x) {
  if constexpr (CHUNKS) {
    if constexpr (std::is_same<T, float>::value) {
      __builtin_nontemporal_store(f32x4{x[0], x[1], x[2], x[3]}, reinterpret_cast<f32x4*>(dst));
      __builtin_nontemporal_store(f32x4{x[4], x[5], x[6], x[7]}, reinterpret_cast<f32x4*>(dst + 4));
    } else {
      typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
      T e[8];
      for (int j = 0; j < 8; ++j) Elem<T>::store(e + j, x[j]);
      u32x4 u;
      __builtin_memcpy(&u, e, 16);
      __builtin_nontemporal_store(u, reinterpret_cast<u32x4*>(dst));
    }
  } else {
    for (int j = 0; j < 8; ++j)
      if (j < nv) Elem<T>::store(dst + j, x[j]);
  }
}

// The exact value of a - b as an unevaluated sum hi + lo.
__device__ __forceinline__ void two_diff(float a, float b, float& hi, float& lo) {
  hi = a - b;
  const float t = hi - a;
  lo = (a - (hi - t)) - (b + t);
}

// The codes (nibble j of dword i: channel 8 i + j) and the group's params of N
// channels x, of which nv belong to the row (FULL: all).  Called by whole
// quads (N = 8) or pairs (N = 16): the lanes of a group.
template <int N, bool FULL>
__device__ __forceinline__ void quantise(float* x, int nv, uint32_t& params, uint32_t* codes) {
  bool wild = false;
  for (int j = 0; j < N; ++j) wild |= !(fabsf(x[j]) <= kMostCached);
  if (wild)
    for (int j = 0; j < N; ++j)
      x[j] = x[j] == x[j] ? fminf(fmaxf(x[j], -kMostCached), kMostCached) : 0.0f;
  float lo = __builtin_inff(), hi = -__builtin_inff();
  for (int j = 0; j < N; ++j)
    if (FULL || j < nv) {
      lo = fminf(lo, x[j]);
      hi = fmaxf(hi, x[j]);
    }
  lo = fminf(lo, __uint_as_float(lane_xor<1>(__float_as_uint(lo))));
  hi = fmaxf(hi, __uint_as_float(lane_xor<1>(__float_as_uint(hi))));
  if constexpr (N == 8) {
    lo = fminf(lo, __uint_as_float(lane_xor<2>(__float_as_uint(lo))));
    hi = fmaxf(hi, __uint_as_float(lane_xor<2>(__float_as_uint(hi))));
  }
  if constexpr (!FULL)
    for (int j = 0; j < N; ++j) x[j] = j < nv ? x[j] : lo;  // code 0 or 1, cleared below
  // m: towards zero in the bits, one step further down for a cut negative
  const uint32_t lb = __float_as_uint(lo);
  const uint32_t mb = (lb & 0xffff0000u) + (lo < 0.0f && (lb & 0xffffu) ? 0x10000u : 0u);
  const float m = __uint_as_float(mb);
  // s: 15 s has 12 significant bits, so the comparison with the exact
  // max - m = d + dl is exact; the estimate is at most two steps low
  float d, dl;
  two_diff(hi, m, d, dl);
  uint32_t sb = 0u;
  if (d > 0.0f) {
    sb = __float_as_uint(fmaxf(d * (1.0f / 15.0f), 0x1p-126f)) & 0xffff0000u;
    for (int i = 0; i < 2; ++i) {
      const float t = 15.0f * __uint_as_float(sb);
      if (t < d || (t == d && dl > 0.0f)) sb += 0x10000u;
    }
  }
  const float s = __uint_as_float(sb);
  params = (sb >> 16) | mb;
  // c: y is near (x - m) / s, so one of the borders on either side of
  // floor(y) + 1/2 is the only one in doubt, and an exact comparison with it
  // settles the code whatever y was rounded to.
  const float r = sb ? __builtin_amdgcn_rcpf(s) : 0.0f;
  const float nm = -m * r;
  // m + (k + 1/2) s: m is a multiple of 2^-7 of its power of two and the rest
  // of 2^-8 of s's, so between |m| = 2^-8 s and 2^12 s the sum spans at most
  // 22 bits and the fused product rounds nothing.
  const float am = fabsf(m);
  if (am == 0.0f || (am >= 0x1p-8f * s && am <= 0x1p12f * s)) {
    for (int i = 0; i < N / 8; ++i) {
      // four codes at a time gather in a float (16 bits, exact)
      float half[2];
      for (int q = 0; q < 2; ++q) {
        float acc = 0.0f;
        for (int j = 3; j >= 0; --j) {
          const float v = x[8 * i + 4 * q + j];
          const float k = floorf(fmaf(v, r, nm)), k5 = k + 0.5f;
          acc = fmaf(acc, 16.0f, v > fmaf(k5, s, m) ? k5 + 0.5f : k);
        }
        half[q] = acc;
      }
      codes[i] = uint32_t(half[0]) | (uint32_t(half[1]) << 16);
    }
  } else {
    for (int i = 0; i < N / 8; ++i) {
      uint32_t w = 0u;
      for (int j = 7; j >= 0; --j) {
        float t, tl;
        two_diff(x[8 * i + j], m, t, tl);
        const float k = fminf(fmaxf(floorf(t * r), 0.0f), 15.0f);
        const float border = (k + 0.5f) * s;
        const int c = int(k) + (t > border || (t == border && tl > 0.0f) ? 1 : 0);
        w = (w << 4) | uint32_t(c > 15 ? 15 : c);
      }
      codes[i] = w;
    }
  }
  if constexpr (!FULL)
    if (nv < 8) codes[0] = nv <= 0 ? 0u : codes[0] & (0xffffffffu >> (4 * (8 - nv)));
}

// N = 16: rows are whole channel groups of 16-byte chunks, and a thread has
// half a group; N = 8: a quarter, whatever the row.
template <typename T, int N, bool CHUNKS>
__global__ __launch_bounds__(kThreads) void cache_write_kernel(CacheRowsParams p, int lanes_shift, int nblk) {
  constexpr bool kFull = N == 16;
  constexpr int kPer = 32 / N;  // threads of a group
  const int bh = blockIdx.x / nblk, b = bh / p.c.heads, h = bh % p.c.heads;
  const int t = (blockIdx.x - bh * nblk) * kThreads + threadIdx.x;
  const int i = t >> lanes_shift, l = t & ((1 << lanes_shift) - 1);
  const int g = l / kPer, o = l % kPer * (N / 8);  // group, first octet
  const int count = p.limit ? min(p.limit[b], p.n) : p.n;
  if (i >= count || g >= p.c.G) return;  // whole groups leave together
  const int64_t pos = int64_t(p.start ? p.start[b] : 0) + i;
  if (pos < 0 || pos >= (int64_t(1) << 31)) return;
  const int64_t row = cache_row(p.c, p.table + size_t(b) * p.cols, p.cols, int(pos), h);
  if (row < 0) return;
  const int ch = 32 * g + 8 * o, nv = p.c.hd - ch;
  const T* k = static_cast<const T*>(p.k) + size_t(b) * p.lk.sb + size_t(h) * p.lk.sh + size_t(i) * p.lk.sn + ch;
  const T* v = static_cast<const T*>(p.v) + size_t(b) * p.lv.sb + size_t(h) * p.lv.sh + size_t(i) * p.lv.sn + ch;
  float xk[N] = {}, xv[N] = {};
  if (kFull || nv > 0)  // rows that end inside the group: its last octets have no channels
    for (int q = 0; q < N; q += 8) {
      load8<T, CHUNKS>(k + q, nv, xk + q);
      load8<T, CHUNKS>(v + q, nv, xv + q);
    }
  uint32_t pk, pv, wk[N / 8], wv[N / 8];
  quantise<N, kFull>(xk, nv, pk, wk);
  quantise<N, kFull>(xv, nv, pv, wv);
  const int G = p.c.G;
  uint32_t* kc = reinterpret_cast<uint32_t*>(p.c.k_codes) + row * (4 * G) + G * o + g;
  uint32_t* vc = reinterpret_cast<uint32_t*>(p.c.v_codes) + row * (4 * G) + 4 * g + o;
  for (int q = 0; q < N / 8; ++q) {
    kc[G * q] = wk[q];
    vc[q] = wv[q];
  }
  if (o == 0) {
    p.c.k_params[row * G + g] = pk;
    p.c.v_params[row * G + g] = pv;
  }
}

// m + c s, rounded once: c s has 12 bits, the fused sum one rounding.
__device__ __forceinline__ void values8(uint32_t w, uint32_t params, float* x) {
  const float s = __uint_as_float(params << 16), m = __uint_as_float(params & 0xffff0000u);
  for (int j = 0; j < 8; ++j) x[j] = fmaf(float((w >> (4 * j)) & 15u), s, m);
}

template <typename T, bool CHUNKS>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(CacheRowsParams p, int lanes_shift, int nblk) {
  const int bh = blockIdx.x / nblk, b = bh / p.c.heads, h = bh % p.c.heads;
  const int t = (blockIdx.x - bh * nblk) * kThreads + threadIdx.x;
  const int i = t >> lanes_shift, l = t & ((1 << lanes_shift) - 1);
  const int g = l >> 2, o = l & 3;
  if (i >= p.n || g >= p.c.G) return;
  const int ch = 32 * g + 8 * o, nv = p.c.hd - ch;
  if (nv <= 0) return;
  const int64_t pos = int64_t(p.start ? p.start[b] : 0) + i;
  const int G = p.c.G;
  int64_t row = -1;
  if (pos >= 0 && pos < p.limit[b])
    row = cache_row(p.c, p.table + size_t(b) * p.cols, p.cols, int(pos), h);
  float xk[8] = {}, xv[8] = {};
  if (row >= 0) {
    const uint32_t wk = reinterpret_cast<const uint32_t*>(p.c.k_codes)[row * (4 * G) + G * o + g];
    const uint32_t wv = reinterpret_cast<const uint32_t*>(p.c.v_codes)[row * (4 * G) + 4 * g + o];
    const uint32_t pk = p.c.k_params[row * G + g], pv = p.c.v_params[row * G + g];
    values8(wk, pk, xk);
    values8(wv, pv, xv);
  }
  const size_t at = (size_t(bh) * p.n + i) * p.c.hd + ch;
  store8<T, CHUNKS>(static_cast<T*>(p.ok) + at, nv, xk);
  store8<T, CHUNKS>(static_cast<T*>(p.ov) + at, nv, xv);
}

template <typename T>
hipError_t launch_rows(const CacheRowsParams& p, bool write, hipStream_t s) {
  // threads of a row, rounded up to a power of two: 2 or 4 per channel group
  const bool halves = write && p.chunks && p.c.hd % 32 == 0;
  const int sh = (p.c.G > 2 ? 4 : p.c.G > 1 ? 3 : 2) - (halves ? 1 : 0);
  const long long threads = (long long)p.n << sh;
  const long long nblk = (threads + kThreads - 1) / kThreads;
  const long long blocks = nblk * p.B * p.c.heads;
  if (threads >= (1LL << 31) || blocks >= (1LL << 31)) return hipErrorInvalidConfiguration;
  const dim3 grid{unsigned(blocks)}, block(kThreads);
  if (write) {
    if (halves) hipLaunchKernelGGL((cache_write_kernel<T, 16, true>), grid, block, 0, s, p, sh, int(nblk));
    else if (p.chunks) hipLaunchKernelGGL((cache_write_kernel<T, 8, true>), grid, block, 0, s, p, sh, int(nblk));
    else hipLaunchKernelGGL((cache_write_kernel<T, 8, false>), grid, block, 0, s, p, sh, int(nblk));
  } else {
    if (p.chunks) hipLaunchKernelGGL((cache_read_kernel<T, true>), grid, block, 0, s, p, sh, int(nblk));
    else hipLaunchKernelGGL((cache_read_kernel<T, false>), grid, block, 0, s, p, sh, int(nblk));
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_cache_write(const CacheRowsParams& p, int dtype, hipStream_t s) {
  if (dtype == kElemBF16) return launch_rows<u16>(p, true, s);
  if (dtype == kElemF16) return launch_rows<h16>(p, true, s);
  return launch_rows<float>(p, true, s);
}

hipError_t launch_cache_read(const CacheRowsParams& p, int dtype, hipStream_t s) {
  if (dtype == kElemBF16) return launch_rows<u16>(p, false, s);
  if (dtype == kElemF16) return launch_rows<h16>(p, false, s);
  return launch_rows<float>(p, false, s);
}

}  // namespace asa
