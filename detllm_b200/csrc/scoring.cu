// scoring.cu -- what a row of logits says about tokens: the log probability
// of a given token, the row's entropy and its most likely tokens, and how far
// a student's row is from a teacher's top list; with the gradients of both.
//
//   m = max x, d_j = (x_j - m) / T, S = sum exp(d_j), S1 = sum exp(d_j) d_j
//   log p_j = d_j - log S          H = log S - S1 / S
//   loss = sum_i q_i (log q_i - log p_id(i)),  q = softmax(u / T)
//   d log p_t / dx_j = [j = t] - p_j
//   dH / dx_j        = -p_j (log p_j + H) = -p_j (d_j - S1 / S)
//   d loss / dx_j    = (p_j - sum_{i: id(i) = j} q_i) / T
//
// An entry of -inf is masked out: exp(-inf) = 0 and 0 * -inf counts as 0.
//
// Arithmetic: every f32 operation is rounded on its own, as in the rest of
// the library, and the order of every sum is fixed by the vocabulary alone,
// so a row has the same bits whatever batch, stride or call it is part of.
// A row is cut into segments of 2,048 entries; a warp takes a segment, its
// lane l the entries of 16-byte vectors l, l + 32, ... of it, and sums are
// relative to the segment's own maximum until the segments are joined.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstring>
#include <map>
#include <mutex>
#include <set>
#include <tuple>
#include <type_traits>

#include "../../include/detgpu.h"
#include "dev_math.cuh"
#include "internal.h"

namespace det {
namespace {

constexpr int kSeg = 2048;                       // entries per segment
constexpr int kPerLane = kSeg / 32;              // entries per lane of a segment
constexpr uint32_t kMaxVocab = 1u << 18;         // as the CDF's alphabet
constexpr int kMaxSegs = (int)(kMaxVocab / kSeg);
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kFull = 0xffffffffu;

// ---- packed f32 pairs ----------------------------------------------------------
using f2 = unsigned long long;
DI f2 pk(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
DI float2 un(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
DI f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
DI f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
DI f2 fma2(unsigned long long a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// c + p where p is a product: written p * 1 + c, which is exact in its
// multiply and rounds once, like the add; `one` is 1.0 at run time, so the
// compiler cannot contract the multiply that made p into the add.
DI f2 addp(f2 p, f2 one, f2 c) { return fma2(p, one, c); }  // exact multiply

DI float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^y for y <= 0, two at a time, after Tang's table-driven method: y = k + i/32
// + f with |f| <= 1/64 (a rounding to a multiple of 1/32 by adding 1.5 * 2^18);
// 2^f as a square, A ((f + B)^2 + D), where B = 46/32 is near 1 / ln 2 and a
// multiple of 1/32, so f + B is one addition (maximal relative error 3.6 *
// 2^-24 with A and D for it that make 2^0 exactly 1; 0.9 with the best B,
// which takes two operations more); A 2^(i/32) from a table of 32 that a warp
// holds one entry per lane and reads with a shuffle (no two lanes conflict);
// 2^k added to the entry's exponent field.  11 rounded f32 operations for an
// entry of a row with its two sums, against 19 for a degree-5 polynomial on
// |f| <= 1/2: issue slots (two for a packed operation) bound the passes over
// 16-bit logits.
// Within 7.1 * 2^-24 of 2^y where that is 2^-122 or more, and 0 below 2^-123.
// NaN gives an unspecified number: callers keep y, which stays NaN, beside it.
constexpr float kYLow = -127.5f;
constexpr float kLog2e = 1.44269504f, kLn2 = 0.693147182f;
constexpr float kExpB = 1.4375f, kExpD = 2.0812597f;
// bits of 0.24109945 * 2^(i/32), less i << 18: adding (32 k + i) << 18 leaves
// those of 0.24109945 * 2^(k + i/32)
static __device__ const uint32_t kExpTable[32] = {
    0x3e76e2c6u, 0x3e784abcu, 0x3e78e880u, 0x3e77bb1eu, 0x3e769d8fu, 0x3e75902bu, 0x3e74934du, 0x3e73a752u,
    0x3e72cc98u, 0x3e720381u, 0x3e714c6eu, 0x3e70a7c5u, 0x3e7015eeu, 0x3e6f9751u, 0x3e6f2c5bu, 0x3e6ed579u,
    0x3e6e931cu, 0x3e6e65b8u, 0x3e6e4dc1u, 0x3e6e4bb0u, 0x3e6e6000u, 0x3e6e8b2eu, 0x3e6ecdbau, 0x3e6f2828u,
    0x3e6f9afcu, 0x3e7026c1u, 0x3e70cc01u, 0x3e718b4cu, 0x3e726533u, 0x3e735a4cu, 0x3e746b2fu, 0x3e759878u,
};
struct Exp2 {
  f2 e, y;  // 2^y, and y as clamped
};
struct ExpParts {
  f2 z, p, y;  // 1.5 * 2^18 + (32 k + i) / 32, 2^f / A, the clamped argument
};
template <bool CLAMP>
DI ExpParts exp_parts(f2 y, f2 one) {
  if constexpr (CLAMP) {
    float2 c = un(y);
    c.x = max_nan(c.x, kYLow);
    c.y = max_nan(c.y, kYLow);
    y = pk(c.x, c.y);
  }
  const f2 magic = pk(393216.0f, 393216.0f), shifted_magic = pk(393216.0f + kExpB, 393216.0f + kExpB);
  const f2 neg = pk(-1.0f, -1.0f);
  const f2 z = addp(y, one, magic);  // y may come straight from a multiply
  const f2 g = addp(y, one, fma2(z, neg, shifted_magic));  // an exact multiply by -1; f + B
  return {z, addp(mul2(g, g), one, pk(kExpD, kExpD)), y};
}
// the table's entry times 2^k; CLAMP: 0 where that is not a normal number
template <bool CLAMP>
DI float exp_scale(uint32_t entry, float z) {
  const int b = (int)(entry + (__float_as_uint(z) << 18));
  return __int_as_float(CLAMP && b < 0x00800000 ? 0 : b);
}
// every lane of the warp takes part; `table`: the lane's entry.  Without CLAMP
// every y that is a number has to be >= kYSafe; the bits are the same.
constexpr float kYSafe = -122.0f;
template <bool CLAMP>
DI Exp2 exp2_warp(f2 y, uint32_t table, f2 one) {
  const ExpParts t = exp_parts<CLAMP>(y, one);
  const float2 z = un(t.z);
  const uint32_t ax = __shfl_sync(kFull, table, __float_as_int(z.x));
  const uint32_t ay = __shfl_sync(kFull, table, __float_as_int(z.y));
  return {mul2(pk(exp_scale<CLAMP>(ax, z.x), exp_scale<CLAMP>(ay, z.y)), t.p), t.y};
}
// one value, any lanes; the same bits
DI float exp2_one(float y, float one) {
  const ExpParts t = exp_parts<true>(pk(y, y), pk(one, one));
  const float z = un(t.z).x;
  return fmul(exp_scale<true>(kExpTable[__float_as_uint(z) & 31], z), un(t.p).x);
}

// ---- element types ---------------------------------------------------------------
template <typename T>
DI float to_f32(T v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(v);
  else return __bfloat162float(v);
}
template <typename T>
DI T from_f32(float v) {  // one rounding, to nearest even
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}
DI float load_any(const void* p, int dtype, size_t i) {
  if (dtype == DET_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == DET_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
DI long long load_id(const void* p, int bytes, size_t i) {
  return bytes == 8 ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

// ---- a segment -------------------------------------------------------------------
// Lane l's vector i of a segment holds its entries (32 i + l) VEC + j.
template <typename T>
struct Seg {
  static constexpr int VEC = 16 / (int)sizeof(T);     // entries per 16 bytes
  static constexpr int NV = kPerLane / VEC;           // vectors per lane
  static constexpr int GROUP = 32 * VEC;              // adjacent entries a warp loads at once
};

template <typename T>
DI void unpack_vec(uint4 w, float* v) {
  if constexpr (std::is_same_v<T, float>) {
    v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y);
    v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
  } else {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        v[2 * i] = __uint_as_float(__byte_perm(u[i], 0, 0x1044));
        v[2 * i + 1] = __uint_as_float(__byte_perm(u[i], 0, 0x3244));
      } else {
        __half2 h;
        memcpy(&h, &u[i], 4);
        const float2 f = __half22float2(h);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
}
// x + c for the pairs of a vector: a 16-bit x is widened by the addition itself
template <typename T>
DI void add_vec(uint4 w, float c, f2 (&d)[8 / sizeof(T)]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  if constexpr (std::is_same_v<T, float>) {
    d[0] = add2(pk(__uint_as_float(u[0]), __uint_as_float(u[1])), pk(c, c));
    d[1] = add2(pk(__uint_as_float(u[2]), __uint_as_float(u[3])), pk(c, c));
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const unsigned short lo = (unsigned short)u[i], hi = (unsigned short)(u[i] >> 16);
      float a, b;
      if constexpr (std::is_same_v<T, __half>) {
        asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(a) : "h"(lo), "f"(c));
        asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(b) : "h"(hi), "f"(c));
      } else {
        asm("add.rn.f32.bf16 %0, %1, %2;" : "=f"(a) : "h"(lo), "f"(c));
        asm("add.rn.f32.bf16 %0, %1, %2;" : "=f"(b) : "h"(hi), "f"(c));
      }
      d[i] = pk(a, b);
    }
  }
}
// 16 bytes that start `bytes` (< 16, even) into the 32 of a and b; `bytes` is
// the same in every lane
DI uint4 shifted(uint4 a, uint4 b, int bytes) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (bytes & 8) {
#pragma unroll
    for (int i = 0; i < 6; i++) w[i] = w[i + 2];
  }
  if (bytes & 4) {
#pragma unroll
    for (int i = 0; i < 5; i++) w[i] = w[i + 1];
  }
  if (bytes & 2) {
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// VEC entries from entry `at` of a row; what is past its end is -inf.  Only
// 16-byte granules that lie in the row as a whole are loaded as such: a row
// that starts `mis` entries into a granule takes two of them per vector.
// RO: nothing writes the row while the kernel runs.
template <bool RO>
DI uint4 load16(const uint4* p) {
  if constexpr (RO) return __ldg(p);
  else return *p;
}
template <typename T, bool RO = true>
DI void load_vec(const T* row, int at, int V, int mis, float* v) {
  constexpr int VEC = Seg<T>::VEC;
  const T* p = row + at;
  if (mis == 0 && at >= 0 && at + VEC <= V) {
    unpack_vec<T>(load16<RO>(reinterpret_cast<const uint4*>(p)), v);
  } else if (mis != 0 && at >= mis && at - mis + 2 * VEC <= V) {
    const uint4* q = reinterpret_cast<const uint4*>(p - mis);
    unpack_vec<T>(shifted(load16<RO>(q), load16<RO>(q + 1), mis * (int)sizeof(T)), v);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j++) v[j] = at + j >= 0 && at + j < V ? to_f32(p[j]) : -INFINITY;
  }
}
template <typename T>
DI uint4 pack_vec(const float* v) {
  uint32_t w[4];
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        memcpy(&w[i], &h, 4);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        memcpy(&w[i], &h, 4);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
DI int misaligned(const T* row) {
  return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}
// A warp's segment on its way: its 16-byte granules (one more where the row
// starts inside one) are copied to shared memory asynchronously, so the next
// segment is fetched while this one is in registers.  What lies past the
// row's end is -inf there.
template <typename T>
constexpr int kStageBytes = kSeg * (int)sizeof(T) + 16;
template <typename T>
DI void stage_granule(uint32_t to, const T* row, int at, int V) {
  constexpr int VEC = Seg<T>::VEC;
  if (at >= 0 && at + VEC <= V) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(row + at) : "memory");
  } else {
    float v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) v[j] = at + j >= 0 && at + j < V ? to_f32(row[at + j]) : -INFINITY;
    const uint4 w = pack_vec<T>(v);
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
  }
}
template <typename T>
DI void stage_issue(const void* buf, const T* row, int g, int V) {
  using G = Seg<T>;
  const int l = threadIdx.x & 31, mis = misaligned(row), first = g * kSeg - mis;
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(buf) + 16 * l;
  if (first >= 0 && first + kSeg + (mis ? G::VEC : 0) <= V) {  // no granule reaches out of the row
    const T* p = row + first + l * G::VEC;
#pragma unroll
    for (int i = 0; i < G::NV; i++)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 512 * i), "l"(p + i * G::GROUP) : "memory");
    if (mis != 0 && l == 0)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 512 * G::NV), "l"(p + kSeg) : "memory");
  } else {
#pragma unroll 1
    for (int i = 0; i < G::NV; i++) stage_granule<T>(to + 512 * i, row, first + (32 * i + l) * G::VEC, V);
    if (mis != 0 && l == 0) stage_granule<T>(to + 512 * G::NV, row, first + kSeg, V);
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}
// waits for the warp's segment and takes it; the buffer is free afterwards
template <typename T>
DI void stage_take(const void* buf, int mis, uint4 (&v)[Seg<T>::NV]) {
  using G = Seg<T>;
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();
  const uint4* w = static_cast<const uint4*>(buf) + (threadIdx.x & 31);
  if (mis == 0) {
#pragma unroll
    for (int i = 0; i < G::NV; i++) v[i] = w[32 * i];
  } else {
#pragma unroll
    for (int i = 0; i < G::NV; i++) v[i] = shifted(w[32 * i], w[32 * i + 1], mis * (int)sizeof(T));
  }
  __syncwarp();
}
DI float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
DI float min3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The largest and smallest of vectors' entries, taken vector by vector; NaN
// loses against a number.
template <typename T>
struct Range {
  float hi = -INFINITY, lo = INFINITY;
  DI void take(uint4 w) {
    hi = max3(max3(hi, __uint_as_float(w.x), __uint_as_float(w.y)), __uint_as_float(w.z), __uint_as_float(w.w));
    lo = min3(min3(lo, __uint_as_float(w.x), __uint_as_float(w.y)), __uint_as_float(w.z), __uint_as_float(w.w));
  }
  DI float high() const { return hi; }
  DI float low() const { return lo; }
};
template <typename P>  // pairs of 16-bit entries
struct PairRange {
  P hi, lo;
  DI PairRange() {
    const uint32_t inf = std::is_same_v<P, __half2> ? 0x7c007c00u : 0x7f807f80u, ninf = inf | 0x80008000u;
    memcpy(&hi, &ninf, 4);
    memcpy(&lo, &inf, 4);
  }
  DI void take(uint4 w) {
    P p[4];
    memcpy(p, &w, 16);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      hi = __hmax2(hi, p[i]);
      lo = __hmin2(lo, p[i]);
    }
  }
  DI float high() const { return fmaxf(to_f32(hi.x), to_f32(hi.y)); }
  DI float low() const { return fminf(to_f32(lo.x), to_f32(lo.y)); }
};
template <>
struct Range<__half> : PairRange<__half2> {};
template <>
struct Range<__nv_bfloat16> : PairRange<__nv_bfloat162> {};

struct Sums {
  float m, s, w;  // maximum, sum of 2^y, sum of 2^y y, with y = (x - m) log2(e) / T
};

DI float warp_max(float v) {
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
DI float warp_sum(float v) {
  for (int o = 16; o > 0; o >>= 1) v = fadd(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
// the sum of s in lanes 0 .. 15, of w in lanes 16 .. 31
DI float warp_sum2(float s, float w) {
  const bool low = (threadIdx.x & 16) == 0;
  float v = fadd(low ? s : w, __shfl_xor_sync(kFull, low ? w : s, 16));
  for (int o = 8; o > 0; o >>= 1) v = fadd(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
DI double warp_sum_d(double v) {
  for (int o = 16; o > 0; o >>= 1) v = dadd(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

// a segment's sums s (in lanes 0 .. 15) and w (in lanes 16 .. 31), of the lanes'
// vectors v with maximum m; a NaN or +inf anywhere leaves w NaN.  Quarters of
// the segment from `entries` on are all -inf and add nothing: they are passed
// over.  KEEP: e becomes 2^y.
template <typename T, bool KEEP, bool CLAMP>
DI float sum_segment(const uint4 (&v)[Seg<T>::NV], int entries, float m, float c, uint32_t table, float one_,
                     float* e) {
  using G = Seg<T>;
  const float base = m == -INFINITY ? 0.0f : -m;
  const f2 one = pk(one_, one_), cc = pk(c, c);
  f2 s[2] = {0, 0}, w[2] = {0, 0};
#pragma unroll
  for (int q = 0; q < 4; q++) {
    if (q * (kSeg / 4) >= entries) {
      if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < kPerLane / 4; i++) e[q * (kPerLane / 4) + i] = 0.0f;
      }
      continue;
    }
#pragma unroll
    for (int i = q * (G::NV / 4); i < (q + 1) * (G::NV / 4); i++) {
      f2 d[G::VEC / 2];
      add_vec<T>(v[i], base, d);
#pragma unroll
      for (int j = 0; j < G::VEC / 2; j++) {
        const Exp2 t = exp2_warp<CLAMP>(mul2(d[j], cc), table, one);
        s[j & 1] = add2(s[j & 1], t.e);
        w[j & 1] = addp(mul2(t.e, t.y), one, w[j & 1]);
        if constexpr (KEEP) {
          const float2 k = un(t.e);
          e[i * G::VEC + 2 * j] = k.x;
          e[i * G::VEC + 2 * j + 1] = k.y;
        }
      }
    }
  }
  const float2 sp = un(add2(s[0], s[1])), wp = un(add2(w[0], w[1]));
  return warp_sum2(fadd(sp.x, sp.y), fadd(wp.x, wp.y));
}
// `low`: the smallest entry.  Where no entry is so far below the maximum that
// its power has to be cleared, the clamp and the clearing are left out (4
// of some 20 operations per pair of entries).
template <typename T, bool KEEP>
DI float segment_sums(const uint4 (&v)[Seg<T>::NV], int entries, float m, float low, float c, uint32_t table,
                      float one, float* e) {
  if (fmul(fsub(low, m), c) >= kYSafe) return sum_segment<T, KEEP, false>(v, entries, m, c, table, one, e);
  return sum_segment<T, KEEP, true>(v, entries, m, c, table, one, e);
}
DI float redux_max(float v) {  // of the warp; a NaN loses against a number
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "r"(kFull));
  return r;
}

DI float redux_min(float v) {
  float r;
  asm volatile("redux.sync.min.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "r"(kFull));
  return r;
}

// y of a segment's maximum under the row's
DI float segment_y(float ms, float m, float c) {
  return ms == -INFINITY ? kYLow : fmaxf(fmul(fsub(ms, m), c), kYLow);
}
// joins a row's segments (one warp; the result in every lane): at(i) gives
// segment i's sums
template <typename F>
DI Sums join_segments(F at, int nseg, float c, float one) {
  const int l = threadIdx.x & 31;
  Sums t[kMaxSegs / 32];
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMaxSegs / 32; i++) {
    t[i] = 32 * i + l < nseg ? at(32 * i + l) : Sums{-INFINITY, 0.0f, 0.0f};
    m = fmaxf(m, t[i].m);
  }
  m = redux_max(m);
  float s = 0.0f, w = 0.0f;
#pragma unroll
  for (int i = 0; i < kMaxSegs / 32; i++) {
    if (32 * i >= nseg) break;
    const float y = segment_y(t[i].m, m, c);
    const float f = exp2_one(y, one);
    s = fadd(s, fmul(f, t[i].s));
    // sum of 2^(y_j + y) (y_j + y) = f (w + y s); NaN stays NaN
    w = fadd(w, fmul(f, fadd(t[i].w, fmul(y, t[i].s))));
  }
  return {m, warp_sum(s), warp_sum(w)};
}

struct RowStats {
  float m, s, s1;
  bool empty, bad;
};
DI RowStats finish_row(const Sums& r) {
  RowStats t;
  t.bad = !(r.w == r.w) || r.m == INFINITY;
  t.empty = !t.bad && r.m == -INFINITY;
  const float nan = __int_as_float(0x7fffffff);
  t.m = t.bad ? nan : r.m;
  t.s = t.bad ? nan : t.empty ? 0.0f : r.s;
  t.s1 = t.bad ? nan : t.empty ? 0.0f : fmul(r.w, kLn2);
  return t;
}
// log S in 64 bits
DI double log_sum(const RowStats& r) {
  return r.bad ? (double)__int_as_float(0x7fffffff) : r.empty ? (double)-INFINITY : log_det((double)r.s);
}

// order of the top list: larger values first, of equal values the lower
// index; keys are distinct, 0 is below every key
DI unsigned long long top_key(float v, uint32_t index) {
  const uint32_t b = __float_as_uint(fadd(v, 0.0f));  // -0 and +0 are equal
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return ((unsigned long long)o << 32) | (0xffffffffu - index);
}
DI float key_value(unsigned long long key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

struct Logits {
  const void* x;
  const uint32_t* rows;  // null: row i of the call is row i of x
  unsigned long long ld;
  int n, vocab;
};
struct ScoreOut {
  float *logprob, *entropy, *stats;
  int32_t* top_ids;
  float* top_logprobs;
  int top;
  uint32_t* flags;
};
struct Teacher {
  const void* ids;
  const void* u;
  unsigned long long ld;
  int id_bytes, dtype, k;
};

// ---- the teacher's list of one row ---------------------------------------------
struct ListShared {
  float max[kWarps], sum[kWarps];
  int bad[kWarps], some[kWarps];
  int id[DET_MAX_TOP];
  float q[DET_MAX_TOP];
  double term[kWarps];
};
struct ListEntry {
  int id;         // -1: not a valid entry
  float q;        // its share of the teacher's distribution
  float d;        // u - max u
  bool some, bad;  // of the list: a valid entry; an id or value that is not allowed
  float s;        // of the list: sum of exp(d / T)
};
// Thread i < k of the block gets entry i (blocks have at least DET_MAX_TOP
// threads).  Begins and ends with the block in step.
DI ListEntry teacher_entry(const Teacher& te, int row, int vocab, float c, float one, ListShared& sh) {
  const int t = threadIdx.x, w = t >> 5, l = t & 31, nw = blockDim.x >> 5;
  long long id = -1;
  float u = -INFINITY;
  if (t < te.k) {
    id = load_id(te.ids, te.id_bytes, (size_t)row * te.ld + t);
    if (id >= 0) u = load_any(te.u, te.dtype, (size_t)row * te.ld + t);
  }
  const bool wrong = id >= vocab || (id >= 0 && !(u < INFINITY));  // NaN, +inf or no such token
  const bool valid = id >= 0 && !wrong && u > -INFINITY;
  float m = warp_max(valid ? u : -INFINITY);
  const int anyw = __any_sync(kFull, wrong), anyv = __any_sync(kFull, valid);
  __syncthreads();
  if (l == 0) {
    sh.max[w] = m;
    sh.bad[w] = anyw;
    sh.some[w] = anyv;
  }
  __syncthreads();
  m = -INFINITY;
  ListEntry r;
  r.some = r.bad = false;
  for (int i = 0; i < nw; i++) {
    m = fmaxf(m, sh.max[i]);
    r.bad |= sh.bad[i] != 0;
    r.some |= sh.some[i] != 0;
  }
  r.d = valid ? fsub(u, m) : 0.0f;
  const float e = valid ? exp2_one(fmul(r.d, c), one) : 0.0f;
  const float ws = warp_sum(e);
  if (l == 0) sh.sum[w] = ws;
  __syncthreads();
  r.s = 0.0f;
  for (int i = 0; i < nw; i++) r.s = fadd(r.s, sh.sum[i]);
  r.id = valid ? (int)id : -1;
  r.q = valid ? fdiv(e, r.s) : 0.0f;
  return r;
}
// the row's loss, in thread 0; z: the logit at the thread's entry.  Ends with
// the block in step.
DI float list_loss(const ListEntry& e, float z, const RowStats& r, double log_s, float temp, ListShared& sh) {
  double term = 0.0;
  if (e.id >= 0 && e.q > 0.0f) {
    const double logq = dsub(ddiv((double)e.d, (double)temp), log_det((double)e.s));
    const double logp =
        r.empty ? (double)-INFINITY : dsub(ddiv(dsub((double)z, (double)r.m), (double)temp), log_s);
    term = dmul((double)e.q, dsub(logq, logp));
  }
  term = warp_sum_d(term);
  if ((threadIdx.x & 31) == 0) sh.term[threadIdx.x >> 5] = term;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < (int)(blockDim.x >> 5); i++) s = dadd(s, sh.term[i]);
  const float nan = __int_as_float(0x7fffffff);
  return e.bad ? nan : !e.some ? 0.0f : r.bad ? nan : (float)s;
}
// The share to take off at the thread's entry: what all entries of its id add
// up to, in their order, at the first of them; 0 and id -1 at the others.
DI float list_share(ListEntry& e, int k, ListShared& sh) {
  __syncthreads();
  if ((int)threadIdx.x < k) {
    sh.id[threadIdx.x] = e.id;
    sh.q[threadIdx.x] = e.q;
  }
  __syncthreads();
  float sum = 0.0f;
  if (e.id < 0) return sum;
  bool first = true;
  for (int i = 0; i < k; i++)
    if (sh.id[i] == e.id) {
      first &= i >= (int)threadIdx.x;
      sum = fadd(sum, sh.q[i]);
    }
  if (!first) e.id = -1;
  return sum;
}

// ---- the top list ------------------------------------------------------------------
// The maximum of every group of adjacent entries is kept while a row's sums
// are taken; the k largest entries lie in the groups whose maxima are among
// the k largest, so only those are read again.  A group is what a warp loads
// at once (128 f32 or 256 16-bit entries), or one lane's 16 bytes of it where
// that would leave too few groups for a list (vocabularies up to 32,768).
constexpr int kSmallVocab = 32768;
constexpr int kCand = 2048;  // keys held before they are cut down to k
struct TopShared {
  unsigned long long key[kCand + kThreads];
  int count, bits[2];
  uint32_t lo, hi;
};
template <typename T>
DI int group_size(int V) {
  return V <= kSmallVocab ? Seg<T>::VEC : Seg<T>::GROUP;
}
// A t that at least k of the block's values reach, and at most k + slack of
// them where values are not equal (0 where there are fewer than k): bit by
// bit below the bits that all of [lo, hi] share; lo <= every value <= hi.
template <typename K, int PER>
DI K kth_largest(const K (&v)[PER], K lo, K hi, int k, int slack, TopShared& sh) {
  const K differ = lo ^ hi;
  int bit = -1;
  if (differ) bit = sizeof(K) == 8 ? 63 - __clzll((long long)differ) : 31 - __clz((int)differ);
  K t = bit < 0 ? lo : lo & ~((K)2 * (((K)1 << bit) - 1) + 1);
  for (int turn = 0; bit >= 0; bit--, turn ^= 1) {
    const K cand = t | ((K)1 << bit);
    int c = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) c += v[i] >= cand;
    c = __reduce_add_sync(kFull, c);
    if ((threadIdx.x & 31) == 0 && c) atomicAdd(&sh.bits[turn], c);
    __syncthreads();
    const int all = sh.bits[turn];
    if (threadIdx.x == 0) sh.bits[turn ^ 1] = 0;
    __syncthreads();
    if (all >= k) t = cand;
    if (all >= k && all <= k + slack) break;
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.bits[0] = sh.bits[1] = 0;
  __syncthreads();
  return t;
}
// keeps the k largest of the block's sh.count keys (distinct); returns the
// smallest of them, or 0 if there are fewer than k
DI unsigned long long cut_to(int k, TopShared& sh) {
  __syncthreads();
  const int n = min(sh.count, kCand + kThreads);
  if (n <= k) {
    const unsigned long long r = 0;
    __syncthreads();
    return r;
  }
  constexpr int PER = (kCand + kThreads) / kThreads;
  unsigned long long v[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int at = i * kThreads + threadIdx.x;
    v[i] = at < n ? sh.key[at] : 0;
  }
  const unsigned long long t = kth_largest<unsigned long long, PER>(v, 0ull, ~0ull, k, 0, sh);
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; i++)
    if (v[i] >= t) sh.key[atomicAdd(&sh.count, 1)] = v[i];
  __syncthreads();
  return t;
}
// adds the entries of groups [g0, g1) whose keys are above `floor`
template <typename T>
DI void collect(const T* __restrict__ x, int V, int mis, const float* gmax, int g0, int g1, unsigned long long floor,
                TopShared& sh) {
  using G = Seg<T>;
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  auto push = [&](float v, int at) {
    const unsigned long long key = top_key(v, (uint32_t)at);
    if (at < V && key > floor) {
      const int slot = atomicAdd(&sh.count, 1);
      if (slot < kCand + kThreads) sh.key[slot] = key;
    }
  };
  if (V <= kSmallVocab) {
    for (int g = g0 + threadIdx.x; g < g1; g += kThreads)
      if (g * G::VEC < V && top_key(gmax[g], (uint32_t)(g * G::VEC)) > floor) {
#pragma unroll
        for (int j = 0; j < G::VEC; j++)
          if (g * G::VEC + j < V) push(to_f32(x[g * G::VEC + j]), g * G::VEC + j);
      }
    return;
  }
  for (int b = g0 + 32 * w; b < g1; b += kThreads) {
    const int mine = b + l;
    const bool want =
        mine < g1 && mine * G::GROUP < V && top_key(gmax[mine], (uint32_t)(mine * G::GROUP)) > floor;
    for (unsigned todo = __ballot_sync(kFull, want); todo; todo &= todo - 1) {
      const int at = (b + __ffs(todo) - 1) * G::GROUP + l * G::VEC;
      float v[G::VEC];
      load_vec<T>(x, at, V, mis, v);
#pragma unroll
      for (int j = 0; j < G::VEC; j++) push(v[j], at + j);
    }
  }
}
template <int PER>
DI unsigned long long list_floor(const float* gmax, int ng, int k, TopShared& sh) {
  uint32_t v[PER], lo = ~0u, hi = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int g = i * kThreads + threadIdx.x;
    const bool is = g < ng;
    v[i] = is ? (uint32_t)(top_key(gmax[g], 0) >> 32) : 0u;
    hi = max(hi, v[i]);
    if (is) lo = min(lo, v[i]);
  }
  hi = __reduce_max_sync(kFull, hi);
  lo = __reduce_min_sync(kFull, lo);
  if ((threadIdx.x & 31) == 0) {
    atomicMax(&sh.hi, hi);
    atomicMin(&sh.lo, lo);
  }
  __syncthreads();
  const uint32_t t = kth_largest<uint32_t, PER>(v, sh.lo, sh.hi, k, k / 4 + 4, sh);
  return t ? ((unsigned long long)t << 32) - 1 : 0;
}
// the row's k largest keys, in order, to sh.key[0 .. k)
template <typename T>
DI void top_list(const T* __restrict__ x, int V, int mis, const float* gmax, int k, TopShared& sh) {
  const int ng = (V + group_size<T>(V) - 1) / group_size<T>(V);
  if (threadIdx.x == 0) sh.count = sh.bits[0] = sh.bits[1] = 0, sh.lo = ~0u, sh.hi = 0;
  __syncthreads();
  // a value that at least k entries reach: about the k-th largest maximum
  unsigned long long floor = 0;
  if (ng > k) {
    floor = ng <= kThreads * 4   ? list_floor<4>(gmax, ng, k, sh)
            : ng <= kThreads * 8 ? list_floor<8>(gmax, ng, k, sh)
                                 : list_floor<kSmallVocab / 4 / kThreads>(gmax, ng, k, sh);
  }
  collect<T>(x, V, mis, gmax, 0, ng, floor, sh);
  __syncthreads();
  if (sh.count > kCand + kThreads) {
    // too many entries reach it (ties, or a row in order): group by group in
    // the order of their indices, cutting the list down as it fills, which
    // raises the floor and passes over groups that cannot add to it
    const int step = (kCand + kThreads - (int)DET_MAX_TOP) / group_size<T>(V);
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (int g = 0; g < ng; g += step) {
      collect<T>(x, V, mis, gmax, g, min(ng, g + step), floor, sh);
      const unsigned long long t = cut_to(k, sh);
      if (t) floor = t;
    }
  } else if (sh.count > kThreads) {
    cut_to(k, sh);
  }
  __syncthreads();
  // at most kThreads keys are left: each finds its rank
  const int n = sh.count;
  const unsigned long long mine = (int)threadIdx.x < n ? sh.key[threadIdx.x] : 0;
  int rank = 0;
  for (int i = 0; i < n; i++) rank += sh.key[i] > mine;
  __syncthreads();
  if ((int)threadIdx.x < n && rank < k) sh.key[rank] = mine;
  __syncthreads();
}

// ---- clusters ------------------------------------------------------------------------
DI uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
DI uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
DI void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
DI void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// *p of block `rank` of the cluster, p an address of one's own shared memory
DI uint32_t remote(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
DI void store_remote(uint32_t at, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }

// what a row's scores are written to (one thread)
DI void write_stats(float* stats, int row, const RowStats& r, double log_s) {
  float* st = stats + (size_t)row * 4;
  st[0] = r.m, st[1] = r.s, st[2] = r.s1, st[3] = (float)log_s;
}
DI void write_scores(const ScoreOut& o, int row, int V, const RowStats& r, double log_s, long long t, float x_t) {
  const float nan = __int_as_float(0x7fffffff);
  if (o.entropy)
    o.entropy[row] = r.bad ? nan : r.empty ? 0.0f : (float)dsub(log_s, ddiv((double)r.s1, (double)r.s));
  if (!o.logprob) return;
  float v;
  if (r.bad || t >= V) v = nan;
  else if (t < 0) v = 0.0f;
  else if (r.empty) v = -INFINITY;
  else v = (float)dsub(dsub((double)x_t, (double)r.m), log_s);
  o.logprob[row] = v;
}

// ---- forward ---------------------------------------------------------------------------
constexpr int kSegThreads = 256, kSegBlocks = 2;
// Two kernels.  In the first, warps take segments in turn, whatever row they
// are of, each with its next one on its way; nothing waits for anything else,
// and the parts are even however many rows there are.  A segment's sums and
// its groups' maxima go to the caller's workspace.  In the second, a block per
// row joins the row's segments and writes its results.
struct Workspace {
  float4* seg;  // [rows][segments]: m, s, w
  float* gmax;  // [rows][groups]
};
enum : int { GROUPS_NONE, GROUPS_LANE, GROUPS_WARP };  // which maxima a top list needs
template <typename T, int GROUPS>
__global__ void __launch_bounds__(kSegThreads, kSegBlocks)
    segments_kernel(Logits L, float temp, Workspace ws, float one) {
  using G = Seg<T>;
  extern __shared__ __align__(16) uint8_t dyn[];  // a stage per warp
  const int V = L.vocab, l = threadIdx.x & 31;
  const int nseg = (V + kSeg - 1) / kSeg, all = gridDim.x * (kSegThreads / 32);
  void* stage = dyn + (threadIdx.x >> 5) * kStageBytes<T>;
  auto at_row = [&](int r) { return static_cast<const T*>(L.x) + (size_t)(L.rows ? L.rows[r] : r) * L.ld; };
  const int first = blockIdx.x * (kSegThreads / 32) + (threadIdx.x >> 5);
  int row = first / nseg, g = first % nseg;
  const int drow = all / nseg, dg = all % nseg;
  if (row < L.n) stage_issue<T>(stage, at_row(row), g, V);
  pdl_trigger();
  const float c = fdiv(kLog2e, temp);
  const uint32_t table = kExpTable[l];
  while (row < L.n) {
    uint4 v[G::NV];
    stage_take<T>(stage, misaligned(at_row(row)), v);
    int nrow = row + drow, ng = g + dg;
    if (ng >= nseg) ng -= nseg, nrow++;
    if (nrow < L.n) stage_issue<T>(stage, at_row(nrow), ng, V);
    Range<T> all_range;
    float gm = -INFINITY;
    const size_t part = (size_t)row * nseg + g;
    float* gmax = ws.gmax + part * (kSeg / G::VEC) + l;
#pragma unroll
    for (int i = 0; i < G::NV; i++) {
      all_range.take(v[i]);
      if constexpr (GROUPS == GROUPS_NONE) continue;
      Range<T> group;
      group.take(v[i]);
      const float lm = group.high();
      if constexpr (GROUPS == GROUPS_LANE) gmax[i * 32] = lm;
      if constexpr (GROUPS == GROUPS_WARP) {
        const float r = redux_max(lm);
        if (l == i) gm = r;
      }
    }
    if constexpr (GROUPS == GROUPS_WARP) {
      if (l < G::NV) ws.gmax[part * G::NV + l] = gm;
    }
    const float m = redux_max(all_range.high()), low = redux_min(all_range.low());
    const float s = segment_sums<T, false>(v, V - g * kSeg, m, low, c, table, one, nullptr);
    const float w = __shfl_sync(kFull, s, 16);
    if (l == 0) ws.seg[part] = make_float4(m, s, w, 0.0f);
    row = nrow;
    g = ng;
  }
}
template <typename T, bool TOP>
__global__ void __launch_bounds__(TOP ? kThreads : (int)DET_MAX_TOP)
    rows_kernel(Logits L, const void* tokens, int id_bytes, Teacher te, float temp, Workspace ws, float* loss,
                ScoreOut o, float one) {
  __shared__ ListShared list;
  const int row = blockIdx.x, V = L.vocab, nseg = (V + kSeg - 1) / kSeg;
  const T* x = static_cast<const T*>(L.x) + (size_t)(L.rows ? L.rows[row] : row) * L.ld;
  const float c = fdiv(kLog2e, temp), nan = __int_as_float(0x7fffffff);
  // what does not depend on the sums, while they are being taken
  ListEntry e;
  float z = 0.0f;
  long long t = -1;
  if (loss) {
    e = teacher_entry(te, row, V, c, one, list);
    if (e.id >= 0) z = to_f32(x[e.id]);
  } else if (o.logprob) {
    t = load_id(tokens, id_bytes, row);
    if (t >= 0 && t < V) z = to_f32(x[t]);
  }
  pdl_wait();
  const float4* seg = ws.seg + (size_t)row * nseg;
  const RowStats r = finish_row(join_segments(
      [&](int i) {
        const float4 f = seg[i];
        return Sums{f.x, f.y, f.z};
      },
      nseg, c, one));
  const double log_s = log_sum(r);
  if (threadIdx.x == 0) {
    if (o.stats) write_stats(o.stats, row, r, log_s);
    if (r.bad && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_NONFINITE);
  }
  if (loss) {
    const float v = list_loss(e, z, r, log_s, temp, list);
    if (threadIdx.x == 0) {
      loss[row] = v;
      if (e.bad && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_BAD_TOKEN);
    }
  } else if (threadIdx.x == 0) {
    write_scores(o, row, V, r, log_s, t, z);
    if (t >= V && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_BAD_TOKEN);
  }
  if constexpr (TOP) {
    __shared__ TopShared top;
    if (!r.bad) top_list<T>(x, V, misaligned(x), ws.gmax + (size_t)row * nseg * (kSeg / group_size<T>(V)), o.top, top);
    if ((int)threadIdx.x < o.top) {
      const size_t at = (size_t)row * o.top + threadIdx.x;
      const unsigned long long key = r.bad ? 0 : top.key[threadIdx.x];
      if (o.top_ids) o.top_ids[at] = r.bad ? -1 : (int32_t)(0xffffffffu - (uint32_t)key);
      if (o.top_logprobs) {
        o.top_logprobs[at] = r.bad     ? nan
                             : r.empty ? -INFINITY
                                       : (float)dsub(dsub((double)key_value(key), (double)r.m), log_s);
      }
    }
  }
}

// ---- gradient --------------------------------------------------------------------------
// dx_j = 2^y_j (a + b y_j) / S + (what the row's own tokens add), y = (x - m)
// log2(e) / T; b is 0 but for the entropy's gradient.
struct GradIn {
  const float *stats, *g, *gh;  // g: of logprob or of the loss; gh: of the entropy, or null
};
struct RowGrad {
  float base, c, as, bs;  // -m, log2(e) / T, a / S, b / S
  bool zero;              // nothing but zeros
};
// the coefficients of a row of scores; gl: what its token adds
DI RowGrad score_grad(const GradIn& in, int row, int V, long long t, float m, float s, float s1, float c, float* gl) {
  const bool empty = m == -INFINITY;
  const float gh = in.gh ? in.gh[row] : 0.0f;
  *gl = !in.g || t < 0 ? 0.0f : t >= V ? __int_as_float(0x7fffffff) : in.g[row];
  const float inv_s = fdiv(1.0f, s);
  return {-m, c, fmul(fadd(-*gl, fmul(gh, fdiv(s1, s))), inv_s), fmul(fmul(-gh, kLn2), inv_s), empty};
}
// and of a row against a list; g_t: gradient of the loss over T
DI RowGrad list_grad(const ListEntry& e, float g_t, float m, float s, float c) {
  const float a = e.bad ? __int_as_float(0x7fffffff) : g_t;
  return {-m, c, fmul(a, fdiv(1.0f, s)), 0.0f, (!e.some && !e.bad) || m == -INFINITY};
}
// gradients of a pair of entries (of one, with the same bits)
template <bool ENTROPY>
DI f2 grad2(f2 e, f2 y, const RowGrad& r, f2 one) {
  if constexpr (ENTROPY) return mul2(e, addp(mul2(y, pk(r.bs, r.bs)), one, pk(r.as, r.as)));
  return mul2(e, pk(r.as, r.as));
}
template <bool ENTROPY>
DI float grad1(float x, const RowGrad& r, float one) {
  const float y = max_nan(fmul(fadd(x, r.base), r.c), kYLow);
  return un(grad2<ENTROPY>(pk(exp2_one(y, one), 0.0f), pk(y, 0.0f), r, pk(one, one))).x;
}

// Blocks (blockIdx.x) of a row (blockIdx.y + row0) take `per` of its 16-byte
// vectors each, their warps runs of 32 U vectors in turn; a vector is one of
// the gradient's, so that stores are whole wherever the row starts.  The next
// run is loaded before this one is worked on, the first before the row's
// coefficients are known.  `out` may be the logits themselves.
constexpr int kGradUnroll = 4, kGradRun = 32 * kGradUnroll;
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(kThreads, 3)
    grad_kernel(Logits L, int row0, int per, const void* tokens, int id_bytes, Teacher te, float temp, GradIn in,
                T* out, unsigned long long out_ld, float one_) {
  constexpr int VEC = Seg<T>::VEC, U = kGradUnroll;
  __shared__ ListShared sh;
  const int row = row0 + blockIdx.y, V = L.vocab, l = threadIdx.x & 31;
  const T* x = static_cast<const T*>(L.x) + (size_t)row * L.ld;
  T* y = out + (size_t)row * out_ld;
  const int my = misaligned(y), mis = (misaligned(x) - my) & (VEC - 1);
  const int nvec = (V + my + VEC - 1) / VEC;
  const int q0 = blockIdx.x * per, q1 = min(nvec, q0 + per);
  // the run at vector q: are all its entries, and the granules they come from, in the row and the block
  auto inside = [&](int q) {
    const int at = q * VEC - my;
    return q + kGradRun <= q1 && at >= mis && at + kGradRun * VEC + (mis ? VEC - mis : 0) <= V;
  };
  auto fetch = [&](int q, uint4(&w)[U]) {
    const T* p = x + (q + l) * VEC - my;
    if (inside(q)) {
      if (mis == 0) {
#pragma unroll
        for (int u = 0; u < U; u++) w[u] = *reinterpret_cast<const uint4*>(p + 32 * u * VEC);
      } else {
#pragma unroll
        for (int u = 0; u < U; u++) {
          const uint4* g = reinterpret_cast<const uint4*>(p - mis + 32 * u * VEC);
          w[u] = shifted(g[0], g[1], mis * (int)sizeof(T));
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int v = q + 32 * u + l, at = v * VEC - my;
        float f[VEC];
#pragma unroll
        for (int j = 0; j < VEC; j++) f[j] = v < q1 && at + j >= 0 && at + j < V ? to_f32(x[at + j]) : 0.0f;
        w[u] = pack_vec<T>(f);
      }
    }
  };
  const int w = threadIdx.x >> 5;
  uint4 cur[U];
  if (q0 + w * kGradRun < q1) fetch(q0 + w * kGradRun, cur);
  const float* st = in.stats + (size_t)row * 4;
  const float m = st[0], s = st[1], c = fdiv(kLog2e, temp);
  const uint32_t table = kExpTable[l];
  RowGrad r;
  int id;
  float add;
  if (te.k) {
    ListEntry e = teacher_entry(te, row, V, c, one_, sh);
    const float g_t = fdiv(in.g[row], temp);
    r = list_grad(e, g_t, m, s, c);
    add = fmul(-g_t, list_share(e, te.k, sh));
    id = e.id;
  } else {
    const long long t = in.g ? load_id(tokens, id_bytes, row) : -1;
    r = score_grad(in, row, V, t, m, s, st[2], c, &add);
    id = threadIdx.x == 0 && t >= 0 && t < V ? (int)t : -1;
  }
  // the values at the row's own tokens, before `out` may overwrite them
  const bool patch = id >= 0 && id >= q0 * VEC - my && id < q1 * VEC - my && !r.zero;
  float mine = 0.0f;
  if (patch) mine = fadd(grad1<ENTROPY>(to_f32(x[id]), r, one_), add);
  __syncthreads();
  const f2 one = pk(one_, one_), cc = pk(c, c);
  auto run = [&](uint4(&v)[U], auto clamp) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      f2 d[VEC / 2];
      add_vec<T>(v[u], r.base, d);
      float f[VEC];
#pragma unroll
      for (int j = 0; j < VEC / 2; j++) {
        const Exp2 e = exp2_warp<decltype(clamp)::value>(mul2(d[j], cc), table, one);
        const float2 gr = un(grad2<ENTROPY>(e.e, e.y, r, one));
        f[2 * j] = gr.x;
        f[2 * j + 1] = gr.y;
      }
      v[u] = pack_vec<T>(f);
    }
  };
  for (int q = q0 + w * kGradRun; q < q1; q += kThreads * U) {
    uint4 next[U];
    if (q + kThreads * U < q1) fetch(q + kThreads * U, next);
    const bool in = inside(q);
    // is no entry so far below the maximum that its power has to be cleared
    Range<T> range;
#pragma unroll
    for (int u = 0; u < U; u++) range.take(cur[u]);
    if (in && fmul(fadd(redux_min(range.low()), r.base), c) >= kYSafe && !r.zero) {
      run(cur, std::false_type{});
    } else if (!r.zero) {
      run(cur, std::true_type{});
    } else {
#pragma unroll
      for (int u = 0; u < U; u++) cur[u] = make_uint4(0, 0, 0, 0);
    }
    T* p = y + (q + l) * VEC - my;
    if (in) {
#pragma unroll
      for (int u = 0; u < U; u++) *reinterpret_cast<uint4*>(p + 32 * u * VEC) = cur[u];
    } else {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int v = q + 32 * u + l, at = v * VEC - my;
        if (v >= q1) continue;
        if (at >= 0 && at + VEC <= V) {
          *reinterpret_cast<uint4*>(y + at) = cur[u];
        } else {
          float f[VEC];
          unpack_vec<T>(cur[u], f);
#pragma unroll
          for (int j = 0; j < VEC; j++)
            if (at + j >= 0 && at + j < V) y[at + j] = from_f32<T>(f[j]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) cur[u] = next[u];
  }
  __syncthreads();
  if (patch) y[id] = from_f32<T>(mine);
}

// ---- both at once ------------------------------------------------------------------------
// Stores a warp's segment: vectors where the row is aligned; elsewhere lane l
// puts together the granule its vector starts in from its neighbour's end and
// its own start.
template <typename T, typename F>
DI void store_segment(T* y, int g, int V, int my, F vec) {
  using G = Seg<T>;
  constexpr int VEC = G::VEC;
  const int l = threadIdx.x & 31, lo = g * kSeg, hi = min(V, lo + kSeg);
  auto put = [&](int at, uint4 w) {  // what of [at, at + VEC) is in [lo, hi)
    if (at >= lo && at + VEC <= hi) {
      *reinterpret_cast<uint4*>(y + at) = w;
    } else {
      float f[VEC];
      unpack_vec<T>(w, f);
#pragma unroll
      for (int j = 0; j < VEC; j++)
        if (at + j >= lo && at + j < hi) y[at + j] = from_f32<T>(f[j]);
    }
  };
  if (my == 0) {
#pragma unroll
    for (int i = 0; i < G::NV; i++) put(lo + (32 * i + l) * VEC, vec(i));
    return;
  }
  uint4 carry = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < G::NV; i++) {
    const uint4 w = vec(i);
    uint4 p;  // of the lane before; lane 0 gets lane 31's, for the next turn
    p.x = __shfl_sync(kFull, w.x, (l + 31) & 31);
    p.y = __shfl_sync(kFull, w.y, (l + 31) & 31);
    p.z = __shfl_sync(kFull, w.z, (l + 31) & 31);
    p.w = __shfl_sync(kFull, w.w, (l + 31) & 31);
    const uint4 before = l == 0 ? carry : p;
    carry = p;
    put(lo + (32 * i + l) * VEC - my, shifted(before, w, 16 - my * (int)sizeof(T)));
    if (i == G::NV - 1 && l == 31) put(lo + kSeg - my, shifted(w, w, 16 - my * (int)sizeof(T)));
  }
}

// Clusters take rows in turn; each of a cluster's warps holds one segment of
// the row, so the row is read once: its exponentials stay in registers until
// every block has all segments' sums, and are scaled and stored then, while
// the next row's segment is on its way.  The entropy's gradient needs y too:
// it keeps the logits and takes their exponentials again.
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(kThreads, 2)
    step_kernel(Logits L, const void* tokens, int id_bytes, Teacher te, float temp, GradIn in, float* loss,
                ScoreOut o, T* out, unsigned long long out_ld, float one_) {
  __shared__ struct {
    float m[kMaxSegs], s[kMaxSegs], w[kMaxSegs];
    ListShared list;
  } sh;
  extern __shared__ __align__(16) uint8_t dyn[];
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int V = L.vocab, w = threadIdx.x >> 5, l = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int nseg = (V + kSeg - 1) / kSeg, clusters = gridDim.x / size;
  const int g = rank * warps + w;
  const bool active = g < nseg;
  void* stage = dyn + w * kStageBytes<T>;
  auto at_row = [&](int r) { return static_cast<const T*>(L.x) + (size_t)r * L.ld; };
  int row = blockIdx.x / size;
  if (row < L.n && active) stage_issue<T>(stage, at_row(row), g, V);
  const float c = fdiv(kLog2e, temp);
  const uint32_t table = kExpTable[l];
  if (size > 1) cluster_arrive();
  for (; row < L.n; row += clusters) {
    const T* x = at_row(row);
    T* y = out + (size_t)row * out_ld;
    uint4 raw[Seg<T>::NV];
    float v[ENTROPY ? 1 : kPerLane];
    float m_seg = -INFINITY, s_seg = 0.0f, w_seg = 0.0f;
    if (active) {
      stage_take<T>(stage, misaligned(x), raw);
      if (row + clusters < L.n) stage_issue<T>(stage, at_row(row + clusters), g, V);
      Range<T> range;
#pragma unroll
      for (int i = 0; i < Seg<T>::NV; i++) range.take(raw[i]);
      m_seg = redux_max(range.high());
      s_seg = segment_sums<T, !ENTROPY>(raw, V - g * kSeg, m_seg, redux_min(range.low()), c, table, one_, v);
      w_seg = __shfl_sync(kFull, s_seg, 16);
      s_seg = __shfl_sync(kFull, s_seg, 0);
    }
    // the row's own tokens, before `out` may overwrite their logits
    ListEntry e;
    long long t = -1;
    int id;
    float share = 0.0f;
    if (te.k) {
      e = teacher_entry(te, row, V, c, one_, sh.list);
      id = e.id;
    } else {
      t = tokens ? load_id(tokens, id_bytes, row) : -1;
      id = threadIdx.x == 0 && t >= 0 && t < V ? (int)t : -1;
    }
    const float z = id >= 0 ? to_f32(x[id]) : 0.0f;
    if (te.k) {
      ListEntry f = e;
      share = list_share(f, te.k, sh.list);
      id = f.id;
    }
    if (size > 1) cluster_wait();
    else __syncthreads();
    if (active && l < (int)size) {
      store_remote(remote(&sh.m[g], l), m_seg);
      store_remote(remote(&sh.s[g], l), s_seg);
      store_remote(remote(&sh.w[g], l), w_seg);
    }
    if (size > 1) {
      cluster_arrive();
      cluster_wait();
    } else {
      __syncthreads();
    }
    const RowStats r =
        finish_row(join_segments([&](int i) { return Sums{sh.m[i], sh.s[i], sh.w[i]}; }, nseg, c, one_));
    if (size > 1) cluster_arrive();
    RowGrad rg;
    float add;
    if (te.k) {
      const float g_t = fdiv(in.g[row], temp);
      rg = list_grad(e, g_t, r.m, r.s, c);
      add = fmul(-g_t, share);
    } else {
      rg = score_grad(in, row, V, t, r.m, r.s, r.s1, c, &add);
    }
    if (active) {
      const f2 one = pk(one_, one_), cc = pk(c, c);
      const float f = fmul(exp2_one(segment_y(m_seg, r.m, c), one_), rg.as);
      // vector i of the segment's gradient
      auto vec = [&](int i) {
        constexpr int VEC = Seg<T>::VEC;
        float x[VEC];
        f2 dx[VEC / 2];
        if constexpr (ENTROPY) add_vec<T>(raw[i], rg.base, dx);
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
          f2 d;
          if constexpr (ENTROPY) {
            const Exp2 ex = exp2_warp<true>(mul2(dx[j / 2], cc), table, one);
            d = grad2<true>(ex.e, ex.y, rg, one);
          } else {
            d = mul2(pk(v[i * VEC + j], v[i * VEC + j + 1]), pk(f, f));
          }
          const float2 dv = un(d);
          x[j] = rg.zero ? 0.0f : dv.x;
          x[j + 1] = rg.zero ? 0.0f : dv.y;
        }
        return pack_vec<T>(x);
      };
      store_segment<T>(y, g, V, misaligned(y), vec);
    }
    if (rank == 0) {
      const double log_s = log_sum(r);
      if (threadIdx.x == 0) {
        if (o.stats) write_stats(o.stats, row, r, log_s);
        if (r.bad && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_NONFINITE);
        if ((te.k ? e.bad : t >= V) && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_BAD_TOKEN);
        if (!te.k) write_scores(o, row, V, r, log_s, t, z);
      }
      if (te.k) {
        const float lv = list_loss(e, z, r, log_s, temp, sh.list);
        if (threadIdx.x == 0) loss[row] = lv;
      }
    }
    __syncthreads();  // the segments are stored
    if (id >= (int)rank * warps * kSeg && id < (int)(rank + 1) * warps * kSeg && !rg.zero)
      y[id] = from_f32<T>(fadd(grad1<ENTROPY>(z, rg, one_), add));
  }
  if (size > 1) cluster_wait();
}

// ---- launches --------------------------------------------------------------------
template <typename F>
cudaError_t by_dtype(int dtype, F f) {
  switch (dtype) {
    case DET_DTYPE_F32: return f(float{});
    case DET_DTYPE_F16: return f(__half{});
    default: return f(__nv_bfloat16{});
  }
}

// Clusters of `c` blocks that the current device holds at once, at least 1
// (cached: the answer depends on the kernel and the launch alone).
int resident_clusters(const void* kern, int c, int threads, size_t smem) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 1;
  static std::mutex mu;
  static std::map<std::tuple<const void*, int, int, int, size_t>, int> known;
  std::lock_guard<std::mutex> lock(mu);
  int& n = known[{kern, dev, c, threads, smem}];
  if (n > 0) return n;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)c);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int got = 0;
  if (cudaOccupancyMaxActiveClusters(&got, kern, &cfg) != cudaSuccess || got < 1) {
    cudaGetLastError();
    got = 1;
  }
  return n = got;
}
// launches `clusters` clusters of c blocks
template <typename... KArgs, typename... Args>
cudaError_t launch_clusters(cudaStream_t s, void (*kern)(KArgs...), int clusters, int c, int threads, size_t smem,
                            Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * c));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = c > 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}
// clusters above 8 blocks have to be allowed, once per kernel and device
cudaError_t allow_large_clusters(const void* kern) {
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> done;
  std::lock_guard<std::mutex> lock(mu);
  if (done.count({kern, dev})) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) done.insert({kern, dev});
  return e;
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
// what a forward call keeps between its two kernels
size_t workspace_bytes(int dtype, int n, int vocab, int top) {
  const size_t nseg = (vocab + kSeg - 1) / kSeg, vec = dtype == DET_DTYPE_F32 ? 4 : 8;
  const size_t groups = !top ? 0 : nseg * kSeg / (vocab <= kSmallVocab ? vec : 32 * vec);
  return align256(n * nseg * sizeof(float4)) + align256(n * groups * sizeof(float));
}
template <typename T, bool TOP>
cudaError_t forward_as(cudaStream_t s, const Logits& L, const void* tokens, int id_bytes, const Teacher& te,
                       float temp, void* workspace, float* loss, const ScoreOut& o) {
  const auto segments = !TOP                       ? segments_kernel<T, GROUPS_NONE>
                        : L.vocab <= kSmallVocab ? segments_kernel<T, GROUPS_LANE>
                                                 : segments_kernel<T, GROUPS_WARP>;
  constexpr int kSegWarps = kSegThreads / 32;
  const size_t smem = kSegWarps * kStageBytes<T>;
  if (cudaError_t e = raise_smem_cap((const void*)segments, smem)) return e;
  const long long nseg = (L.vocab + kSeg - 1) / kSeg, blocks = (L.n * nseg + kSegWarps - 1) / kSegWarps;
  const int fit = resident_clusters((const void*)segments, 1, kSegThreads, smem);
  Workspace ws;
  ws.seg = static_cast<float4*>(workspace);
  ws.gmax = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + align256(L.n * nseg * sizeof(float4)));
  segments<<<(unsigned)(blocks < fit ? blocks : fit), kSegThreads, smem, s>>>(L, temp, ws, 1.0f);
  if (cudaError_t e = cudaGetLastError()) return e;
  const Launch launch{s, nullptr, nullptr, true};
  return launch_k(launch, rows_kernel<T, TOP>, dim3(L.n), dim3(TOP ? kThreads : DET_MAX_TOP), 0, L, tokens, id_bytes,
                  te, temp, ws, loss, o, 1.0f);
}
cudaError_t launch_forward(cudaStream_t s, int dtype, const Logits& L, const void* tokens, int id_bytes,
                           const Teacher& te, float temp, void* workspace, float* loss, const ScoreOut& o) {
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return o.top ? forward_as<T, true>(s, L, tokens, id_bytes, te, temp, workspace, loss, o)
                 : forward_as<T, false>(s, L, tokens, id_bytes, te, temp, workspace, loss, o);
  });
}

template <typename T, bool ENTROPY>
cudaError_t grad_as(cudaStream_t s, const Logits& L, const void* tokens, int id_bytes, const Teacher& te, float temp,
                    const GradIn& in, void* out, unsigned long long out_ld) {
  constexpr int VEC = Seg<T>::VEC;
  const int nvec = (L.vocab + VEC - 1) / VEC + 1;  // one more where a row starts inside a vector
  // up to 8 runs per warp, fewer where that would leave SMs without a block
  const int step = kThreads * kGradUnroll;
  int per = 8 * step;
  while (per > step && (long long)L.n * ((nvec + per - 1) / per) < 8 * device_sms()) per -= step;
  while (per > kGradRun && (long long)L.n * ((nvec + per - 1) / per) < device_sms()) per /= 2;
  const int blocks = (nvec + per - 1) / per;
  for (int r = 0; r < L.n; r += 65535) {
    grad_kernel<T, ENTROPY><<<dim3(blocks, L.n - r < 65535 ? L.n - r : 65535), kThreads, 0, s>>>(
        L, r, per, tokens, id_bytes, te, temp, in, static_cast<T*>(out), out_ld, 1.0f);
    if (cudaError_t e = cudaGetLastError()) return e;
  }
  return cudaSuccess;
}
cudaError_t launch_grad(cudaStream_t s, int dtype, const Logits& L, const void* tokens, int id_bytes,
                        const Teacher& te, float temp, const GradIn& in, void* out, unsigned long long out_ld) {
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return in.gh ? grad_as<T, true>(s, L, tokens, id_bytes, te, temp, in, out, out_ld)
                 : grad_as<T, false>(s, L, tokens, id_bytes, te, temp, in, out, out_ld);
  });
}

template <typename T, bool ENTROPY>
cudaError_t step_as(cudaStream_t s, const Logits& L, const void* tokens, int id_bytes, const Teacher& te, float temp,
                    const GradIn& in, float* loss, const ScoreOut& o, void* out, unsigned long long out_ld) {
  const auto kern = step_kernel<T, ENTROPY>;
  // a warp per segment; at least DET_MAX_TOP threads, one per list entry
  const int nseg = (L.vocab + kSeg - 1) / kSeg, c = (nseg + kWarps - 1) / kWarps;
  const int need = (nseg + c - 1) / c, warps = need < (int)DET_MAX_TOP / 32 ? (int)DET_MAX_TOP / 32 : need;
  const size_t smem = warps * kStageBytes<T>;
  if (cudaError_t e = raise_smem_cap((const void*)kern, smem)) return e;
  if (c > 8)
    if (cudaError_t e = allow_large_clusters((const void*)kern)) return e;
  const int fit = resident_clusters((const void*)kern, c, 32 * warps, smem);
  return launch_clusters(s, kern, L.n < fit ? L.n : fit, c, 32 * warps, smem, L, tokens, id_bytes, te, temp, in, loss,
                         o, static_cast<T*>(out), out_ld, 1.0f);
}
cudaError_t launch_step(cudaStream_t s, int dtype, const Logits& L, const void* tokens, int id_bytes,
                        const Teacher& te, float temp, const GradIn& in, float* loss, const ScoreOut& o, void* out,
                        unsigned long long out_ld) {
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return in.gh ? step_as<T, true>(s, L, tokens, id_bytes, te, temp, in, loss, o, out, out_ld)
                 : step_as<T, false>(s, L, tokens, id_bytes, te, temp, in, loss, o, out, out_ld);
  });
}

// ---- argument checks ----------------------------------------------------------------
size_t dtype_size(int dtype) { return dtype == DET_DTYPE_F32 ? 4 : 2; }

det_status check_logits(const void* logits, int dtype, uint32_t n, uint32_t vocab, uint64_t ld) {
  if (!logits || dtype < DET_DTYPE_F32 || dtype > DET_DTYPE_BF16) return DET_ERR_INVALID_ARGUMENT;
  if (vocab == 0) return DET_ERR_CDF_EMPTY;
  if (vocab > kMaxVocab) return DET_ERR_CDF_TOO_MANY_SYMBOLS;
  if (n > DET_SCORE_MAX_ROWS || ld > (1ull << 40)) return DET_ERR_INVALID_ARGUMENT;
  if ((uintptr_t)logits % dtype_size(dtype)) return DET_ERR_INVALID_ARGUMENT;
  return DET_OK;
}
// the gradient goes over the logits exactly, or nowhere near them: equal
// strides side by side, or ranges that do not meet
det_status check_grad(const void* logits, int dtype, uint32_t n, uint32_t vocab, uint64_t ld, const void* grad,
                      uint64_t grad_ld) {
  if (!grad || (n > 1 && grad_ld < vocab) || grad_ld > (1ull << 40)) return DET_ERR_INVALID_ARGUMENT;
  const size_t sz = dtype_size(dtype);
  if ((uintptr_t)grad % sz) return DET_ERR_INVALID_ARGUMENT;
  const uintptr_t a = (uintptr_t)logits, b = (uintptr_t)grad;
  if (a == b) return n == 1 || ld == grad_ld ? DET_OK : DET_ERR_INVALID_ARGUMENT;
  const size_t an = ((size_t)(n - 1) * ld + vocab) * sz, bn = ((size_t)(n - 1) * grad_ld + vocab) * sz;
  if (a + an <= b || b + bn <= a) return DET_OK;
  if (n == 1 || ld != grad_ld) return DET_ERR_INVALID_ARGUMENT;
  const size_t pitch = ld * sz, off = (b > a ? b - a : pitch - (a - b) % pitch) % pitch, row = vocab * sz;
  return off >= row && off + row <= pitch ? DET_OK : DET_ERR_INVALID_ARGUMENT;
}
det_status check_ids(const void* ids, int id_bytes) {
  if (!ids || (id_bytes != 4 && id_bytes != 8) || (uintptr_t)ids % id_bytes) return DET_ERR_INVALID_ARGUMENT;
  return DET_OK;
}
det_status check_list(const void* ids, int id_bytes, const void* teacher, int teacher_dtype, uint32_t k, uint32_t n,
                      uint64_t ld, float temperature) {
  if (det_status st = check_ids(ids, id_bytes)) return st;
  if (!teacher || teacher_dtype < DET_DTYPE_F32 || teacher_dtype > DET_DTYPE_BF16 ||
      (uintptr_t)teacher % dtype_size(teacher_dtype))
    return DET_ERR_INVALID_ARGUMENT;
  if (k == 0 || k > DET_MAX_TOP || (n > 1 && ld < k) || ld > (1ull << 40)) return DET_ERR_INVALID_ARGUMENT;
  if (!(temperature >= DET_MIN_TEMPERATURE && temperature <= DET_MAX_TEMPERATURE)) return DET_ERR_INVALID_ARGUMENT;
  return DET_OK;
}
det_status check_workspace(const void* workspace, size_t size, int dtype, uint32_t n, uint32_t vocab, uint32_t top) {
  if (!workspace || (uintptr_t)workspace % 16 || size < workspace_bytes(dtype, (int)n, (int)vocab, (int)top))
    return DET_ERR_INVALID_ARGUMENT;
  return DET_OK;
}
det_status check_device() {
  int cnt = 0;
  return cudaGetDeviceCount(&cnt) != cudaSuccess || cnt == 0 ? DET_ERR_NO_DEVICE : DET_OK;
}
det_status launched(cudaError_t e) {
  return e == cudaSuccess ? DET_OK : e == cudaErrorMemoryAllocation ? DET_ERR_DEVICE_OOM : DET_ERR_CUDA;
}

const Teacher kNoTeacher{nullptr, nullptr, 0, 4, DET_DTYPE_F32, 0};

}  // namespace

cudaError_t launch_token_scores(const Launch& L, const float* logits, int V, const uint32_t* rows,
                                const uint32_t* tokens, int n, int top, float* logprob, float* entropy,
                                int32_t* top_ids, float* top_logprobs, void* workspace) {
  const Logits x{logits, rows, (unsigned long long)V, n, V};
  const ScoreOut o{logprob, entropy, nullptr, top_ids, top_logprobs, top, L.err};
  if (L.launches) *L.launches += 2;
  return launch_forward(L.stream, DET_DTYPE_F32, x, tokens, 4, kNoTeacher, 1.0f, workspace, nullptr, o);
}
cudaError_t launch_distill_loss(const Launch& L, const float* logits, int V, const uint32_t* rows, int n,
                                const int32_t* ids, const float* teacher, int k, float temperature, float* loss,
                                void* workspace) {
  const Logits x{logits, rows, (unsigned long long)V, n, V};
  const Teacher te{ids, teacher, (unsigned long long)k, 4, DET_DTYPE_F32, k};
  const ScoreOut o{nullptr, nullptr, nullptr, nullptr, nullptr, 0, L.err};
  if (L.launches) *L.launches += 2;
  return launch_forward(L.stream, DET_DTYPE_F32, x, nullptr, 4, te, temperature, workspace, loss, o);
}

size_t scores_workspace_bytes(int n, int V, int top) { return workspace_bytes(DET_DTYPE_F32, n, V, top); }

static_assert(DET_SCORE_NONFINITE == (int)ERRF_CDF_NONFINITE && DET_SCORE_BAD_TOKEN == (int)ERRF_SYMBOL,
              "the flags are the session's error bits");
}  // namespace det

using namespace det;

extern "C" {

size_t det_scores_workspace(int dtype, uint32_t n, uint32_t vocab, uint32_t top) {
  if (dtype < DET_DTYPE_F32 || dtype > DET_DTYPE_BF16 || vocab > kMaxVocab || n > DET_SCORE_MAX_ROWS) return 0;
  return workspace_bytes(dtype, (int)n, (int)vocab, (int)top);
}

det_status det_token_scores_device(const void* logits, int dtype, uint32_t n, uint32_t vocab, uint64_t ld,
                                   const void* tokens, int token_bytes, uint32_t top, float* logprob, float* entropy,
                                   float* stats, int32_t* top_ids, float* top_logprobs, uint32_t* flags,
                                   void* workspace, size_t workspace_size, void* stream) {
  if (n == 0) return DET_OK;
  if (det_status st = check_logits(logits, dtype, n, vocab, ld)) return st;
  if (logprob)
    if (det_status st = check_ids(tokens, token_bytes)) return st;
  if (top > DET_MAX_TOP || top > vocab || (top && !top_ids && !top_logprobs)) return DET_ERR_INVALID_ARGUMENT;
  if (det_status st = check_workspace(workspace, workspace_size, dtype, n, vocab, top)) return st;
  if (det_status st = check_device()) return st;
  const Logits L{logits, nullptr, ld, (int)n, (int)vocab};
  const ScoreOut o{logprob, entropy, stats, top_ids, top_logprobs, (int)top, flags};
  return launched(launch_forward(static_cast<cudaStream_t>(stream), dtype, L, tokens, token_bytes, kNoTeacher, 1.0f,
                                 workspace, nullptr, o));
}

det_status det_token_scores_grad_device(const void* logits, int dtype, uint32_t n, uint32_t vocab, uint64_t ld,
                                        const void* tokens, int token_bytes, const float* stats,
                                        const float* grad_logprob, const float* grad_entropy, void* grad,
                                        uint64_t grad_ld, void* stream) {
  if (n == 0) return DET_OK;
  if (det_status st = check_logits(logits, dtype, n, vocab, ld)) return st;
  if (det_status st = check_grad(logits, dtype, n, vocab, ld, grad, grad_ld)) return st;
  if (!stats || (!grad_logprob && !grad_entropy)) return DET_ERR_INVALID_ARGUMENT;
  if (grad_logprob)
    if (det_status st = check_ids(tokens, token_bytes)) return st;
  if (det_status st = check_device()) return st;
  const Logits L{logits, nullptr, ld, (int)n, (int)vocab};
  return launched(launch_grad(static_cast<cudaStream_t>(stream), dtype, L, tokens, token_bytes, kNoTeacher, 1.0f,
                              GradIn{stats, grad_logprob, grad_entropy}, grad, grad_ld));
}

det_status det_token_scores_step_device(const void* logits, int dtype, uint32_t n, uint32_t vocab, uint64_t ld,
                                        const void* tokens, int token_bytes, const float* grad_logprob,
                                        const float* grad_entropy, float* logprob, float* entropy, float* stats,
                                        void* grad, uint64_t grad_ld, uint32_t* flags, void* stream) {
  if (n == 0) return DET_OK;
  if (det_status st = check_logits(logits, dtype, n, vocab, ld)) return st;
  if (det_status st = check_grad(logits, dtype, n, vocab, ld, grad, grad_ld)) return st;
  if (!stats || (!grad_logprob && !grad_entropy)) return DET_ERR_INVALID_ARGUMENT;
  if (logprob || grad_logprob)
    if (det_status st = check_ids(tokens, token_bytes)) return st;
  if (det_status st = check_device()) return st;
  const Logits L{logits, nullptr, ld, (int)n, (int)vocab};
  const ScoreOut o{logprob, entropy, stats, nullptr, nullptr, 0, flags};
  return launched(launch_step(static_cast<cudaStream_t>(stream), dtype, L, logprob || grad_logprob ? tokens : nullptr,
                              token_bytes, kNoTeacher, 1.0f, GradIn{nullptr, grad_logprob, grad_entropy}, nullptr, o,
                              grad, grad_ld));
}

det_status det_distill_loss_device(const void* logits, int dtype, uint32_t n, uint32_t vocab, uint64_t ld,
                                   const void* ids, int id_bytes, const void* teacher, int teacher_dtype, uint32_t k,
                                   uint64_t list_ld, float temperature, float* loss, float* stats, uint32_t* flags,
                                   void* workspace, size_t workspace_size, void* stream) {
  if (n == 0) return DET_OK;
  if (det_status st = check_logits(logits, dtype, n, vocab, ld)) return st;
  if (det_status st = check_list(ids, id_bytes, teacher, teacher_dtype, k, n, list_ld, temperature)) return st;
  if (!loss) return DET_ERR_INVALID_ARGUMENT;
  if (det_status st = check_workspace(workspace, workspace_size, dtype, n, vocab, 0)) return st;
  if (det_status st = check_device()) return st;
  const Logits L{logits, nullptr, ld, (int)n, (int)vocab};
  const Teacher te{ids, teacher, list_ld, id_bytes, teacher_dtype, (int)k};
  const ScoreOut o{nullptr, nullptr, stats, nullptr, nullptr, 0, flags};
  return launched(launch_forward(static_cast<cudaStream_t>(stream), dtype, L, nullptr, 4, te, temperature,
                                 workspace, loss, o));
}

det_status det_distill_grad_device(const void* logits, int dtype, uint32_t n, uint32_t vocab, uint64_t ld,
                                   const void* ids, int id_bytes, const void* teacher, int teacher_dtype, uint32_t k,
                                   uint64_t list_ld, float temperature, const float* stats, const float* grad_loss,
                                   void* grad, uint64_t grad_ld, void* stream) {
  if (n == 0) return DET_OK;
  if (det_status st = check_logits(logits, dtype, n, vocab, ld)) return st;
  if (det_status st = check_grad(logits, dtype, n, vocab, ld, grad, grad_ld)) return st;
  if (det_status st = check_list(ids, id_bytes, teacher, teacher_dtype, k, n, list_ld, temperature)) return st;
  if (!stats || !grad_loss) return DET_ERR_INVALID_ARGUMENT;
  if (det_status st = check_device()) return st;
  const Logits L{logits, nullptr, ld, (int)n, (int)vocab};
  const Teacher te{ids, teacher, list_ld, id_bytes, teacher_dtype, (int)k};
  return launched(launch_grad(static_cast<cudaStream_t>(stream), dtype, L, nullptr, 4, te, temperature,
                              GradIn{stats, grad_loss, nullptr}, grad, grad_ld));
}

det_status det_distill_step_device(const void* logits, int dtype, uint32_t n, uint32_t vocab, uint64_t ld,
                                   const void* ids, int id_bytes, const void* teacher, int teacher_dtype, uint32_t k,
                                   uint64_t list_ld, float temperature, const float* grad_loss, float* loss,
                                   float* stats, void* grad, uint64_t grad_ld, uint32_t* flags, void* stream) {
  if (n == 0) return DET_OK;
  if (det_status st = check_logits(logits, dtype, n, vocab, ld)) return st;
  if (det_status st = check_grad(logits, dtype, n, vocab, ld, grad, grad_ld)) return st;
  if (det_status st = check_list(ids, id_bytes, teacher, teacher_dtype, k, n, list_ld, temperature)) return st;
  if (!loss || !stats || !grad_loss) return DET_ERR_INVALID_ARGUMENT;
  if (det_status st = check_device()) return st;
  const Logits L{logits, nullptr, ld, (int)n, (int)vocab};
  const Teacher te{ids, teacher, list_ld, id_bytes, teacher_dtype, (int)k};
  const ScoreOut o{nullptr, nullptr, stats, nullptr, nullptr, 0, flags};
  return launched(launch_step(static_cast<cudaStream_t>(stream), dtype, L, nullptr, 4, te, temperature,
                              GradIn{nullptr, grad_loss, nullptr}, loss, o, grad, grad_ld));
}

}  // extern "C"
