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
// the library, and the order of every sum is fixed by the vocabulary and the
// element type alone, so a row has the same bits whatever batch or stride it
// is part of (the gradients of the step kernel and of the gradient kernel are
// scaled in another order and may differ in their last bits).  Sums and sums'
// joins are f32, logarithms and what is made of them 64 bits, and gradients
// are rounded once to the logits' type.  A row is cut into segments of 2,048
// entries; a warp takes a segment, its lane l the entries of 16-byte vectors l,
// l + 32, ... of it, and sums are relative to the segment's own maximum until
// the segments are joined.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstring>
#include <tuple>
#include <type_traits>

#include "../../include/detgpu.h"
#include "dev_math.cuh"
#include "internal.h"
#include "known.h"

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
// Within 7.1 * 2^-24 of 2^y from y = -123.953 on, and 0 below that: there the
// entry times 2^k is no normal number any more.
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
template <bool RO>
DI uint4 load16(const uint4* p) {
  if constexpr (RO) return __ldg(p);
  else return *p;
}
// The vector at entry `at` of a row (RO: that nothing writes from the kernel's
// launch on, so not in a kernel whose own pdl_wait() waits for the row); what is
// past the row's end is -inf.  Only 16-byte granules that lie in the row as a
// whole are loaded as such: a row that starts `mis` entries into a granule takes
// two of them.
template <typename T, bool RO = true>
DI uint4 row_vec(const T* row, int at, int V, int mis) {
  constexpr int VEC = Seg<T>::VEC;
  const T* p = row + at;
  if (mis == 0 && at + VEC <= V) return load16<RO>(reinterpret_cast<const uint4*>(p));
  if (mis != 0 && at >= mis && at - mis + 2 * VEC <= V) {
    const uint4* q = reinterpret_cast<const uint4*>(p - mis);
    return shifted(load16<RO>(q), load16<RO>(q + 1), mis * (int)sizeof(T));
  }
  float v[VEC];
#pragma unroll
  for (int j = 0; j < VEC; j++) v[j] = at + j < V ? to_f32(p[j]) : -INFINITY;
  return pack_vec<T>(v);
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
// segment i's sums.  WHOLE: w too; otherwise w only says if the row is bad (0
// or NaN).
template <bool WHOLE, typename F>
DI Sums join_segments(F at, int nseg, float c, uint32_t table, float one) {
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
    const float f = un(exp2_warp<true>(pk(y, y), table, pk(one, one)).e).x;
    s = fadd(s, fmul(f, t[i].s));
    // sum of 2^(y_j + y) (y_j + y) = f (w + y s); NaN stays NaN
    if constexpr (WHOLE) w = fadd(w, fmul(f, fadd(t[i].w, fmul(y, t[i].s))));
    else if (__any_sync(kFull, !(t[i].w == t[i].w))) w = __int_as_float(0x7fffffff);
  }
  if constexpr (WHOLE) {
    const float v = warp_sum2(s, w);
    return {m, __shfl_sync(kFull, v, 0), __shfl_sync(kFull, v, 16)};
  }
  return {m, warp_sum(s), w};
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
constexpr int kListWarps = 16;  // of a block that takes a row's list, at most
struct ListShared {
  float max[kListWarps], sum[kListWarps];
  int bad[kListWarps], some[kListWarps];
  int id[DET_MAX_TOP];
  float q[DET_MAX_TOP];
  double term[kListWarps];
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
DI ListEntry teacher_entry(const Teacher& te, int row, int vocab, float c, uint32_t table, float one,
                           ListShared& sh) {
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
  const float y = fmul(r.d, c), p = un(exp2_warp<true>(pk(y, y), table, pk(one, one)).e).x, e = valid ? p : 0.0f;
  const float ws = warp_sum(e);
  if (l == 0) sh.sum[w] = ws;
  __syncthreads();
  r.s = 0.0f;
  for (int i = 0; i < nw; i++) r.s = fadd(r.s, sh.sum[i]);
  r.id = valid ? (int)id : -1;
  r.q = valid ? fdiv(e, r.s) : 0.0f;
  return r;
}
// log q of the thread's entry, in 64 bits
DI double list_logq(const ListEntry& e, float temp) {
  return e.id >= 0 ? dsub(ddiv((double)e.d, (double)temp), log_det((double)e.s)) : 0.0;
}
// the row's loss, in thread 0; z: the logit at the thread's entry.  Ends with
// the block in step.
DI float list_loss(const ListEntry& e, double logq, float z, const RowStats& r, double log_s, float temp,
                   ListShared& sh) {
  double term = 0.0;
  if (e.id >= 0 && e.q > 0.0f) {
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
// the k largest, so only those are read again.  A group is what 32, 8 or 1
// lanes load at once (2^lg lanes of 16 bytes): the largest of them that leaves
// 2 k groups, so that the entries above the k-th largest maximum are not many
// more than k.  That is never more than kMaxGroups.
constexpr int kRowThreads = DET_MAX_TOP;  // of a row's block: a thread per list entry
constexpr int kMaxGroups = 2048;
constexpr int kCand = 2304;               // keys held before they are cut down to k
__host__ __device__ constexpr int group_lanes_log2(int V, int k, int vec) {
  return V >= 2 * k * 32 * vec ? 5 : V >= 2 * k * 8 * vec ? 3 : 0;
}
struct TopShared {
  unsigned long long key[kCand];
  int bin[256];
  uint16_t group[kMaxGroups];
  int count, groups, bits[3], floor_bin;
  uint32_t lo, hi;
};

// The largest t that at least k of the block's values (distinct, or 0) reach,
// bit by bit; done early once exactly k do.
template <int PER>
DI unsigned long long kth_largest(const unsigned long long (&v)[PER], int k, TopShared& sh) {
  unsigned long long t = 0;
  for (int bit = 63, turn = 0; bit >= 0; bit--) {
    const unsigned long long cand = t | (1ull << bit);
    int c = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) c += v[i] >= cand;
    c = __reduce_add_sync(kFull, c);
    if ((threadIdx.x & 31) == 0 && c) atomicAdd(&sh.bits[turn], c);
    __syncthreads();
    const int all = sh.bits[turn];
    // the counter of the turn before: everyone has read it, and it is used
    // again in two turns, behind another barrier
    const int before = turn == 0 ? 2 : turn - 1;
    if (threadIdx.x == 0) sh.bits[before] = 0;
    turn = turn == 2 ? 0 : turn + 1;
    if (all >= k) t = cand;
    if (all == k) break;
  }
  __syncthreads();
  if (threadIdx.x < 3) sh.bits[threadIdx.x] = 0;
  __syncthreads();
  return t;
}
// keeps the k largest of the block's sh.count keys (distinct); returns the
// smallest of them, or 0 if there are fewer than k
DI unsigned long long cut_to(int k, TopShared& sh) {
  __syncthreads();
  const int n = min(sh.count, kCand);
  __syncthreads();
  if (n <= k) return 0;
  constexpr int PER = kCand / kRowThreads;
  unsigned long long v[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int at = i * kRowThreads + threadIdx.x;
    v[i] = at < n ? sh.key[at] : 0;
  }
  const unsigned long long t = kth_largest<PER>(v, k, sh);
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; i++)
    if (v[i] >= t) sh.key[atomicAdd(&sh.count, 1)] = v[i];
  __syncthreads();
  return t;
}
// adds the entries of a vector whose keys are above `floor`
template <typename T>
DI void push_vec(uint4 w, int at, int V, unsigned long long floor, TopShared& sh) {
  float v[Seg<T>::VEC];
  unpack_vec<T>(w, v);
#pragma unroll
  for (int j = 0; j < Seg<T>::VEC; j++) {
    const unsigned long long key = top_key(v[j], (uint32_t)(at + j));
    if (at + j < V && key > floor) {
      const int slot = atomicAdd(&sh.count, 1);
      if (slot < kCand) sh.key[slot] = key;
    }
  }
}
// The row's k largest keys, in order, to sh.key[0 .. k); PER groups per thread
// cover them all.  `meanwhile` runs while their maxima are on their way; the
// list is not made where it gives false.
template <typename T, int PER, typename F>
DI void top_list(const T* __restrict__ x, int V, int mis, const float* gmax, int k, TopShared& sh, F meanwhile) {
  constexpr int VEC = Seg<T>::VEC;
  const int lg = group_lanes_log2(V, k, VEC), size = VEC << lg, ng = (V + size - 1) / size;
  const int tid = threadIdx.x, l = tid & 31;
  float f[PER];
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int g = i * kRowThreads + tid;
    f[i] = g < ng ? gmax[g] : 0.0f;
  }
  if (!meanwhile()) return;
  // the maxima, as ordered integers
  uint32_t v[PER], lo = ~0u, hi = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int g = i * kRowThreads + tid;
    v[i] = g < ng ? (uint32_t)(top_key(f[i], 0) >> 32) : 0u;
    hi = max(hi, v[i]);
    if (g < ng) lo = min(lo, v[i]);
  }
  if (tid == 0) sh.count = sh.groups = sh.bits[0] = sh.bits[1] = sh.bits[2] = 0, sh.lo = ~0u, sh.hi = 0;
  for (int i = tid; i < 256; i += kRowThreads) sh.bin[i] = 0;
  __syncthreads();
  hi = __reduce_max_sync(kFull, hi);
  lo = __reduce_min_sync(kFull, lo);
  if (l == 0) {
    atomicMax(&sh.hi, hi);
    atomicMin(&sh.lo, lo);
  }
  __syncthreads();
  // a value that at least k of them reach: the lower end of the bin, of 256
  // between the smallest and the largest, that the k-th largest is in.  The bins
  // are equally wide in the ordered integers: with a maximum of 0 or less among
  // them they span exponents down to 0, and many groups reach the floor.
  uint32_t floor = 0;
  if (ng > k) {
    lo = sh.lo;
    const int shift = max(0, 24 - __clz((int)(sh.hi - lo)));
#pragma unroll
    for (int i = 0; i < PER; i++)
      if (i * kRowThreads + tid < ng) atomicAdd(&sh.bin[(v[i] - lo) >> shift], 1);
    __syncthreads();
    if (tid < 32) {
      int own = 0, c[8];
#pragma unroll
      for (int i = 0; i < 8; i++) own += c[i] = sh.bin[8 * l + i];
      int above = own;  // of this lane's bins and those above
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_down_sync(kFull, above, o);
        if (l + o < 32) above += t;
      }
      if (above >= k && above - own < k) {
        int n = above - own, b = 7;
        while ((n += c[b]) < k) b--;
        sh.floor_bin = 8 * l + b;
      }
    }
    __syncthreads();
    floor = lo + ((uint32_t)sh.floor_bin << shift);
  }
  // the groups that reach it
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int g = i * kRowThreads + tid;
    const bool in = g < ng && v[i] >= floor;
    const unsigned who = __ballot_sync(kFull, in);
    int base = 0;
    if (l == 0 && who) base = atomicAdd(&sh.groups, __popc(who));
    base = __shfl_sync(kFull, base, 0);
    if (in) sh.group[base + __popc(who & ((1u << l) - 1))] = g;
  }
  __syncthreads();
  const int items = sh.groups << lg;
  const bool few = sh.groups <= 4 * k + 64;
  unsigned long long key_floor = floor ? ((unsigned long long)floor << 32) - 1 : 0;
  if (few) {
    // the usual case: their vectors, as many as can be on their way at once
    constexpr int U = 8;
    for (int j0 = tid; j0 < items; j0 += U * kRowThreads) {
      uint4 w[U];
      int at[U];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int j = j0 + u * kRowThreads;
        at[u] = j < items ? ((sh.group[j >> lg] << lg) + (j & ((1 << lg) - 1))) * VEC : V;
        if (at[u] < V) w[u] = row_vec<T>(x, at[u], V, mis);
      }
#pragma unroll
      for (int u = 0; u < U; u++)
        if (at[u] < V) push_vec<T>(w[u], at[u], V, key_floor, sh);
    }
  }
  __syncthreads();
  if (!few || sh.count > kCand) {
    // too many groups or entries reach the floor (ties, a row in order, or a wide
    // bin): group by group in the order of their indices, cutting the list down
    // as it fills, which raises the floor and passes over the groups that cannot
    // add to it.  1,024 rows of 128,256 f32, top 20: 376 us with the last 256
    // entries masked out, 126 without.
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
    const int step = max(1, (kCand - (int)DET_MAX_TOP) / size);
    int g = 0;
    while (g < ng) {
      // as many groups as surely fit, of those that can add something
      const int room = (kCand - sh.count) / size;
      __syncthreads();
      int g1 = g;
      if (room > 0) {
        g1 = min(ng, g + min(step, room));
        for (int j = tid; j < (g1 - g) << lg; j += kRowThreads) {
          const int q = g + (j >> lg), a = ((g << lg) + j) * VEC;
          if (a < V && top_key(gmax[q], (uint32_t)(q * size)) > key_floor)
            push_vec<T>(row_vec<T>(x, a, V, mis), a, V, key_floor, sh);
        }
      }
      g = g1;
      __syncthreads();
      if (sh.count > kCand - size) {
        const unsigned long long t = cut_to(k, sh);
        if (t) key_floor = t;
      }
      __syncthreads();
    }
  }
  if (sh.count > 2 * kRowThreads) cut_to(k, sh);
  __syncthreads();
  // at most two keys per thread are left: each finds its rank
  const int n = sh.count, second = kRowThreads + tid;
  const unsigned long long a = tid < n ? sh.key[tid] : 0, b = second < n ? sh.key[second] : 0;
  int ra = 0, rb = 0;
  for (int i = 0; i < n; i++) {
    const unsigned long long o = sh.key[i];
    ra += o > a;
    rb += o > b;
  }
  __syncthreads();
  if (a && ra < k) sh.key[ra] = a;
  if (b && rb < k) sh.key[rb] = b;
  __syncthreads();
}

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
// row joins the row's segments and writes its results.  (One kernel with a
// block or cluster per row loses to uneven rounds of rows and at the rows'
// ends: 136 us against 122 for 1,024 rows of 128,256 f32 logits, with the same
// arithmetic and the cache flushed before each.)
//
// The first kernel reads each logit once.  1,024 rows of 128,256 f32: 90 us,
// 5.8 TB/s of 6.5 copied; of 151,936 bf16: 90 us, 3.5 TB/s.  The latter is
// bound by issue slots: 11.6 instructions per 32 entries, of which the 5.5
// packed ones take two slots each, fill 87% of them.  Other numbers of warps
// and blocks per SM measured the same or up to 5% slower, segments of 1,024
// entries 20% slower.  The second takes 9 us for 1,024 rows, 20 us with lists
// of 20.
struct Workspace {
  float4* seg;  // [rows][segments]: m, s, w
  float* gmax;  // [rows][groups]
};
// LG: which maxima a top list needs, of 2^LG lanes' vectors; -1: none
template <typename T, int LG>
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
  const float c = fdiv(kLog2e, temp);
  const uint32_t table = kExpTable[l];
  pdl_enter();
  if (row < L.n) stage_issue<T>(stage, at_row(row), g, V);
  while (row < L.n) {
    uint4 v[G::NV];
    stage_take<T>(stage, misaligned(at_row(row)), v);
    int nrow = row + drow, ng = g + dg;
    if (ng >= nseg) ng -= nseg, nrow++;
    if (nrow < L.n) stage_issue<T>(stage, at_row(nrow), ng, V);
    Range<T> all_range;
    float gm = -INFINITY;
    const size_t part = (size_t)row * nseg + g;
    float* gmax = ws.gmax + ((part * (kSeg / G::VEC)) >> (LG < 0 ? 0 : LG));
#pragma unroll
    for (int i = 0; i < G::NV; i++) {
      all_range.take(v[i]);
      if constexpr (LG >= 0) {
        Range<T> group;
        group.take(v[i]);
        float gh = group.high();
        if constexpr (LG == 5) {
          gh = redux_max(gh);
          if (l == i) gm = gh;
        } else {
          for (int o = 1; o < 1 << LG; o <<= 1) gh = fmaxf(gh, __shfl_xor_sync(kFull, gh, o));
          if ((l & ((1 << LG) - 1)) == 0) gmax[(i * 32 + l) >> LG] = gh;
        }
      }
    }
    if constexpr (LG == 5) {
      if (l < G::NV) gmax[l] = gm;
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
__global__ void __launch_bounds__(kRowThreads, 7)
    rows_kernel(Logits L, const void* tokens, int id_bytes, Teacher te, float temp, Workspace ws, float* loss,
                ScoreOut o, float one) {
  __shared__ ListShared list;
  const int row = blockIdx.x, V = L.vocab, nseg = (V + kSeg - 1) / kSeg;
  const T* x = static_cast<const T*>(L.x) + (size_t)(L.rows ? L.rows[row] : row) * L.ld;
  const float c = fdiv(kLog2e, temp), nan = __int_as_float(0x7fffffff);
  const uint32_t table = kExpTable[threadIdx.x & 31];
  // what does not depend on the sums, while they are being taken: inputs of the
  // call, which are complete, as segments_kernel waits before it triggers
  ListEntry e;
  float z = 0.0f;
  double logq = 0.0;
  long long t = -1;
  if (loss) {
    e = teacher_entry(te, row, V, c, table, one, list);
    if (e.id >= 0) z = to_f32(x[e.id]);
    logq = list_logq(e, temp);
  } else if (o.logprob) {
    t = load_id(tokens, id_bytes, row);
    if (t >= 0 && t < V) z = to_f32(x[t]);
  }
  pdl_wait();
  RowStats r;
  double log_s;
  auto scores = [&]() {
    const float4* seg = ws.seg + (size_t)row * nseg;
    r = finish_row(join_segments<true>(
        [&](int i) {
          const float4 f = seg[i];
          return Sums{f.x, f.y, f.z};
        },
        nseg, c, table, one));
    log_s = log_sum(r);
    if (threadIdx.x == 0) {
      if (o.stats) write_stats(o.stats, row, r, log_s);
      if (r.bad && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_NONFINITE);
      if (!loss) write_scores(o, row, V, r, log_s, t, z);
      if (t >= V && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_BAD_TOKEN);
    }
    return !r.bad;
  };
  if constexpr (TOP) {
    __shared__ TopShared top;
    const int lg = group_lanes_log2(V, o.top, Seg<T>::VEC);
    const float* gmax = ws.gmax + (((size_t)row * nseg * (kSeg / Seg<T>::VEC)) >> lg);
    if (V <= (Seg<T>::VEC << lg) * 8 * kRowThreads) top_list<T, 8>(x, V, misaligned(x), gmax, o.top, top, scores);
    else top_list<T, kMaxGroups / kRowThreads>(x, V, misaligned(x), gmax, o.top, top, scores);
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
  } else {
    scores();
    if (loss) {
      const float v = list_loss(e, logq, z, r, log_s, temp, list);
      if (threadIdx.x == 0) {
        loss[row] = v;
        if (e.bad && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_BAD_TOKEN);
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

// Bound by memory for f32 logits, which are read and written once: 166 us for
// 1,024 rows of 128,256, 6.3 TB/s of 6.5 copied.  For 16-bit logits at 5.5 TB/s
// (113 us for 1,024 rows of 151,936 bf16), where half of the issue slots are
// used and warps wait for loads and at the block's start.
//
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
  const float c = fdiv(kLog2e, temp);
  const uint32_t table = kExpTable[l];
  uint4 cur[U];
  pdl_enter();
  if (q0 + w * kGradRun < q1) fetch(q0 + w * kGradRun, cur);
  const float* st = in.stats + (size_t)row * 4;
  const float m = st[0], s = st[1];
  RowGrad r;
  int id;
  float add;
  if (te.k) {
    ListEntry e = teacher_entry(te, row, V, c, table, one_, sh);
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
  if (my == 0 && lo + kSeg <= V) {
    uint4* p = reinterpret_cast<uint4*>(y + lo) + l;
#pragma unroll
    for (int i = 0; i < G::NV; i++) p[32 * i] = vec(i);
    return;
  }
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

// Three kernels.  The first gathers what the gradient's coefficients and the
// logits at a row's own tokens are, before `out` may overwrite those.  The
// third writes the rows' scores and adds the part of their own tokens.
//
// In the second, clusters draw rows; each of a cluster's warps holds one
// segment of the row, so the row is read once: its exponentials stay in
// registers until all segments' sums are there, and are scaled and stored
// then, while the next row's segment is on its way.  (The entropy's gradient
// needs y too: it keeps the logits and takes their exponentials again.)  A
// warp sends its sums to every block of the cluster, where an mbarrier counts
// their bytes: no barrier that all warps stop at, and no fence, which would
// also wait for the last row's stores and the next segment's copies.  The sums
// have two places and two mbarriers; a warp sends the row after next only when
// it has the next row's sums, which every warp sent after it read the row's.
//
// 1,024 rows of 128,256 bf16 logits: 147 us, memory read and written once in 81
// us; 177 us with a cluster barrier per row, 182 us as sums and gradient over
// memory, 190 us and more as tasks that a persistent grid draws, sums a chunk
// of rows ahead of gradients that find their logits in the L2 cache (two passes'
// instructions).  Bound by the exchange: a warp has half of its time nothing to
// do until the row's slowest segment has sent its sums, and 64 exponentials per
// lane leave registers for 16 warps per SM.
struct StepWork {
  float4* coef;      // per row: of the loss over T, or of minus logprob; of the entropy; 1 where all is zeros
  float* z;          // per row and entry: the logit at its token
  uint32_t* ticket;  // [0]: rows drawn; [1]: not 0 once a wait has run out
};
template <typename T>
__global__ void __launch_bounds__(kThreads)
    step_gather_kernel(Logits L, const void* tokens, int id_bytes, Teacher te, float temp, GradIn in, StepWork ws,
                       uint32_t first) {
  const int row = blockIdx.x * kWarps + (threadIdx.x >> 5), l = threadIdx.x & 31, V = L.vocab;
  // Every block waits, and none triggers before it does (none triggers at all):
  // the next two kernels read the call's inputs before their own waits.
  pdl_wait();
  if (row >= L.n) return;
  if (row == 0 && l == 0) ws.ticket[0] = first, ws.ticket[1] = 0;
  const T* x = static_cast<const T*>(L.x) + (size_t)row * L.ld;
  const float nan = __int_as_float(0x7fffffff);
  if (te.k) {
    bool some = false, bad = false;
    for (int i = l; i < te.k; i += 32) {
      const long long id = load_id(te.ids, te.id_bytes, (size_t)row * te.ld + i);
      if (id < 0) continue;
      const float u = load_any(te.u, te.dtype, (size_t)row * te.ld + i);
      bad |= id >= V || !(u < INFINITY);
      some |= u > -INFINITY;
      if (id < V) ws.z[(size_t)row * te.k + i] = to_f32(x[id]);
    }
    some = __any_sync(kFull, some);
    bad = __any_sync(kFull, bad);
    if (l == 0)
      ws.coef[row] = make_float4(bad ? nan : fdiv(in.g[row], temp), 0.0f, !some && !bad ? 1.0f : 0.0f, 0.0f);
  } else if (l == 0) {
    const long long t = tokens ? load_id(tokens, id_bytes, row) : -1;
    if (t >= 0 && t < V) ws.z[row] = to_f32(x[t]);
    const float gl = !in.g || t < 0 ? 0.0f : t >= V ? nan : in.g[row];
    ws.coef[row] = make_float4(-gl, in.gh ? in.gh[row] : 0.0f, 0.0f, 0.0f);
  }
}
// the coefficients of a row: a_g, a_h as in StepWork, of the loss over T or of
// minus the logprob, and of the entropy
DI RowGrad row_grad(float a_g, float a_h, bool zero, const RowStats& r, float c) {
  const float inv_s = fdiv(1.0f, r.s);
  const float a = a_h == 0.0f ? a_g : fadd(a_g, fmul(a_h, fdiv(r.s1, r.s)));
  return {-r.m, c, fmul(a, inv_s), fmul(fmul(-a_h, kLn2), inv_s), zero || r.empty};
}
// The gradient of segment g of a row with maximum m to y, from its logits
// (ENTROPY) or from their exponentials under the segment's maximum.
template <typename T, bool ENTROPY>
DI void grad_segment(const uint4 (&raw)[Seg<T>::NV], const float* v, float m_seg, float m, const RowGrad& rg, float c,
                     uint32_t table, float one_, T* y, int g, int V) {
  using G = Seg<T>;
  const f2 one = pk(one_, one_), cc = pk(c, c);
  const float y_seg = segment_y(m_seg, m, c);
  const float f = fmul(un(exp2_warp<true>(pk(y_seg, y_seg), table, one).e).x, rg.as);
  // vector i of the segment's gradient
  auto vec = [&](int i) {
    constexpr int VEC = G::VEC;
    if (rg.zero) return make_uint4(0, 0, 0, 0);
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
      x[j] = dv.x;
      x[j + 1] = dv.y;
    }
    return pack_vec<T>(x);
  };
  store_segment<T>(y, g, V, misaligned(y), vec);
}
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
DI void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
DI uint32_t shared_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// the address of one's own shared memory in block `rank` of the cluster
DI uint32_t remote(uint32_t p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(p), "r"(rank));
  return r;
}
// 16 bytes to a block of the cluster, counted by its mbarrier (in a launch with
// clusters: without them the instruction is not there)
DI void send(uint32_t at, uint32_t bar, float4 v) {
  asm volatile(
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(at),
      "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(bar)
      : "memory");
}
DI bool bar_done(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// waits for the barrier's phase, `limit_ns` at most (and min_tries at least, as
// the clock runs on while the GPU does something else)
DI bool bar_wait(uint32_t bar, uint32_t parity, unsigned long long limit_ns, int min_tries) {
  if (bar_done(bar, parity)) return true;
  unsigned long long t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  int tries = 0;
  do {
    if (bar_done(bar, parity)) return true;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  } while (++tries < min_tries || t - t0 < limit_ns);
  return false;
}
// SELFTEST: waits of 20 ms, one of which runs out: the last block of the first
// cluster expects one arrival more than comes on its second barrier.
template <bool SELFTEST>
struct StepWait {
  static constexpr unsigned long long ns = SELFTEST ? 20000000ull : 1000000000ull;
  static constexpr int tries = SELFTEST ? 16 : 4096;
};
template <typename T, bool ENTROPY, bool SELFTEST = false>
__global__ void __launch_bounds__(kThreads, 2)
    step_kernel(Logits L, float temp, StepWork ws, float* stats, T* out, unsigned long long out_ld, float one_) {
  using G = Seg<T>;
  __shared__ float4 seg[2][kMaxSegs];
  __shared__ __align__(8) unsigned long long bars[2];
  extern __shared__ __align__(16) uint8_t dyn[];
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int V = L.vocab, w = threadIdx.x >> 5, l = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int nseg = (V + kSeg - 1) / kSeg, clusters = gridDim.x / size;
  const int g = rank * warps + w;
  const bool active = g < nseg;
  void* stage = dyn + w * kStageBytes<T>;
  auto at_row = [&](int r) { return static_cast<const T*>(L.x) + (size_t)r * L.ld; };
  int row = blockIdx.x / size, next = row + clusters;
  // before pdl_wait(): the logits are complete, as step_gather_kernel has waited
  // in all blocks, and only this kernel writes over them.  The kernel after this
  // one reads inputs alone before its wait, so it may be launched already.
  if (active) stage_issue<T>(stage, at_row(row), g, V);
  pdl_trigger();
  const float c = fdiv(kLog2e, temp);
  const uint32_t table = kExpTable[l], bar = shared_at(bars);
  if (threadIdx.x == 0) {
    // a lone block's warps arrive themselves
    const int count = size > 1 ? 1 : nseg;
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\nmbarrier.init.shared::cta.b64 [%0 + 8], %2;" ::"r"(bar),
                 "r"(count), "r"(SELFTEST && blockIdx.x == size - 1 ? count + 1 : count)
                 : "memory");
    if (size > 1) asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // the barriers are set before anyone sends to them
  if (size > 1) cluster_sync();
  else __syncthreads();
  pdl_wait();  // the first kernel's results are there, and its reads done
  const uint32_t to = l < (int)size ? l : 0;
  const uint32_t place = remote(shared_at(&seg[0][g < kMaxSegs ? g : 0]), to), to_bar = remote(bar, to);
  if (active) {
    for (int turn = 0; row < L.n; turn++) {
      const int half = turn & 1;
      uint4 raw[G::NV];
      float v[ENTROPY ? 1 : kPerLane];
      // block 0's first warp draws the row after next, which goes with its sums
      uint32_t after = 0;
      if (g == 0 && l == 0) after = atomicAdd(ws.ticket, 1u);
      if (size > 1 && threadIdx.x == 0)
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar + 8 * half), "r"(16 * nseg)
                     : "memory");
      const float4 coef = ws.coef[row];
      stage_take<T>(stage, misaligned(at_row(row)), raw);
      if (next < L.n) stage_issue<T>(stage, at_row(next), g, V);
      Range<T> range;
#pragma unroll
      for (int i = 0; i < G::NV; i++) range.take(raw[i]);
      const float m_seg = redux_max(range.high());
      const float sum = segment_sums<T, !ENTROPY>(raw, V - g * kSeg, m_seg, redux_min(range.low()), c, table, one_, v);
      const float s_seg = __shfl_sync(kFull, sum, 0), w_seg = __shfl_sync(kFull, sum, 16);
      after = __shfl_sync(kFull, after, 0);
      const float4 mine = make_float4(m_seg, s_seg, w_seg, __uint_as_float(after));
      if (size > 1) {
        if (l < (int)size) send(place + half * (uint32_t)sizeof(seg[0]), to_bar + 8 * half, mine);
      } else if (l == 0) {
        seg[half][g] = mine;
        asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(bar + 8 * half) : "memory");
      }
      // The wait ends: the other warps run, and send what this one waits for
      // without waiting for this row.  Should it run out, the warp says so and
      // leaves behind this row, without sending again, so the cluster's other
      // warps' waits run out too and the rows it had drawn stay undone: the next
      // kernel makes all of the call's results NaN.
      using Wait = StepWait<SELFTEST>;
      const bool there = __all_sync(kFull, bar_wait(bar + 8 * half, (turn >> 1) & 1, Wait::ns, Wait::tries));
      if (!there && l == 0) atomicOr(ws.ticket + 1, 1u);
      auto sums_of = [&](int i) {
        const float4 f = seg[half][i];
        return Sums{f.x, f.y, f.z};
      };
      // the sum of 2^y y is for the entropy's gradient, and for one warp to write
      const RowStats r = finish_row(ENTROPY || g == 0 ? join_segments<true>(sums_of, nseg, c, table, one_)
                                                      : join_segments<false>(sums_of, nseg, c, table, one_));
      const int drawn = (int)__float_as_uint(seg[half][0].w);
      const RowGrad rg = row_grad(coef.x, coef.y, coef.z != 0.0f, r, c);
      if (g == 0 && l == 0) {
        float* st = stats + (size_t)row * 4;
        st[0] = r.m, st[1] = r.s, st[2] = r.s1;
      }
      grad_segment<T, ENTROPY>(raw, v, m_seg, r.m, rg, c, table, one_, out + (size_t)row * out_ld, g, V);
      row = there ? next : L.n;
      next = drawn;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");  // of a warp that left early
  }
  // nobody leaves while another block may still send to it
  if (size > 1) {
    __syncwarp();
    cluster_sync();
  }
}
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(kRowThreads)
    step_rows_kernel(Logits L, const void* tokens, int id_bytes, Teacher te, float temp, GradIn in, StepWork ws,
                     float* loss, ScoreOut o, T* out, unsigned long long out_ld, float one) {
  __shared__ ListShared list;
  const int row = blockIdx.x, V = L.vocab;
  const float c = fdiv(kLog2e, temp);
  const uint32_t table = kExpTable[threadIdx.x & 31];
  ListEntry e;
  double logq = 0.0;
  long long t = -1;
  int id, own;
  float share = 0.0f;
  // the call's inputs, complete since step_gather_kernel waited
  if (loss) {
    e = teacher_entry(te, row, V, c, table, one, list);
    logq = list_logq(e, temp);
    own = e.id;
    ListEntry f = e;
    share = list_share(f, te.k, list);
    id = f.id;
  } else {
    t = tokens ? load_id(tokens, id_bytes, row) : -1;
    own = id = threadIdx.x == 0 && t >= 0 && t < V ? (int)t : -1;
  }
  pdl_wait();
  const float z = own >= 0 ? ws.z[(size_t)row * (loss ? te.k : 1) + threadIdx.x] : 0.0f;
  const float4 coef = ws.coef[row];
  // a wait ran out: whichever rows were not finished, all of them are NaN
  const bool lost = ws.ticket[1] != 0;
  const float nan = __int_as_float(0x7fffffff);
  float* st = o.stats + (size_t)row * 4;
  T* y = out + (size_t)row * out_ld;
  RowStats r;
  r.m = lost ? nan : st[0], r.s = lost ? nan : st[1], r.s1 = lost ? nan : st[2];
  r.bad = !(r.m == r.m), r.empty = r.m == -INFINITY;
  const double log_s = log_sum(r);
  const RowGrad rg = row_grad(coef.x, coef.y, coef.z != 0.0f, r, c);
  if (lost) {
    for (int j = threadIdx.x; j < V; j += kRowThreads) y[j] = from_f32<T>(nan);
  } else if (id >= 0 && !rg.zero) {
    const float add = loss ? fmul(-coef.x, share) : -coef.x;
    y[id] = from_f32<T>(fadd(grad1<ENTROPY>(z, rg, one), add));
  }
  if (threadIdx.x == 0) {
    st[3] = (float)log_s;
    if (lost) st[0] = st[1] = st[2] = nan;
    if (r.bad && o.flags) atomicOr(o.flags, (uint32_t)(lost ? DET_SCORE_TIMEOUT : DET_SCORE_NONFINITE));
    if ((loss ? e.bad : t >= V) && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_BAD_TOKEN);
    if (!loss) write_scores(o, row, V, r, log_s, t, z);
  }
  if (loss) {
    const float v = list_loss(e, logq, z, r, log_s, temp, list);
    if (threadIdx.x == 0) loss[row] = lost ? nan : v;
  }
}

// Rows of few segments, few enough that an SM has them all at once: scores
// without a top list, or scores and gradient, in one kernel with a block per row
// and a warp per segment.  All of a row is read before any of its gradient is
// written.  Bound by latency: one load, the sums, the list's sums and a 64-bit
// logarithm follow one another.  What it saves are launches, of two or three.
// bf16, us per call, in a stream and in a graph, against the kernels above:
//                                   148 x 2,000          148 x 32,000
//   scores                      13.7 -> 11.1, 5.0 -> 3.6   13.6 -> 11.2, 6.4 -> 5.1
//   distillation loss           12.6 -> 10.2, 5.3 -> 6.3   13.3 -> 11.4, 7.0 -> 7.6
//   scores and gradient         15.9 -> 11.5, 8.6 -> 5.6   15.7 -> 11.4, 13.6 -> 7.2
//   entropy's gradient too      15.8 -> 11.6, 11.0 -> 7.0  18.8 -> 11.7, 17.6 -> 8.8
//   distillation and gradient   15.2 -> 10.9, 10.3 -> 8.3  15.5 -> 11.0, 14.5 -> 10.0
// With more rows than that it loses: 592 x 32,000 31.5 -> 38.2 for the last,
// 17.0 -> 18.6 for the first.  With a top list the block's warps are too few for
// the list: 9 -> 11 us for 1 x 2,000, 9 -> 16 for 1 x 32,000.
enum { kScores, kGrad, kGradEntropy };
constexpr int kSmallSegs = kListWarps;
template <typename T, int MODE>
__global__ void __launch_bounds__(32 * kSmallSegs)
    small_rows_kernel(Logits L, const void* tokens, int id_bytes, Teacher te, float temp, GradIn in, float* loss,
                      ScoreOut o, T* out, unsigned long long out_ld, float one) {
  using G = Seg<T>;
  constexpr bool ENTROPY = MODE == kGradEntropy;
  __shared__ ListShared list;
  __shared__ float4 seg[kSmallSegs];
  const int row = blockIdx.x, V = L.vocab, g = threadIdx.x >> 5, l = threadIdx.x & 31;
  const int nseg = (V + kSeg - 1) / kSeg;
  const float c = fdiv(kLog2e, temp), nan = __int_as_float(0x7fffffff);
  const uint32_t table = kExpTable[l];
  pdl_enter();
  const T* x = static_cast<const T*>(L.x) + (size_t)(L.rows ? L.rows[row] : row) * L.ld;
  const int mis = misaligned(x);
  uint4 raw[G::NV];
  float v[MODE == kGrad ? kPerLane : 1], m_seg = -INFINITY;
  if (g < nseg) {
#pragma unroll
    for (int i = 0; i < G::NV; i++) raw[i] = row_vec<T, false>(x, g * kSeg + (32 * i + l) * G::VEC, V, mis);
    Range<T> range;
#pragma unroll
    for (int i = 0; i < G::NV; i++) range.take(raw[i]);
    m_seg = redux_max(range.high());
    const float s =
        segment_sums<T, MODE == kGrad>(raw, V - g * kSeg, m_seg, redux_min(range.low()), c, table, one, v);
    const float w = __shfl_sync(kFull, s, 16);
    if (l == 0) seg[g] = make_float4(m_seg, s, w, 0.0f);
  }
  // the row's own tokens, and the gradient's coefficients (as in StepWork)
  ListEntry e;
  double logq = 0.0;
  long long t = -1;
  int id = -1;
  float z = 0.0f, share = 0.0f, a_g = 0.0f, a_h = 0.0f;
  bool zero = false;
  if (te.k) {
    e = teacher_entry(te, row, V, c, table, one, list);
    if (e.id >= 0) z = to_f32(x[e.id]);
    logq = list_logq(e, temp);
    if constexpr (MODE != kScores) {
      ListEntry f = e;
      share = list_share(f, te.k, list);
      id = f.id;
      a_g = e.bad ? nan : fdiv(in.g[row], temp);
      zero = !e.some && !e.bad;
    }
  } else {
    if (tokens) t = load_id(tokens, id_bytes, row);
    if (t >= 0 && t < V) z = to_f32(x[t]);
    if constexpr (MODE != kScores) {
      if (threadIdx.x == 0 && t >= 0 && t < V) id = (int)t;
      a_g = -(!in.g || t < 0 ? 0.0f : t >= V ? nan : in.g[row]);
      a_h = in.gh ? in.gh[row] : 0.0f;
    }
  }
  __syncthreads();  // the sums are there, and the row is read
  const RowStats r = finish_row(join_segments<true>(
      [&](int i) {
        const float4 f = seg[i];
        return Sums{f.x, f.y, f.z};
      },
      nseg, c, table, one));
  if constexpr (MODE != kScores) {
    const RowGrad rg = row_grad(a_g, a_h, zero, r, c);
    T* y = out + (size_t)row * out_ld;
    if (g < nseg) grad_segment<T, ENTROPY>(raw, v, m_seg, r.m, rg, c, table, one, y, g, V);
    __syncthreads();  // behind the rest of the row's gradient:
    if (id >= 0 && !rg.zero)
      y[id] = from_f32<T>(fadd(grad1<ENTROPY>(z, rg, one), te.k ? fmul(-a_g, share) : -a_g));
  }
  const double log_s = threadIdx.x < max(1, te.k) ? log_sum(r) : 0.0;
  if (threadIdx.x == 0) {
    if (o.stats) write_stats(o.stats, row, r, log_s);
    if (r.bad && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_NONFINITE);
    if ((te.k ? e.bad : t >= V) && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_BAD_TOKEN);
    if (!te.k) write_scores(o, row, V, r, log_s, t, z);
  }
  if (te.k) {
    const float sum = list_loss(e, logq, z, r, log_s, temp, list);
    if (threadIdx.x == 0) loss[row] = sum;
  }
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

// Blocks of a kernel that the current device holds at once (cached: the answer
// depends on the kernel and the launch alone).
cudaError_t resident_blocks(const void* kern, int threads, size_t smem, int* out) {
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  static Known<std::tuple<const void*, int, int, size_t>, int> known;
  return known.get({kern, dev, threads, smem}, out, [&](int* n) {
    int per = 0, sms = 0;
    cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, threads, smem);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) cudaGetLastError();
    *n = per * sms;
    return e == cudaSuccess && *n <= 0 ? cudaErrorInvalidConfiguration : e;
  });
}

// How a kernel with a warp per segment takes rows of nseg segments: clusters of
// c blocks of `warps` warps, `fit` of which the current device holds at once.
// Of 4 to 8 warps per block (as many as segments, if those are fewer; 16 blocks
// per cluster at most) the fewest that hold 93% of the most rows at once: a
// row's segments wait for one another, so an SM is kept busy by blocks of
// several rows.  4,096 rows of 128,256 bf16 logits: 570 us in 31 clusters of 16
// blocks of 4 warps, 609 in 33 of 8 of 8; but of 151,936: 761 us in 26 of 10 of
// 8, 947 in 24 of 15 of 5.  Below 4 warps more of the time goes into the sends:
// 1,024 rows of 65,000 take 126 us in blocks of 2, 85 in blocks of 4.  Cached,
// likewise.
struct ClusterPlan {
  int c = 0, warps = 0, fit = 0;
};
cudaError_t cluster_plan(const void* kern, int nseg, size_t stage, ClusterPlan* out) {
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  if (cudaError_t e = raise_smem_cap(kern, kWarps * stage)) return e;
  static Known<std::tuple<const void*, int, int>, ClusterPlan> known;
  return known.get({kern, dev, nseg}, out, [&](ClusterPlan* best) {
    // clusters above 8 blocks have to be allowed
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) return e;
    ClusterPlan plans[kWarps];
    int n = 0, most = 0;
    for (int w = nseg < 4 ? nseg : 4; w <= kWarps; w++) {
      ClusterPlan p;
      p.c = (nseg + w - 1) / w;
      p.warps = (nseg + p.c - 1) / p.c;
      if (p.c > 16 || p.warps != w) continue;
      if (p.c == 1) {
        if (cudaError_t e = resident_blocks(kern, 32 * w, w * stage, &p.fit)) return e;
      } else {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)p.c);
        cfg.blockDim = dim3((unsigned)(32 * w));
        cfg.dynamicSmemBytes = w * stage;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = p.c;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaError_t e = cudaOccupancyMaxActiveClusters(&p.fit, kern, &cfg)) {
          cudaGetLastError();
          return e;
        }
      }
      plans[n++] = p;
      most = most < p.fit ? p.fit : most;
    }
    for (int i = 0; i < n && best->fit == 0; i++)
      if (100 * plans[i].fit >= 93 * most) *best = plans[i];
    return best->fit > 0 ? cudaSuccess : cudaErrorInvalidConfiguration;
  });
}
// launches `clusters` clusters of c blocks, with programmatic stream
// serialization
template <typename... KArgs, typename... Args>
cudaError_t launch_clusters(cudaStream_t s, void (*kern)(KArgs...), int clusters, int c, int threads, size_t smem,
                            Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * c));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = c;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = c > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
// Whether small_rows_kernel takes the rows: all of them at once, at 16 warps per
// SM.
int small_warps(int nseg) { return nseg < 4 ? 4 : nseg; }  // a thread per list entry
bool small_rows(int n, int vocab) {
  const int nseg = (vocab + kSeg - 1) / kSeg;
  return nseg <= kSmallSegs && n <= device_sms() * (16 / small_warps(nseg));
}
int forward_launches(int n, int vocab, int top) { return !top && small_rows(n, vocab) ? 1 : 2; }
template <typename T, int MODE>
cudaError_t small_as(cudaStream_t s, const Logits& L, const void* tokens, int id_bytes, const Teacher& te, float temp,
                     const GradIn& in, float* loss, const ScoreOut& o, void* out, unsigned long long out_ld) {
  const int warps = small_warps((L.vocab + kSeg - 1) / kSeg);
  return launch_k(Launch{s, nullptr, nullptr, true}, small_rows_kernel<T, MODE>, dim3(L.n), dim3(32 * warps), 0, L,
                  tokens, id_bytes, te, temp, in, loss, o, static_cast<T*>(out), out_ld, 1.0f);
}
// what a forward call keeps between its two kernels
size_t workspace_bytes(int dtype, int n, int vocab, int top) {
  const size_t nseg = (vocab + kSeg - 1) / kSeg, vec = dtype == DET_DTYPE_F32 ? 4 : 8;
  const size_t groups = !top ? 0 : nseg * kSeg / (vec << group_lanes_log2(vocab, top, (int)vec));
  return align256(n * nseg * sizeof(float4)) + align256(n * groups * sizeof(float));
}
template <typename T, bool TOP>
cudaError_t forward_as(cudaStream_t s, const Logits& L, const void* tokens, int id_bytes, const Teacher& te,
                       float temp, void* workspace, float* loss, const ScoreOut& o) {
  if (!TOP && small_rows(L.n, L.vocab))
    return small_as<T, kScores>(s, L, o.logprob ? tokens : nullptr, id_bytes, te, temp, GradIn{}, loss, o, nullptr, 0);
  const int lg = TOP ? group_lanes_log2(L.vocab, o.top, Seg<T>::VEC) : -1;
  const auto segments = lg < 0    ? segments_kernel<T, -1>
                        : lg == 0 ? segments_kernel<T, 0>
                        : lg == 3 ? segments_kernel<T, 3>
                                  : segments_kernel<T, 5>;
  constexpr int kSegWarps = kSegThreads / 32;
  const size_t smem = kSegWarps * kStageBytes<T>;
  if (cudaError_t e = raise_smem_cap((const void*)segments, smem)) return e;
  const long long nseg = (L.vocab + kSeg - 1) / kSeg, blocks = (L.n * nseg + kSegWarps - 1) / kSegWarps;
  int fit = 0;
  if (cudaError_t e = resident_blocks((const void*)segments, kSegThreads, smem, &fit)) return e;
  Workspace ws;
  ws.seg = static_cast<float4*>(workspace);
  ws.gmax = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + align256(L.n * nseg * sizeof(float4)));
  const Launch launch{s, nullptr, nullptr, true};
  if (cudaError_t e = launch_k(launch, segments, dim3((unsigned)(blocks < fit ? blocks : fit)), dim3(kSegThreads), smem,
                               L, temp, ws, 1.0f))
    return e;
  return launch_k(launch, rows_kernel<T, TOP>, dim3(L.n), dim3(kRowThreads), 0, L, tokens, id_bytes,
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
  // Runs per warp, up to 8: the waves of blocks, times a block's runs and what
  // it costs beside them (half a run's time; a list takes about two)
  const int step = kThreads * kGradUnroll;
  int per = step, fit = 0;
  if (cudaError_t e = resident_blocks((const void*)grad_kernel<T, ENTROPY>, kThreads, 0, &fit)) return e;
  float least = 0.0f;
  for (int runs = 1; runs <= 8; runs++) {
    const long long all = (long long)L.n * ((nvec + runs * step - 1) / (runs * step));
    const float cost = (float)((all + fit - 1) / fit) * (runs + (te.k ? 2.0f : 0.5f));
    if (runs == 1 || cost < least) least = cost, per = runs * step;
  }
  // and less than a run of each warp where SMs would be without a block
  while (per > kGradRun && (long long)L.n * ((nvec + per - 1) / per) < device_sms()) per /= 2;
  const int blocks = (nvec + per - 1) / per;
  const Launch launch{s, nullptr, nullptr, true};
  for (int r = 0; r < L.n; r += 65535) {
    if (cudaError_t e = launch_k(launch, grad_kernel<T, ENTROPY>, dim3(blocks, L.n - r < 65535 ? L.n - r : 65535),
                                 dim3(kThreads), 0, L, r, per, tokens, id_bytes, te, temp, in, static_cast<T*>(out),
                                 out_ld, 1.0f))
      return e;
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

size_t step_workspace_bytes(size_t n, int k) {
  return align256(n * sizeof(float4)) + align256(n * k * sizeof(float)) + align256(2 * sizeof(uint32_t));
}
// the three kernels; `most`: clusters at most
template <typename T, bool ENTROPY, bool SELFTEST = false>
cudaError_t clusters_as(cudaStream_t s, const Logits& L, const void* tokens, int id_bytes, const Teacher& te,
                        float temp, const GradIn& in, void* workspace, float* loss, const ScoreOut& o, void* out,
                        unsigned long long out_ld, int most) {
  const size_t n = L.n, k = te.k ? te.k : 1;
  uint8_t* at = static_cast<uint8_t*>(workspace);
  auto take = [&](size_t bytes) {
    uint8_t* p = at;
    at += align256(bytes);
    return p;
  };
  StepWork ws;
  ws.coef = reinterpret_cast<float4*>(take(n * sizeof(float4)));
  ws.z = reinterpret_cast<float*>(take(n * k * sizeof(float)));
  ws.ticket = reinterpret_cast<uint32_t*>(take(2 * sizeof(uint32_t)));
  const auto kern = step_kernel<T, ENTROPY, SELFTEST>;
  ClusterPlan plan;
  if (cudaError_t e = cluster_plan((const void*)kern, (L.vocab + kSeg - 1) / kSeg, kStageBytes<T>, &plan)) return e;
  const int fit = plan.fit < most ? plan.fit : most, clusters = L.n < fit ? L.n : fit;
  const Launch launch{s, nullptr, nullptr, true};
  if (cudaError_t e = launch_k(launch, step_gather_kernel<T>, dim3((L.n + kWarps - 1) / kWarps), dim3(kThreads), 0, L,
                               tokens, id_bytes, te, temp, in, ws, 2 * clusters))
    return e;
  T* y = static_cast<T*>(out);
  if (cudaError_t e = launch_clusters(s, kern, clusters, plan.c, 32 * plan.warps, plan.warps * kStageBytes<T>, L, temp,
                                      ws, o.stats, y, out_ld, 1.0f))
    return e;
  return launch_k(launch, step_rows_kernel<T, ENTROPY>, dim3(L.n), dim3(kRowThreads), 0, L, tokens, id_bytes, te, temp,
                  in, ws, loss, o, y, out_ld, 1.0f);
}
template <typename T, bool ENTROPY>
cudaError_t step_as(cudaStream_t s, const Logits& L, const void* tokens, int id_bytes, const Teacher& te, float temp,
                    const GradIn& in, void* workspace, float* loss, const ScoreOut& o, void* out,
                    unsigned long long out_ld) {
  if (small_rows(L.n, L.vocab))
    return small_as<T, ENTROPY ? kGradEntropy : kGrad>(s, L, tokens, id_bytes, te, temp, in, loss, o, out, out_ld);
  return clusters_as<T, ENTROPY>(s, L, tokens, id_bytes, te, temp, in, workspace, loss, o, out, out_ld, L.n);
}
cudaError_t launch_step(cudaStream_t s, int dtype, const Logits& L, const void* tokens, int id_bytes,
                        const Teacher& te, float temp, const GradIn& in, void* workspace, float* loss,
                        const ScoreOut& o, void* out, unsigned long long out_ld) {
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return in.gh ? step_as<T, true>(s, L, tokens, id_bytes, te, temp, in, workspace, loss, o, out, out_ld)
                 : step_as<T, false>(s, L, tokens, id_bytes, te, temp, in, workspace, loss, o, out, out_ld);
  });
}

// ---- argument checks ----------------------------------------------------------------
constexpr uint64_t kMaxLd = 1ull << 36;  // with DET_SCORE_MAX_ROWS rows of 4 bytes: below 2^64

size_t dtype_size(int dtype) { return dtype == DET_DTYPE_F32 ? 4 : 2; }

det_status check_logits(const void* logits, int dtype, uint32_t n, uint32_t vocab, uint64_t ld) {
  if (!logits || dtype < DET_DTYPE_F32 || dtype > DET_DTYPE_BF16) return DET_ERR_INVALID_ARGUMENT;
  if (vocab == 0) return DET_ERR_CDF_EMPTY;
  if (vocab > kMaxVocab) return DET_ERR_CDF_TOO_MANY_SYMBOLS;
  if (n > DET_SCORE_MAX_ROWS || ld > kMaxLd) return DET_ERR_INVALID_ARGUMENT;
  if ((uintptr_t)logits % dtype_size(dtype)) return DET_ERR_INVALID_ARGUMENT;
  return DET_OK;
}
// the gradient goes over the logits exactly, or nowhere near them: equal
// strides side by side, or ranges that do not meet
det_status check_grad(const void* logits, int dtype, uint32_t n, uint32_t vocab, uint64_t ld, const void* grad,
                      uint64_t grad_ld) {
  if (!grad || (n > 1 && grad_ld < vocab) || grad_ld > kMaxLd) return DET_ERR_INVALID_ARGUMENT;
  const size_t sz = dtype_size(dtype);
  if ((uintptr_t)grad % sz) return DET_ERR_INVALID_ARGUMENT;
  const uintptr_t a = (uintptr_t)logits, b = (uintptr_t)grad;
  if (a == b) return n == 1 || ld == grad_ld ? DET_OK : DET_ERR_INVALID_ARGUMENT;
  const size_t an = ((size_t)(n - 1) * ld + vocab) * sz, bn = ((size_t)(n - 1) * grad_ld + vocab) * sz;
  if (b > a ? b - a >= an : a - b >= bn) return DET_OK;
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
  if (k == 0 || k > DET_MAX_TOP || (n > 1 && ld < k) || ld > kMaxLd) return DET_ERR_INVALID_ARGUMENT;
  if (!(temperature >= DET_MIN_TEMPERATURE && temperature <= DET_MAX_TEMPERATURE)) return DET_ERR_INVALID_ARGUMENT;
  return DET_OK;
}
det_status check_workspace(const void* workspace, size_t size, size_t need) {
  return workspace && (uintptr_t)workspace % 16 == 0 && size >= need ? DET_OK : DET_ERR_INVALID_ARGUMENT;
}
det_status check_device() {
  static std::atomic<bool> seen{false};
  if (seen.load(std::memory_order_relaxed)) return DET_OK;
  int cnt = 0;
  if (cudaGetDeviceCount(&cnt) != cudaSuccess || cnt == 0) return DET_ERR_NO_DEVICE;
  seen.store(true, std::memory_order_relaxed);
  return DET_OK;
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
  if (L.launches) *L.launches += forward_launches(n, V, top);
  return launch_forward(L.stream, DET_DTYPE_F32, x, tokens, 4, kNoTeacher, 1.0f, workspace, nullptr, o);
}
cudaError_t launch_distill_loss(const Launch& L, const float* logits, int V, const uint32_t* rows, int n,
                                const int32_t* ids, const float* teacher, int k, float temperature, float* loss,
                                void* workspace) {
  const Logits x{logits, rows, (unsigned long long)V, n, V};
  const Teacher te{ids, teacher, (unsigned long long)k, 4, DET_DTYPE_F32, k};
  const ScoreOut o{nullptr, nullptr, nullptr, nullptr, nullptr, 0, L.err};
  if (L.launches) *L.launches += forward_launches(n, V, 0);
  return launch_forward(L.stream, DET_DTYPE_F32, x, nullptr, 4, te, temperature, workspace, loss, o);
}

size_t scores_workspace_bytes(int n, int V, int top) { return workspace_bytes(DET_DTYPE_F32, n, V, top); }

// One run of the step on zero logits in rows of `vocab`, with a list of k ids or
// (k = 0) with tokens, in two clusters that take several rows each; everything
// it writes to is 0 before.  *all, *none: are all of its results NaN, none of
// them; *flags: what it set.
template <bool SELFTEST>
cudaError_t step_selftest_run(int vocab, int k, bool* all, bool* none, uint32_t* flags) {
  using T = __nv_bfloat16;
  constexpr int n = 12, kIds = 2;
  // logits | gradient | ids | f32: ones (the gradients of the results) | teacher | results, stats | flags | workspace
  const size_t row_bytes = align256((size_t)n * vocab * sizeof(T)), small = 4096;
  const size_t bytes = 2 * row_bytes + 5 * small + step_workspace_bytes(n, kIds);
  uint8_t* mem = nullptr;
  if (cudaError_t e = cudaMalloc(&mem, bytes)) return e;
  T* grad = reinterpret_cast<T*>(mem + row_bytes);
  int32_t* ids = reinterpret_cast<int32_t*>(mem + 2 * row_bytes);
  float* ones = reinterpret_cast<float*>(mem + 2 * row_bytes + small);
  float* u = reinterpret_cast<float*>(mem + 2 * row_bytes + 2 * small);
  float* res = reinterpret_cast<float*>(mem + 2 * row_bytes + 3 * small);  // logprob or loss, entropy, stats
  uint32_t* flag = reinterpret_cast<uint32_t*>(mem + 2 * row_bytes + 4 * small);
  const Logits L{mem, nullptr, (unsigned long long)vocab, n, vocab};
  const Teacher te{ids, u, kIds, 4, DET_DTYPE_F32, k};
  const ScoreOut o{k ? nullptr : res, k ? nullptr : res + n, res + 2 * n, nullptr, nullptr, 0, flag};
  float one[n], host[6 * n];
  for (float& v : one) v = 1.0f;
  cudaError_t e = cudaMemset(mem, 0, bytes);
  if (e == cudaSuccess) e = cudaMemcpy(ones, one, sizeof(one), cudaMemcpyHostToDevice);
  if (e == cudaSuccess)
    e = clusters_as<T, false, SELFTEST>(nullptr, L, ids, 4, k ? te : kNoTeacher, 1.0f, GradIn{nullptr, ones, nullptr},
                                        mem + 2 * row_bytes + 5 * small, k ? res : nullptr, o, grad, vocab, 2);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpy(flags, flag, 4, cudaMemcpyDeviceToHost);
  if (e == cudaSuccess) e = cudaMemcpy(host, res, sizeof(host), cudaMemcpyDeviceToHost);
  *all = *none = true;
  auto look = [&](bool is_nan) {
    *all &= is_nan;
    *none &= !is_nan;
  };
  for (int i = 0; i < 6 * n; i++)
    if (!k || i < n || i >= 2 * n) look(host[i] != host[i]);
  for (size_t at = 0; at < (size_t)n * vocab && e == cudaSuccess;) {
    uint16_t part[2048];
    const size_t m = (size_t)n * vocab - at < 2048 ? (size_t)n * vocab - at : 2048;
    e = cudaMemcpy(part, grad + at, 2 * m, cudaMemcpyDeviceToHost);
    for (size_t i = 0; i < m; i++) look((part[i] & 0x7fff) > 0x7f80);
    at += m;
  }
  cudaFree(mem);
  return e;
}

static_assert(DET_SCORE_NONFINITE == (int)ERRF_CDF_NONFINITE && DET_SCORE_BAD_TOKEN == (int)ERRF_SYMBOL,
              "the flags are the session's error bits");
}  // namespace det

using namespace det;

extern "C" {

det_status det_step_timeout_selftest(int device) {
  int cnt = 0;
  if (cudaGetDeviceCount(&cnt) != cudaSuccess || cnt == 0) return DET_ERR_NO_DEVICE;
  if (device < 0 || device >= cnt) return DET_ERR_INVALID_ARGUMENT;
  if (cudaSetDevice(device) != cudaSuccess) return DET_ERR_CUDA;
  bool reported = true;
  for (int vocab : {5000, 40000})  // a block per row, and a cluster
    for (int k : {0, 2}) {
      bool all, none;
      uint32_t flags = 0;
      if (step_selftest_run<true>(vocab, k, &all, &none, &flags) != cudaSuccess) return DET_ERR_CUDA;
      reported &= flags == DET_SCORE_TIMEOUT && all;
      if (step_selftest_run<false>(vocab, k, &all, &none, &flags) != cudaSuccess || flags || !none) return DET_ERR_CUDA;
    }
  return reported ? DET_ERR_TIMEOUT : DET_OK;
}

size_t det_scores_workspace(int dtype, uint32_t n, uint32_t vocab, uint32_t top) {
  if (dtype < DET_DTYPE_F32 || dtype > DET_DTYPE_BF16 || vocab > kMaxVocab || n > DET_SCORE_MAX_ROWS) return 0;
  return workspace_bytes(dtype, (int)n, (int)vocab, (int)top);
}

size_t det_step_workspace(uint32_t n, uint32_t vocab, uint32_t k) {
  if (n > DET_SCORE_MAX_ROWS || vocab > kMaxVocab || k > DET_MAX_TOP) return 0;
  return step_workspace_bytes(n, k ? (int)k : 1);
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
  if (det_status st = check_workspace(workspace, workspace_size, workspace_bytes(dtype, (int)n, (int)vocab, (int)top))) return st;
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
                                        void* grad, uint64_t grad_ld, uint32_t* flags, void* workspace,
                                        size_t workspace_size, void* stream) {
  if (n == 0) return DET_OK;
  if (det_status st = check_logits(logits, dtype, n, vocab, ld)) return st;
  if (det_status st = check_grad(logits, dtype, n, vocab, ld, grad, grad_ld)) return st;
  if (!stats || (!grad_logprob && !grad_entropy)) return DET_ERR_INVALID_ARGUMENT;
  if (logprob || grad_logprob)
    if (det_status st = check_ids(tokens, token_bytes)) return st;
  if (det_status st = check_workspace(workspace, workspace_size, step_workspace_bytes(n, 1))) return st;
  if (det_status st = check_device()) return st;
  const Logits L{logits, nullptr, ld, (int)n, (int)vocab};
  const ScoreOut o{logprob, entropy, stats, nullptr, nullptr, 0, flags};
  return launched(launch_step(static_cast<cudaStream_t>(stream), dtype, L, logprob || grad_logprob ? tokens : nullptr,
                              token_bytes, kNoTeacher, 1.0f, GradIn{nullptr, grad_logprob, grad_entropy}, workspace,
                              nullptr, o, grad, grad_ld));
}

det_status det_distill_loss_device(const void* logits, int dtype, uint32_t n, uint32_t vocab, uint64_t ld,
                                   const void* ids, int id_bytes, const void* teacher, int teacher_dtype, uint32_t k,
                                   uint64_t list_ld, float temperature, float* loss, float* stats, uint32_t* flags,
                                   void* workspace, size_t workspace_size, void* stream) {
  if (n == 0) return DET_OK;
  if (det_status st = check_logits(logits, dtype, n, vocab, ld)) return st;
  if (det_status st = check_list(ids, id_bytes, teacher, teacher_dtype, k, n, list_ld, temperature)) return st;
  if (!loss) return DET_ERR_INVALID_ARGUMENT;
  if (det_status st = check_workspace(workspace, workspace_size, workspace_bytes(dtype, (int)n, (int)vocab, 0))) return st;
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
                                   float* stats, void* grad, uint64_t grad_ld, uint32_t* flags, void* workspace,
                                   size_t workspace_size, void* stream) {
  if (n == 0) return DET_OK;
  if (det_status st = check_logits(logits, dtype, n, vocab, ld)) return st;
  if (det_status st = check_grad(logits, dtype, n, vocab, ld, grad, grad_ld)) return st;
  if (det_status st = check_list(ids, id_bytes, teacher, teacher_dtype, k, n, list_ld, temperature)) return st;
  if (!loss || !stats || !grad_loss) return DET_ERR_INVALID_ARGUMENT;
  if (det_status st = check_workspace(workspace, workspace_size, step_workspace_bytes(n, (int)k))) return st;
  if (det_status st = check_device()) return st;
  const Logits L{logits, nullptr, ld, (int)n, (int)vocab};
  const Teacher te{ids, teacher, list_ld, id_bytes, teacher_dtype, (int)k};
  const ScoreOut o{nullptr, nullptr, stats, nullptr, nullptr, 0, flags};
  return launched(launch_step(static_cast<cudaStream_t>(stream), dtype, L, nullptr, 4, te, temperature,
                              GradIn{nullptr, grad_loss, nullptr}, workspace, loss, o, grad, grad_ld));
}

}  // extern "C"
