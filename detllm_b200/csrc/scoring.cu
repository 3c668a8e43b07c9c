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
constexpr int kThreads = 256;
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

// exp(d) for d <= 0, two at a time: d = k ln 2 + r with |r| <= ln 2 / 2 (a
// two-part ln 2 whose parts times k are exact), exp(r) by a degree-5 minimax
// polynomial 1 + r + r^2 q(r) (relative error 1.06e-7), 2^k added to the
// exponent field.  Below kExpLow the result is +0 (the exponent field goes
// negative there and the integer maximum clears it); it is within 3.1 * 2^-24
// of exp(d) for d >= -87.  NaN gives an unspecified number: callers keep d,
// which stays NaN, beside it.
constexpr float kExpLow = -88.13f;  // k = -127, r = -0.10
struct Exp2 {
  f2 e, d;  // exp, and the argument as clamped
};
DI Exp2 exp2_lanes(f2 d, f2 one) {
  float2 c = un(d);
  c.x = max_nan(c.x, kExpLow);
  c.y = max_nan(c.y, kExpLow);
  d = pk(c.x, c.y);
  const f2 magic = pk(12582912.0f, 12582912.0f), nmagic = pk(-12582912.0f, -12582912.0f);
  const f2 z = addp(mul2(d, pk(1.44269504f, 1.44269504f)), one, magic);
  const f2 k = add2(z, nmagic);
  const f2 nhi = pk(-0.693145751953125f, -0.693145751953125f);
  const f2 nlo = pk(-1.4286197256296873e-06f, -1.4286197256296873e-06f);
  // k has 7 bits and the parts of ln 2 have 15: exact products
  const f2 r = fma2(k, nlo, fma2(k, nhi, d));
  f2 q = addp(mul2(pk(0.008312501f, 0.008312501f), r), one, pk(0.04189033f, 0.04189033f));
  q = addp(mul2(q, r), one, pk(0.16667116f, 0.16667116f));
  q = addp(mul2(q, r), one, pk(0.4999923f, 0.4999923f));
  const f2 p = add2(addp(mul2(q, mul2(r, r)), one, r), pk(1.0f, 1.0f));
  const float2 pf = un(p), zf = un(z);
  const int ex = max(__float_as_int(pf.x) + (__float_as_int(zf.x) << 23), 0);
  const int ey = max(__float_as_int(pf.y) + (__float_as_int(zf.y) << 23), 0);
  return {pk(__int_as_float(ex), __int_as_float(ey)), d};
}
DI float exp1(float d, float one) { return un(exp2_lanes(pk(d, d), pk(one, one)).e).x; }

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
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
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
template <typename T>
DI void load_segment(const T* __restrict__ row, int g, int V, int mis, float (&v)[kPerLane]) {
  using G = Seg<T>;
  const int base = g * kSeg + (threadIdx.x & 31) * G::VEC;
  if (mis == 0 && (g + 1) * kSeg <= V) {
    const uint4* p = reinterpret_cast<const uint4*>(row + base);
    uint4 w[G::NV];
#pragma unroll
    for (int i = 0; i < G::NV; i++) w[i] = __ldg(p + 32 * i);
#pragma unroll
    for (int i = 0; i < G::NV; i++) unpack_vec<T>(w[i], v + i * G::VEC);
  } else {
#pragma unroll
    for (int i = 0; i < G::NV; i++) load_vec<T>(row, base + i * G::GROUP, V, mis, v + i * G::VEC);
  }
}

struct Sums {
  float m, s, s1;
};

DI float warp_max(float v) {
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
DI float warp_sum(float v) {
  for (int o = 16; o > 0; o >>= 1) v = fadd(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
DI double warp_sum_d(double v) {
  for (int o = 16; o > 0; o >>= 1) v = dadd(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

// maximum, sum of exp((x - m) / T) and the same weighted by (x - m) / T over
// one segment's 64 entries per lane; a NaN or +inf anywhere leaves s1 NaN.
// `m`: the segment's maximum.
template <bool SCALED>
DI Sums segment_sums(const float (&x)[kPerLane], float m, float inv_t, float one_) {
  const float base = m == -INFINITY ? 0.0f : -m;
  const f2 nm = pk(base, base), one = pk(one_, one_), it = pk(inv_t, inv_t);
  f2 s[2] = {0, 0}, w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < kPerLane / 2; i++) {
    f2 d = add2(pk(x[2 * i], x[2 * i + 1]), nm);
    if constexpr (SCALED) d = mul2(d, it);
    const Exp2 e = exp2_lanes(d, one);
    s[i & 1] = add2(s[i & 1], e.e);
    w[i & 1] = addp(mul2(e.e, e.d), one, w[i & 1]);
  }
  const float2 sp = un(add2(s[0], s[1])), wp = un(add2(w[0], w[1]));
  return {m, warp_sum(fadd(sp.x, sp.y)), warp_sum(fadd(wp.x, wp.y))};
}
DI float redux_max(float v) {  // of the warp; a NaN loses against a number
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "r"(kFull));
  return r;
}

// joins a row's segments (one warp; the result in every lane)
DI Sums join_segments(const float* sm, const float* ss, const float* sw, int nseg, float inv_t, float one) {
  const int l = threadIdx.x & 31;
  float m = -INFINITY;
  for (int i = l; i < nseg; i += 32) m = fmaxf(m, sm[i]);
  m = warp_max(m);
  float s = 0.0f, w = 0.0f;
  for (int i = l; i < nseg; i += 32) {
    const bool empty = sm[i] == -INFINITY;
    const float d = empty ? kExpLow : fmaxf(fmul(fsub(sm[i], m), inv_t), kExpLow);
    const float f = exp1(d, one);
    s = fadd(s, fmul(f, ss[i]));
    // sum of exp(d_j + d) (d_j + d) = f (S1 + d S); NaN stays NaN
    w = fadd(w, fmul(f, fadd(sw[i], fmul(d, ss[i]))));
  }
  return {m, warp_sum(s), warp_sum(w)};
}

struct RowStats {
  float m, s, s1;
  double log_s;
  bool empty, bad;
};
DI RowStats finish_row(const Sums& r) {
  RowStats t;
  t.bad = !(r.s1 == r.s1) || r.m == INFINITY;
  t.empty = !t.bad && r.m == -INFINITY;
  const float nan = __int_as_float(0x7fffffff);
  t.m = t.bad ? nan : r.m;
  t.s = t.bad ? nan : t.empty ? 0.0f : r.s;
  t.s1 = t.bad ? nan : t.empty ? 0.0f : r.s1;
  t.log_s = t.bad ? (double)nan : t.empty ? (double)-INFINITY : log_det((double)r.s);
  return t;
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
  float red[2][kThreads / 32];
  int bad[kThreads / 32], some[kThreads / 32];
};
struct ListEntry {
  int id;       // -1: not a valid entry
  float q;      // its share of the teacher's distribution
  double logq;
};
// thread i < k of the block gets entry i (kThreads >= DET_MAX_TOP); *some: the
// list has a valid entry; *bad: an id or value that is not allowed
DI ListEntry teacher_entry(const Teacher& te, int row, int vocab, float temp, float one, ListShared& sh, bool* some,
                           bool* bad) {
  const int t = threadIdx.x, w = t >> 5, l = t & 31;
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
  if (l == 0) {
    sh.red[0][w] = m;
    sh.bad[w] = anyw;
    sh.some[w] = anyv;
  }
  __syncthreads();
  m = -INFINITY;
  int b = 0, so = 0;
  for (int i = 0; i < kThreads / 32; i++) {
    m = fmaxf(m, sh.red[0][i]);
    b |= sh.bad[i];
    so |= sh.some[i];
  }
  const double du = valid ? ddiv(dsub((double)u, (double)m), (double)temp) : 0.0;
  const float e = valid ? exp1(fmaxf((float)du, kExpLow), one) : 0.0f;
  const float ws = warp_sum(e);
  if (l == 0) sh.red[1][w] = ws;
  __syncthreads();
  float s = 0.0f;
  for (int i = 0; i < kThreads / 32; i++) s = fadd(s, sh.red[1][i]);
  *some = so != 0;
  *bad = b != 0;
  ListEntry r;
  r.id = valid ? (int)id : -1;
  r.q = valid ? fdiv(e, s) : 0.0f;
  r.logq = valid ? dsub(du, log_det((double)s)) : 0.0;
  return r;
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
};
template <typename T>
DI int group_size(int V) {
  return V <= kSmallVocab ? Seg<T>::VEC : Seg<T>::GROUP;
}
template <typename T>
size_t groups_of(int V) {
  const int g = V <= kSmallVocab ? Seg<T>::VEC : Seg<T>::GROUP, nseg = (V + kSeg - 1) / kSeg;
  return (size_t)nseg * (kSeg / g);
}

// the largest t such that at least k of the block's values are >= t (0 where
// there are fewer than k): bit by bit, done early once exactly k are
template <typename K, int PER>
DI K kth_largest(const K (&v)[PER], int k, TopShared& sh) {
  K t = 0;
  for (int bit = (int)sizeof(K) * 8 - 1, turn = 0; bit >= 0; bit--, turn ^= 1) {
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
    if (all == k) break;
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
  const unsigned long long t = kth_largest<unsigned long long, PER>(v, k, sh);
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
// the row's k largest keys, in order, to sh.key[0 .. k)
template <typename T>
DI void top_list(const T* __restrict__ x, int V, int mis, const float* gmax, int k, TopShared& sh) {
  const int ng = (V + group_size<T>(V) - 1) / group_size<T>(V);
  if (threadIdx.x == 0) sh.count = sh.bits[0] = sh.bits[1] = 0;
  __syncthreads();
  // a value that at least k entries reach: the k-th largest maximum
  unsigned long long floor = 0;
  if (ng > k) {
    constexpr int PER = kSmallVocab / Seg<T>::VEC / kThreads;  // as many groups as there can be, or more
    static_assert(PER * kThreads >= (int)kMaxVocab / Seg<T>::GROUP, "every group has a place");
    uint32_t v[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
      const int g = i * kThreads + threadIdx.x;
      v[i] = g < ng ? (uint32_t)(top_key(gmax[g], 0) >> 32) : 0u;
    }
    const uint32_t t = kth_largest<uint32_t, PER>(v, k, sh);
    floor = t ? ((unsigned long long)t << 32) - 1 : 0;
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

// ---- forward ---------------------------------------------------------------------------
// One cluster per row (of one block where there are rows enough): its warps
// take segments in turn, their sums and group maxima go to block 0, which
// joins them and writes the row's results.
struct ForwardShared {
  float m[kMaxSegs], s[kMaxSegs], w[kMaxSegs];
  RowStats row;
  ListShared list;
  double dred[kThreads / 32];
};
template <typename T, bool TOP, bool SCALED>
__global__ void __launch_bounds__(kThreads, 2)
    forward_kernel(Logits L, const void* tokens, int id_bytes, Teacher te, float temp, float* loss, ScoreOut o,
                   float one) {
  using G = Seg<T>;
  __shared__ ForwardShared sh;
  extern __shared__ float dyn[];  // TOP: group maxima, then a TopShared
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int row = blockIdx.x / size, V = L.vocab, w = threadIdx.x >> 5, l = threadIdx.x & 31;
  const T* x = static_cast<const T*>(L.x) + (size_t)(L.rows ? L.rows[row] : row) * L.ld;
  const int nseg = (V + kSeg - 1) / kSeg, mis = misaligned(x);
  const float inv_t = SCALED ? fdiv(1.0f, temp) : 1.0f;
  if (size > 1) cluster_arrive();  // block 0 runs before anyone writes to it
  bool first = size > 1;
  for (int g = rank * (kThreads / 32) + w; g < nseg; g += size * (kThreads / 32)) {
    float v[kPerLane];
    load_segment<T>(x, g, V, mis, v);
    float m = -INFINITY, gm = -INFINITY;
    float lm[G::NV];
#pragma unroll
    for (int i = 0; i < G::NV; i++) {
      lm[i] = v[i * G::VEC];
#pragma unroll
      for (int j = 1; j < G::VEC; j++) lm[i] = fmaxf(lm[i], v[i * G::VEC + j]);
      m = fmaxf(m, lm[i]);
      if constexpr (TOP) {
        const float r = redux_max(lm[i]);
        if (l == i) gm = r;
      }
    }
    m = redux_max(m);
    const Sums r = segment_sums<SCALED>(v, m, inv_t, one);
    if (first) cluster_wait();
    first = false;
    if (l == 0) {
      store_remote(remote(&sh.m[g], 0), r.m);
      store_remote(remote(&sh.s[g], 0), r.s);
      store_remote(remote(&sh.w[g], 0), r.s1);
    }
    if constexpr (TOP) {
      if (V <= kSmallVocab) {
#pragma unroll
        for (int i = 0; i < G::NV; i++) store_remote(remote(&dyn[g * (kSeg / G::VEC) + i * 32 + l], 0), lm[i]);
      } else if (l < G::NV) {
        store_remote(remote(&dyn[g * G::NV + l], 0), gm);
      }
    }
  }
  if (size > 1) {
    if (first) cluster_wait();
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }
  if (w == 0) {
    const RowStats r = finish_row(join_segments(sh.m, sh.s, sh.w, nseg, inv_t, one));
    if (l == 0) {
      sh.row = r;
      if (o.stats) {
        float* st = o.stats + (size_t)row * 4;
        st[0] = r.m, st[1] = r.s, st[2] = r.s1, st[3] = (float)r.log_s;
      }
      if (r.bad && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_NONFINITE);
    }
  }
  __syncthreads();
  const RowStats r = sh.row;
  const float nan = __int_as_float(0x7fffffff);
  if (loss) {
    bool some, bad;
    const ListEntry e = teacher_entry(te, row, V, temp, one, sh.list, &some, &bad);
    double term = 0.0;
    if (e.id >= 0 && e.q > 0.0f) {
      const double z = (double)to_f32(x[e.id]);
      const double logp = r.empty ? (double)-INFINITY : dsub(ddiv(dsub(z, (double)r.m), (double)temp), r.log_s);
      term = dmul((double)e.q, dsub(e.logq, logp));
    }
    term = warp_sum_d(term);
    if (l == 0) sh.dred[w] = term;
    __syncthreads();
    if (threadIdx.x == 0) {
      double s = 0.0;
      for (int i = 0; i < kThreads / 32; i++) s = dadd(s, sh.dred[i]);
      loss[row] = bad ? nan : !some ? 0.0f : r.bad ? nan : (float)s;
      if (bad && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_BAD_TOKEN);
    }
    return;
  }
  if (threadIdx.x == 0) {
    if (o.entropy) {
      o.entropy[row] = r.bad     ? nan
                       : r.empty ? 0.0f
                                 : (float)dsub(r.log_s, ddiv((double)r.s1, (double)r.s));
    }
    if (o.logprob) {
      const long long t = load_id(tokens, id_bytes, row);
      float v;
      if (r.bad || t >= V) v = nan;
      else if (t < 0) v = 0.0f;
      else if (r.empty) v = -INFINITY;
      else v = (float)dsub(dsub((double)to_f32(x[t]), (double)r.m), r.log_s);
      o.logprob[row] = v;
      if (t >= V && o.flags) atomicOr(o.flags, (uint32_t)DET_SCORE_BAD_TOKEN);
    }
  }
  if constexpr (TOP) {
    TopShared& top = *reinterpret_cast<TopShared*>(dyn + (size_t)nseg * (kSeg / group_size<T>(V)));
    if (!r.bad) top_list<T>(x, V, mis, dyn, o.top, top);
    if ((int)threadIdx.x < o.top) {
      const size_t at = (size_t)row * o.top + threadIdx.x;
      const unsigned long long key = r.bad ? 0 : top.key[threadIdx.x];
      if (o.top_ids) o.top_ids[at] = r.bad ? -1 : (int32_t)(0xffffffffu - (uint32_t)key);
      if (o.top_logprobs) {
        o.top_logprobs[at] = r.bad     ? nan
                             : r.empty ? -INFINITY
                                       : (float)dsub(dsub((double)key_value(key), (double)r.m), r.log_s);
      }
    }
  }
}

// ---- gradient --------------------------------------------------------------------------
// dx_j = exp(d_j) (a + b d_j) + (what the row's own tokens add).  `as`, `bs`
// are a and b over S.
struct GradIn {
  const float *stats, *g, *gh;  // g: of logprob or of the loss; gh: of the entropy, or null
};
struct RowGrad {
  float base, inv_t, as, bs;  // base: -m
  bool zero;                  // nothing but zeros
};
struct GradShared {
  ListShared list;
  int id[DET_MAX_TOP];
  float add[DET_MAX_TOP];
};
// gradients of a pair of entries
template <bool ENTROPY, bool SCALED>
DI f2 grad2(f2 x, const RowGrad& r, f2 one) {
  f2 d = add2(x, pk(r.base, r.base));
  if constexpr (SCALED) d = mul2(d, pk(r.inv_t, r.inv_t));
  const Exp2 e = exp2_lanes(d, one);
  if constexpr (ENTROPY) return mul2(e.e, addp(mul2(e.d, pk(r.bs, r.bs)), one, pk(r.as, r.as)));
  return mul2(e.e, pk(r.as, r.as));
}
// the row's coefficients, and in sh what its tokens add: id[i] (or -1) and
// add[i] for i < the returned count.  Ends with a barrier.
DI int row_grad(int row, int V, const void* tokens, int id_bytes, const Teacher& te, float temp, const GradIn& in,
                float m, float s, float s1, float one, GradShared& sh, RowGrad& r) {
  const float nan = __int_as_float(0x7fffffff);
  const bool empty = m == -INFINITY;
  const float g = in.g ? in.g[row] : 0.0f;
  float a, b = 0.0f;
  bool blank = false;
  int k = 1;
  if (te.k) {
    bool some, bad;
    const ListEntry e = teacher_entry(te, row, V, temp, one, sh.list, &some, &bad);
    blank = !some && !bad;
    a = bad ? nan : fdiv(g, temp);
    k = te.k;
    if ((int)threadIdx.x < k) {
      sh.id[threadIdx.x] = e.id;
      sh.add[threadIdx.x] = e.q;
    }
    __syncthreads();
    // an id that is listed twice: its first entry takes the sum, in order
    float sum = 0.0f;
    bool first = true;
    if ((int)threadIdx.x < k && e.id >= 0)
      for (int i = 0; i < k; i++)
        if (sh.id[i] == e.id) {
          if (i < (int)threadIdx.x) first = false;
          sum = fadd(sum, sh.add[i]);
        }
    __syncthreads();
    if ((int)threadIdx.x < k) {
      if (!first) sh.id[threadIdx.x] = -1;
      sh.add[threadIdx.x] = fmul(-a, sum);
    }
  } else {
    const float gh = in.gh ? in.gh[row] : 0.0f;
    const long long t = in.g ? load_id(tokens, id_bytes, row) : -1;
    const float gl = t < 0 ? 0.0f : t >= V ? nan : g;
    a = fadd(-gl, fmul(gh, fdiv(s1, s)));
    b = -gh;
    if (threadIdx.x == 0) {
      sh.id[0] = t >= 0 && t < V ? (int)t : -1;
      sh.add[0] = gl;
    }
  }
  const float inv_s = fdiv(1.0f, s);
  r.zero = blank || empty;
  r.base = -m;
  r.inv_t = fdiv(1.0f, temp);
  r.as = fmul(a, inv_s);
  r.bs = fmul(b, inv_s);
  __syncthreads();
  return k;
}

// Blocks (blockIdx.x) of a row (blockIdx.y + row0) take `per` of its 16-byte
// vectors each; a vector is one of the gradient's, so that stores are whole
// wherever the row starts.  `out` may be the logits themselves.
constexpr int kGradUnroll = 4;
template <typename T, bool ENTROPY, bool SCALED>
__global__ void __launch_bounds__(kThreads)
    grad_kernel(Logits L, int row0, int per, const void* tokens, int id_bytes, Teacher te, float temp, GradIn in,
                T* out, unsigned long long out_ld, float one_) {
  constexpr int VEC = Seg<T>::VEC;
  __shared__ GradShared sh;
  const int row = row0 + blockIdx.y, V = L.vocab;
  const T* x = static_cast<const T*>(L.x) + (size_t)row * L.ld;
  T* y = out + (size_t)row * out_ld;
  const float* st = in.stats + (size_t)row * 4;
  RowGrad r;
  const int k = row_grad(row, V, tokens, id_bytes, te, temp, in, st[0], st[1], st[2], one_, sh, r);
  const f2 one = pk(one_, one_);
  const int my = misaligned(y), mis = (misaligned(x) - my) & (VEC - 1);
  const int nvec = (V + my + VEC - 1) / VEC;
  const int q0 = blockIdx.x * per, q1 = min(nvec, q0 + per);
  // the values at the row's own tokens, before `out` may overwrite them
  const int id = (int)threadIdx.x < k ? sh.id[threadIdx.x] : -1;
  const bool patch = id >= 0 && id >= q0 * VEC - my && id < q1 * VEC - my && !r.zero;
  float mine = 0.0f;
  if (patch) {
    const float v = to_f32(x[id]);
    mine = fadd(un(grad2<ENTROPY, SCALED>(pk(v, v), r, one)).x, sh.add[threadIdx.x]);
  }
  __syncthreads();
  for (int q = q0 + threadIdx.x; q < q1; q += kThreads * kGradUnroll) {
    float v[kGradUnroll][VEC];
#pragma unroll
    for (int u = 0; u < kGradUnroll; u++) {
      const int at = (q + u * kThreads) * VEC - my;
      if (q + u * kThreads < q1) load_vec<T, false>(x, at, V, mis, v[u]);
    }
#pragma unroll
    for (int u = 0; u < kGradUnroll; u++) {
      const int at = (q + u * kThreads) * VEC - my;
      if (q + u * kThreads >= q1) continue;
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        const float2 gr = un(grad2<ENTROPY, SCALED>(pk(v[u][j], v[u][j + 1]), r, one));
        v[u][j] = r.zero ? 0.0f : gr.x;
        v[u][j + 1] = r.zero ? 0.0f : gr.y;
      }
      if (at >= 0 && at + VEC <= V) {
        *reinterpret_cast<uint4*>(y + at) = pack_vec<T>(v[u]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; j++)
          if (at + j >= 0 && at + j < V) y[at + j] = from_f32<T>(v[u][j]);
      }
    }
  }
  __syncthreads();
  if (patch) y[id] = from_f32<T>(mine);
}

// ---- launches --------------------------------------------------------------------
template <typename F>
cudaError_t by_dtype(int dtype, F f) {
  switch (dtype) {
    case DET_DTYPE_F32: f(float{}); break;
    case DET_DTYPE_F16: f(__half{}); break;
    default: f(__nv_bfloat16{}); break;
  }
  return cudaGetLastError();
}

// Blocks per row: enough for the GPU (two blocks of 8 warps per SM) while
// every warp keeps a segment.
int cluster_for(int n, int vocab) {
  const int nseg = (vocab + kSeg - 1) / kSeg, sms = device_sms();
  int c = 1;
  while (c < 8 && (long long)n * c < 2 * sms && nseg > c * (kThreads / 32)) c *= 2;
  return c;
}
template <typename T, bool TOP, bool SCALED>
cudaError_t forward_as(cudaStream_t s, const Logits& L, const void* tokens, int id_bytes, const Teacher& te,
                       float temp, float* loss, const ScoreOut& o) {
  const size_t smem = TOP ? groups_of<T>(L.vocab) * sizeof(float) + sizeof(TopShared) : 0;
  if (cudaError_t e = raise_smem_cap((const void*)forward_kernel<T, TOP, SCALED>, smem)) return e;
  const int c = cluster_for(L.n, L.vocab);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(L.n * c));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = c > 1;
  return cudaLaunchKernelEx(&cfg, forward_kernel<T, TOP, SCALED>, L, tokens, id_bytes, te, temp, loss, o, 1.0f);
}
cudaError_t launch_forward(cudaStream_t s, int dtype, const Logits& L, const void* tokens, int id_bytes,
                           const Teacher& te, float temp, float* loss, const ScoreOut& o) {
  cudaError_t e = cudaSuccess;
  const cudaError_t last = by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    e = o.top         ? forward_as<T, true, false>(s, L, tokens, id_bytes, te, temp, loss, o)
        : temp == 1.0f ? forward_as<T, false, false>(s, L, tokens, id_bytes, te, temp, loss, o)
                       : forward_as<T, false, true>(s, L, tokens, id_bytes, te, temp, loss, o);
  });
  return e ? e : last;
}
template <typename T, bool ENTROPY, bool SCALED>
cudaError_t grad_as(cudaStream_t s, const Logits& L, const void* tokens, int id_bytes, const Teacher& te, float temp,
                    const GradIn& in, void* out, unsigned long long out_ld) {
  constexpr int VEC = Seg<T>::VEC;
  const int nvec = (L.vocab + VEC - 1) / VEC + 1;  // one more where a row starts inside a vector
  const int step = kThreads * kGradUnroll;
  int per = 4 * step;
  while (per > step && (long long)L.n * ((nvec + per - 1) / per) < 8 * device_sms()) per -= step;
  const int blocks = (nvec + per - 1) / per;
  for (int r = 0; r < L.n; r += 65535) {
    grad_kernel<T, ENTROPY, SCALED><<<dim3(blocks, L.n - r < 65535 ? L.n - r : 65535), kThreads, 0, s>>>(
        L, r, per, tokens, id_bytes, te, temp, in, static_cast<T*>(out), out_ld, 1.0f);
    if (cudaError_t e = cudaGetLastError()) return e;
  }
  return cudaSuccess;
}
cudaError_t launch_grad(cudaStream_t s, int dtype, const Logits& L, const void* tokens, int id_bytes,
                        const Teacher& te, float temp, const GradIn& in, void* out, unsigned long long out_ld) {
  cudaError_t e = cudaSuccess;
  const cudaError_t last = by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    e = in.gh           ? grad_as<T, true, false>(s, L, tokens, id_bytes, te, temp, in, out, out_ld)
        : temp == 1.0f ? grad_as<T, false, false>(s, L, tokens, id_bytes, te, temp, in, out, out_ld)
                       : grad_as<T, false, true>(s, L, tokens, id_bytes, te, temp, in, out, out_ld);
  });
  return e ? e : last;
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
                                int32_t* top_ids, float* top_logprobs) {
  const Logits x{logits, rows, (unsigned long long)V, n, V};
  const ScoreOut o{logprob, entropy, nullptr, top_ids, top_logprobs, top, L.err};
  if (L.launches) ++*L.launches;
  return launch_forward(L.stream, DET_DTYPE_F32, x, tokens, 4, kNoTeacher, 1.0f, nullptr, o);
}
cudaError_t launch_distill_loss(const Launch& L, const float* logits, int V, const uint32_t* rows, int n,
                                const int32_t* ids, const float* teacher, int k, float temperature, float* loss) {
  const Logits x{logits, rows, (unsigned long long)V, n, V};
  const Teacher te{ids, teacher, (unsigned long long)k, 4, DET_DTYPE_F32, k};
  const ScoreOut o{nullptr, nullptr, nullptr, nullptr, nullptr, 0, L.err};
  if (L.launches) ++*L.launches;
  return launch_forward(L.stream, DET_DTYPE_F32, x, nullptr, 4, te, temperature, loss, o);
}

static_assert(DET_SCORE_NONFINITE == (int)ERRF_CDF_NONFINITE && DET_SCORE_BAD_TOKEN == (int)ERRF_SYMBOL,
              "the flags are the session's error bits");
}  // namespace det

using namespace det;

extern "C" {

det_status det_token_scores_device(const void* logits, int dtype, uint32_t n, uint32_t vocab, uint64_t ld,
                                   const void* tokens, int token_bytes, uint32_t top, float* logprob, float* entropy,
                                   float* stats, int32_t* top_ids, float* top_logprobs, uint32_t* flags,
                                   void* stream) {
  if (n == 0) return DET_OK;
  if (det_status st = check_logits(logits, dtype, n, vocab, ld)) return st;
  if (logprob)
    if (det_status st = check_ids(tokens, token_bytes)) return st;
  if (top > DET_MAX_TOP || top > vocab || (top && !top_ids && !top_logprobs)) return DET_ERR_INVALID_ARGUMENT;
  if (det_status st = check_device()) return st;
  const Logits L{logits, nullptr, ld, (int)n, (int)vocab};
  const ScoreOut o{logprob, entropy, stats, top_ids, top_logprobs, (int)top, flags};
  return launched(launch_forward(static_cast<cudaStream_t>(stream), dtype, L, tokens, token_bytes, kNoTeacher, 1.0f,
                                 nullptr, o));
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
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cudaError_t e = launch_forward(s, dtype, L, tokens, token_bytes, kNoTeacher, 1.0f, nullptr, o))
    return launched(e);
  return launched(launch_grad(s, dtype, L, tokens, token_bytes, kNoTeacher, 1.0f,
                              GradIn{stats, grad_logprob, grad_entropy}, grad, grad_ld));
}

det_status det_distill_loss_device(const void* logits, int dtype, uint32_t n, uint32_t vocab, uint64_t ld,
                                   const void* ids, int id_bytes, const void* teacher, int teacher_dtype, uint32_t k,
                                   uint64_t list_ld, float temperature, float* loss, float* stats, uint32_t* flags,
                                   void* stream) {
  if (n == 0) return DET_OK;
  if (det_status st = check_logits(logits, dtype, n, vocab, ld)) return st;
  if (det_status st = check_list(ids, id_bytes, teacher, teacher_dtype, k, n, list_ld, temperature)) return st;
  if (!loss) return DET_ERR_INVALID_ARGUMENT;
  if (det_status st = check_device()) return st;
  const Logits L{logits, nullptr, ld, (int)n, (int)vocab};
  const Teacher te{ids, teacher, list_ld, id_bytes, teacher_dtype, (int)k};
  const ScoreOut o{nullptr, nullptr, stats, nullptr, nullptr, 0, flags};
  return launched(launch_forward(static_cast<cudaStream_t>(stream), dtype, L, nullptr, 4, te, temperature, loss, o));
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
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cudaError_t e = launch_forward(s, dtype, L, nullptr, 4, te, temperature, loss, o)) return launched(e);
  return launched(
      launch_grad(s, dtype, L, nullptr, 4, te, temperature, GradIn{stats, grad_loss, nullptr}, grad, grad_ld));
}

}  // extern "C"
