// AdamW over a list of separate tensors in as few launches as their pointers need, states in 32 or in 8 bits
// (the update rule of noise_adamw_step, train/main.py:13-14, without a flat parameter buffer):
//   g' = s g,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// with one device-side step count t per tensor, so a captured launch replays correctly.
//
// Bound: HBM, 28 bytes per fp32 value with 32-bit states, 16 with 8-bit ones.  Pointers and sizes travel as kernel arguments
// (nothing is uploaded, nothing outlives the call); a workgroup takes 1024 values of one tensor (4096, four vectors per
// thread, reached 4.9 instead of 5.2 TB/s at 150 M values: many short workgroups keep the accesses in flight close together).
//
// 8-bit states: m and r = sqrt(v) as e4m3 values with one fp32 scale = max|.| / 448 per 256 consecutive values of a tensor,
// i.e. one wave's four values per lane.  r rather than v: its range within a block (2^18 : 1) is then v's 2^36 : 1.  A
// positive r never becomes zero (it would leave m / eps).  The new moments are formed and rounded in 64 bits, by the rule's own
// operations, each rounded once: m = RN(RN(b1 m) + RN((1 - b1) g)), the root and both divisions to the nearest double.  Sums of
// short numbers land on the border between two codes, or a scale halfway between two floats, by far more often than by chance
// (b1 = 0.9: one scale in 600 of a model's list), and then an ulp of a double decides the code.  A block with a non-finite
// moment gets a NaN scale, which the next step shows in its parameters.
#include "token.h"

namespace {

constexpr int ADAM_MAX = 96;         // tensors per launch: 36 bytes each in the 4 KB of kernel arguments
constexpr int ADAM_UNIT = 1024;      // values per workgroup: one vector per thread, one block of values per wave
constexpr int ADAM_BLOCK = 256;      // values per scale of the 8-bit states
constexpr int ADAM_MASK_WORDS = 64;  // 64-bit words of the active mask per launch of the coefficient kernel

struct AdamList {
  void* p[ADAM_MAX];
  const void* g[ADAM_MAX];
  long off[ADAM_MAX];        // first value of the tensor's states (a multiple of ADAM_BLOCK)
  int end_unit[ADAM_MAX];    // workgroups of tensors 0..i
  int numel_lo[ADAM_MAX];    // values in the tensor's last workgroup
  int count;
};
struct AdamIndex {
  int idx[ADAM_MAX];
};
struct AdamCoef {
  float beta1, beta2, omb1, omb2, eps, decay, grad_scale;
  double dbeta1, dbeta2, domb1, domb2;
};
struct AdamMask {
  unsigned long long w[ADAM_MASK_WORDS];
};

// step[i] += 1 and [lr / (1 - b1^t) | sqrt(1 - b2^t)] of every active tensor.
__global__ __launch_bounds__(256) void adam_coef_kernel(long long* __restrict__ step, float2* __restrict__ coef, int first,
                                                        int n, AdamMask mask, double lr, double b1, double b2) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n || !((mask.w[i >> 6] >> (i & 63)) & 1)) return;
  const long long t = step[first + i] + 1;
  step[first + i] = t;
  coef[first + i] = make_float2((float)(lr / (1.0 - pow(b1, (double)t))), (float)sqrt(1.0 - pow(b2, (double)t)));
}

// Which tensor a workgroup works on: binary search over the running counts (uniform, scalar loads).
__device__ __forceinline__ int adam_find(const AdamList& l, int unit) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (unit < l.end_unit[mid]) hi = mid; else lo = mid + 1;
  }
  return lo;
}

// Four values of a tensor, elementwise where the address does not allow a vector access or the tensor ends inside
// (FULL: neither can be).
template <bool FULL, typename T>
__device__ __forceinline__ void load4(const T* base, int i, int n, bool vec, float (&out)[4]) {
  if (FULL || (vec && i + 4 <= n)) {
    load_vec<T, 4>(base + i, out);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = i + j < n ? (float)base[i + j] : 0.f;
  }
}
template <bool FULL, typename T>
__device__ __forceinline__ void store4(T* base, int i, int n, bool vec, const float (&in)[4]) {
  if (FULL || (vec && i + 4 <= n)) {
    store_vec<T, 4>(base + i, in);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) base[i + j] = (T)in[j];
  }
}

// p, g and the states of one workgroup's values
template <typename P, typename G>
struct AdamUnit {
  P* p;
  const G* g;
  size_t state;      // first value in the state buffers
  float2 coef;
  int n;             // values, ADAM_UNIT except in a tensor's last workgroup
  bool vec;
};
template <typename P, typename G>
__device__ __forceinline__ AdamUnit<P, G> adam_unit(const AdamList& l, const AdamIndex& ix, const float2* coef) {
  const int unit = blockIdx.x, t = adam_find(l, unit);
  const int local = unit - (t ? l.end_unit[t - 1] : 0);
  const size_t at = (size_t)local * ADAM_UNIT;
  AdamUnit<P, G> u;
  u.p = (P*)l.p[t] + at;
  u.g = (const G*)l.g[t] + at;
  u.state = (size_t)l.off[t] + at;
  u.coef = coef[ix.idx[t]];
  u.n = unit == l.end_unit[t] - 1 ? l.numel_lo[t] : ADAM_UNIT;
  u.vec = ((uintptr_t)u.p % (4 * sizeof(P))) == 0 && ((uintptr_t)u.g % (4 * sizeof(G))) == 0;
  return u;
}

template <bool FULL, typename P, typename G>
__device__ __forceinline__ void adam32_unit(const AdamUnit<P, G>& t, float* m, float* v, const AdamCoef& c) {
  const int n = t.n, whole = (n + 3) & ~3;   // the states are padded to blocks of 256: a vector never leaves them
  const int i = threadIdx.x * 4;
  if (!FULL && i >= n) return;
  float pv[4], gv[4], mv[4], vv[4];
  load4<FULL>(t.p, i, n, t.vec, pv);
  load4<FULL>(t.g, i, n, t.vec, gv);
  load4<FULL>(m, i, whole, true, mv);
  load4<FULL>(v, i, whole, true, vv);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float gi = gv[j] * c.grad_scale;
    mv[j] = mv[j] * c.beta1 + c.omb1 * gi;
    vv[j] = vv[j] * c.beta2 + c.omb2 * (gi * gi);
    const float denom = sqrtf(vv[j]) / t.coef.y + c.eps;
    pv[j] = pv[j] * c.decay - t.coef.x * (mv[j] / denom);
  }
  store4<FULL>(t.p, i, n, t.vec, pv);
  store4<FULL>(m, i, whole, true, mv);
  store4<FULL>(v, i, whole, true, vv);
}

template <typename P, typename G>
__global__ __launch_bounds__(256) void adam32_kernel(AdamList l, AdamIndex ix, const float2* __restrict__ coef,
                                                     float* __restrict__ ms, float* __restrict__ vs, AdamCoef c) {
  const AdamUnit<P, G> t = adam_unit<P, G>(l, ix, coef);
  if (t.vec && t.n == ADAM_UNIT) adam32_unit<true>(t, ms + t.state, vs + t.state, c);
  else adam32_unit<false>(t, ms + t.state, vs + t.state, c);
}

// Largest of a 32-bit value over the wave, in a scalar register: four steps as DPP operands, then one value per 16 lanes.
__device__ __forceinline__ unsigned wave_max_u32(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));
  v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));
  const unsigned a = __builtin_amdgcn_readlane((int)v, 0), b = __builtin_amdgcn_readlane((int)v, 16);
  const unsigned c = __builtin_amdgcn_readlane((int)v, 32), d = __builtin_amdgcn_readlane((int)v, 48);
  return max(max(a, b), max(c, d));
}

// Largest magnitude of the wave's values, four per lane, found on the bits of the doubles (their order is the integers', and a NaN or
// infinity is above all others): the high words first, then, where several lanes share the highest, the low words.
__device__ __forceinline__ double block_top(const double (&x)[4]) {
  const double t = __builtin_fmax(__builtin_fmax(fabs(x[0]), fabs(x[1])), __builtin_fmax(fabs(x[2]), fabs(x[3])));
  const double sum = (x[0] + x[1]) + (x[2] + x[3]);            // a NaN is lost in the maximum, not here
  const unsigned hi = sum != sum ? 0x7ff80000u : (unsigned)(__double_as_longlong(t) >> 32), lo = (unsigned)__double_as_longlong(t);
  const unsigned th = wave_max_u32(hi);
  const unsigned long long who = __ballot(hi == th);
  unsigned tl;
  if ((who & (who - 1)) == 0) tl = (unsigned)__builtin_amdgcn_readlane((int)lo, __builtin_ctzll(who));
  else tl = wave_max_u32(hi == th ? lo : 0u);
  return __longlong_as_double((long long)((unsigned long long)th << 32 | tl));
}

// a / b to the nearest double, with 1 / b to its last bits: the product's remainder is exact and corrects it.
__device__ __forceinline__ double divide64(double a, double b, double inv) {
  const double q = a * inv;
  return __builtin_fma(__builtin_fma(-q, b, a), inv, q);
}

// sqrt of a value >= 0 in 64 bits to about 46: the hardware's reciprocal root (2^-23) and one step of Newton's method; EXACT: another
// one, which leaves little but its own rounding.
template <bool EXACT>
__device__ __forceinline__ double root64(double v) {
  const double y = __builtin_amdgcn_rsq(v + 1e-300), h = 0.5 * y;      // 1e-300: zero gives zero
  double s = v * y;
  s = __builtin_fma(h, __builtin_fma(-s, s, v), s);
  return EXACT ? __builtin_fma(h, __builtin_fma(-s, s, v), s) : s;
}

// Four values of a 256-value block as e4m3 codes under the scale max / 448 (`top`: that maximum), rounded as x / scale would be.
// What is rounded to 8 bits is a float of x / scale that is cut off, with its lowest bit set where something was lost, so that
// the second rounding sees which side of a border the value lies on.  All borders have few bits: the 29 that the cut takes are
// zero there.  The product x * (1 / scale) decides wherever it is further from that than it can be wrong (NEAR units of a
// double's last place); where one of a lane's four is nearer, exact(j) and its true quotient do.
template <bool POSITIVE, unsigned NEAR, typename Exact>
__device__ __forceinline__ unsigned quantise4(const double (&x)[4], double top, float& scale, Exact exact) {
  scale = (float)divide64(top, 448.0, 1.0 / 448.0);
  // 1 / scale to the last bits of a double: a float's reciprocal and two steps of Newton's method; a block whose scale is below
  // the normal floats is divided by it
  const double d = (double)scale;
  double inv = (double)__builtin_amdgcn_rcpf(scale);
  inv = __builtin_fma(__builtin_fma(-d, inv, 1.0), inv, inv);
  inv = __builtin_fma(__builtin_fma(-d, inv, 1.0), inv, inv);
  if (!(scale > 1e-36f && scale < 1e36f)) inv = scale > 0.f ? 1.0 / d : 0.0;
  unsigned long long b[4];
  unsigned away = 0xffffffffu;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    b[j] = (unsigned long long)__double_as_longlong(x[j] * inv);
    away = min(away, ((unsigned)b[j] + NEAR) & 0x1fffffffu);
    b[j] = (b[j] & 0xffffffffe0000000ull) | 0x20000000ull;
  }
  if (away <= 2 * NEAR) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const unsigned long long t = (unsigned long long)__double_as_longlong(divide64(exact(j), d, inv));
      b[j] = (t & 0xffffffffe0000000ull) | ((t & 0x1fffffffull) ? 0x20000000ull : 0ull);
    }
  }
  float q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) q[j] = __builtin_amdgcn_fmed3f((float)__longlong_as_double((long long)b[j]), POSITIVE && x[j] > 0.0 ? 0x1p-9f : -448.f, 448.f);
  int code = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  code = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], code, true);
  if (!(top < INFINITY)) scale = __int_as_float(0x7fc00000);
  return (unsigned)code;
}

// a / b: the hardware's reciprocal and one correction (within one unit of the last place); the division itself where b or its
// reciprocal is near the ends of the range.
__device__ __forceinline__ float quotient(float a, float b) {
  const float y = __builtin_amdgcn_rcpf(b), q = a * y;
  float r = __builtin_fmaf(__builtin_fmaf(-q, b, a), y, q);
  if (!(b > 1e-30f && b < 1e30f)) r = a / b;
  return r;
}

template <bool FULL, typename P, typename G>
__device__ __forceinline__ void adam8_unit(const AdamUnit<P, G>& t, unsigned* ms, float* mscale, unsigned* rs, float* rscale,
                                           const AdamCoef& c) {
  const int n = t.n, i = threadIdx.x * 4, b = i & ~(ADAM_BLOCK - 1);   // the wave's block of values
  if (!FULL && b >= n) return;
  const float inv_root = 1.f / t.coef.y;
  float pv[4], gv[4], cm[4], cr[4];
  const size_t q = (t.state + i) / 4, sc = (t.state + b) / ADAM_BLOCK;
  load4<FULL>(t.p, i, n, t.vec, pv);
  load4<FULL>(t.g, i, n, t.vec, gv);
  const unsigned mc = ms[q], rc = rs[q];
  const double sm = (double)mscale[sc], sr = (double)rscale[sc];
  {
    const auto m0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc, false), m1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc, true);
    const auto r0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)rc, false), r1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)rc, true);
    cm[0] = m0[0], cm[1] = m0[1], cm[2] = m1[0], cm[3] = m1[1];
    cr[0] = r0[0], cr[1] = r0[1], cr[2] = r1[0], cr[3] = r1[1];
  }
  const double fr = c.dbeta2 * (sr * sr);
  double m[4], v[4], r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double gi = (double)(gv[j] * c.grad_scale);
    m[j] = c.dbeta1 * ((double)cm[j] * sm) + c.domb1 * gi;    // the old m is exact: a code has 4 bits, a scale 24
    v[j] = __builtin_fma((double)(cr[j] * cr[j]), fr, c.domb2 * (gi * gi));   // a few units of the last place; a code's square has 8 bits
    r[j] = root64<false>(v[j]);
    const float denom = (float)r[j] * inv_root + c.eps;
    pv[j] = pv[j] * c.decay - t.coef.x * quotient((float)m[j], denom);
  }
  store4<FULL>(t.p, i, n, t.vec, pv);
  float nm, nr;
  ms[q] = quantise4<false, 4>(m, block_top(m), nm, [&](int j) { return m[j]; });
  // r is off by 2^-46 of itself: 2^6 units of its last place
  rs[q] = quantise4<true, 512>(r, root64<true>(block_top(v)), nr, [&](int j) {
    const double gi = (double)(gv[j] * c.grad_scale), ro = (double)cr[j] * sr;
    return root64<true>(c.dbeta2 * (ro * ro) + c.domb2 * (gi * gi));
  });
  if ((threadIdx.x & 63) == 0) {
    mscale[sc] = nm;
    rscale[sc] = nr;
  }
}

template <typename P, typename G>
__global__ __launch_bounds__(256) void adam8_kernel(AdamList l, AdamIndex ix, const float2* __restrict__ coef,
                                                    unsigned* __restrict__ ms, float* __restrict__ mscale,
                                                    unsigned* __restrict__ rs, float* __restrict__ rscale, AdamCoef c) {
  const AdamUnit<P, G> t = adam_unit<P, G>(l, ix, coef);
  if (t.vec && t.n == ADAM_UNIT) adam8_unit<true>(t, ms, mscale, rs, rscale, c);
  else adam8_unit<false>(t, ms, mscale, rs, rscale, c);
}

template <typename P, typename G>
void adam_launch(int grid, const AdamList& l, const AdamIndex& ix, const float2* coef, void* m, float* msc, void* v, float* vsc,
                 const AdamCoef& c, bool small, hipStream_t st) {
  if (small)
    hipLaunchKernelGGL((adam8_kernel<P, G>), dim3(grid), dim3(256), 0, st, l, ix, coef, (unsigned*)m, msc, (unsigned*)v, vsc, c);
  else
    hipLaunchKernelGGL((adam32_kernel<P, G>), dim3(grid), dim3(256), 0, st, l, ix, coef, (float*)m, (float*)v, c);
}

}  // namespace

// Counts the steps of the tensors whose bit is set in `active` (host array of (n + 63) / 64 words) and leaves their
// coefficients for noise_adamw_multi.
NOISE_EXPORT int noise_adamw_multi_begin(long long* step, float* coef, const unsigned long long* active, int n, double lr,
                                         double beta1, double beta2, void* stream) {
  NOISE_REQUIRE(step && coef && active && n > 0, "noise_adamw_multi_begin: bad argument");
  const int per = ADAM_MASK_WORDS * 64;
  for (int first = 0; first < n; first += per) {
    const int m = n - first < per ? n - first : per;
    AdamMask mask;
    for (int i = 0; i < ADAM_MASK_WORDS; ++i) mask.w[i] = i < (m + 63) / 64 ? active[first / 64 + i] : 0;
    hipLaunchKernelGGL(adam_coef_kernel, dim3(noise_cdiv(m, 256)), dim3(256), 0, (hipStream_t)stream, step, (float2*)coef, first, m,
                       mask, lr, beta1, beta2);
    NOISE_CHECK_LAUNCH("noise_adamw_multi_begin");
  }
  return 0;
}

// One update of `count` tensors of one parameter type and one gradient type.  p, g, numel, off and index are host arrays:
// tensor i has numel[i] values at p[i] / g[i], its states start at value off[i], its coefficients are number index[i].
NOISE_EXPORT int noise_adamw_multi(const unsigned long long* p, const unsigned long long* g, const long* numel, const long* off,
                                   const int* index, int count, int pdtype, int gdtype, int bits, const float* coef, void* m,
                                   float* mscale, void* v, float* vscale, double lr, double beta1, double beta2, double eps,
                                   double weight_decay, double grad_scale, void* stream) {
  NOISE_REQUIRE(p && g && numel && off && index && coef && m && v && count > 0, "noise_adamw_multi: bad argument");
  NOISE_REQUIRE(bits == 32 || (bits == 8 && mscale && vscale), "noise_adamw_multi: states have 32 bits, or 8 with scales");
  NOISE_REQUIRE(pdtype >= NOISE_F32 && pdtype <= NOISE_F16 && (gdtype == pdtype || (pdtype == NOISE_F32 && gdtype >= NOISE_F32 && gdtype <= NOISE_F16)),
                "noise_adamw_multi: gradients have the parameters' type, or any for fp32 parameters");
  for (int i = 0; i < count; ++i)
    NOISE_REQUIRE(numel[i] >= 0 && (numel[i] == 0 || (p[i] && g[i])) && off[i] >= 0 && off[i] % ADAM_BLOCK == 0,
                  "noise_adamw_multi: tensor %d: null pointer or bad size", i);
  AdamCoef c;
  c.beta1 = (float)beta1, c.beta2 = (float)beta2, c.omb1 = (float)(1.0 - beta1), c.omb2 = (float)(1.0 - beta2);
  c.eps = (float)eps, c.decay = (float)(1.0 - lr * weight_decay), c.grad_scale = (float)grad_scale;
  c.dbeta1 = beta1, c.dbeta2 = beta2, c.domb1 = 1.0 - beta1, c.domb2 = 1.0 - beta2;
  const bool small = bits == 8;
  for (int i = 0; i < count;) {
    AdamList l;
    AdamIndex ix;
    long units = 0;
    l.count = 0;
    for (; i < count && l.count < ADAM_MAX; ++i) {
      if (numel[i] == 0) continue;
      const long u = (numel[i] + ADAM_UNIT - 1) / ADAM_UNIT;
      // a grid holds at most 2^32 threads
      if (units + u > (1L << 23)) {
        NOISE_REQUIRE(l.count > 0, "noise_adamw_multi: a tensor of %ld values is too large", numel[i]);
        break;
      }
      units += u;
      const int k = l.count++;
      l.p[k] = (void*)p[i];
      l.g[k] = (const void*)g[i];
      l.off[k] = off[i];
      l.end_unit[k] = (int)units;
      l.numel_lo[k] = (int)(numel[i] - (u - 1) * ADAM_UNIT);
      ix.idx[k] = index[i];
    }
    if (l.count == 0) break;
    const float2* cf = (const float2*)coef;
    hipStream_t st = (hipStream_t)stream;
    const int key = pdtype * 3 + gdtype;
#define GO(P, G) adam_launch<P, G>((int)units, l, ix, cf, m, mscale, v, vscale, c, small, st)
    if (key == 0) GO(float, float);
    else if (key == 1) GO(float, bf16_t);
    else if (key == 2) GO(float, f16_t);
    else if (key == 4) GO(bf16_t, bf16_t);
    else GO(f16_t, f16_t);
#undef GO
    NOISE_CHECK_LAUNCH("noise_adamw_multi");
  }
  return 0;
}
