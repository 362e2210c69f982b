// AdamW over a list of separate tensors in as few launches as their pointers need, states in 32 or in 8 bits
// (the update rule of noise_adamw_step, train/main.py:13-14, without a flat parameter buffer):
//   g' = s g,  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2,
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// with one device-side step count t per tensor, so a captured launch replays correctly.
//
// Bound: HBM, 28 bytes per fp32 value with 32-bit states, 16 with 8-bit ones.  Pointers and sizes travel as kernel arguments
// (nothing is uploaded, nothing outlives the call); a workgroup takes 4096 values of one tensor, all of a thread's loads
// requested before the first use.
//
// 8-bit states: m and r = sqrt(v) as e4m3 values with one fp32 scale = max|.| / 448 per 256 consecutive values of a tensor,
// i.e. one wave's four values per lane.  r rather than v: its range within a block (2^18 : 1) is then v's 2^36 : 1.  A
// positive r never becomes zero (it would leave m / eps).  The new moments are formed and rounded in 64 bits: 8-bit values
// then depend on the inputs alone and not on the order of fp32 operations next to a rounding border.  A block with a
// non-finite moment gets a NaN scale, which the next step shows in its parameters.
#include "token.h"

namespace {

constexpr int ADAM_MAX = 96;         // tensors per launch: 36 bytes each in the 4 KB of kernel arguments
constexpr int ADAM_UNIT = 4096;      // values per workgroup
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

// p, g and the states of one workgroup's 4096 values
template <typename P, typename G>
struct AdamUnit {
  P* p;
  const G* g;
  size_t state;      // first value in the state buffers
  float2 coef;
  int n;             // values, 4096 except in a tensor's last workgroup
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
  float pv[4][4], gv[4][4], mv[4][4], vv[4][4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int i = (u * 256 + threadIdx.x) * 4;
    load4<FULL>(t.p, i, n, t.vec, pv[u]);
    load4<FULL>(t.g, i, n, t.vec, gv[u]);
    load4<FULL>(m, i, whole, true, mv[u]);
    load4<FULL>(v, i, whole, true, vv[u]);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int i = (u * 256 + threadIdx.x) * 4;
    if (!FULL && i >= n) break;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float gi = gv[u][j] * c.grad_scale;
      const float mi = mv[u][j] * c.beta1 + c.omb1 * gi;
      const float vi = vv[u][j] * c.beta2 + c.omb2 * (gi * gi);
      const float denom = sqrtf(vi) / t.coef.y + c.eps;
      pv[u][j] = pv[u][j] * c.decay - t.coef.x * (mi / denom);
      mv[u][j] = mi;
      vv[u][j] = vi;
    }
    store4<FULL>(t.p, i, n, t.vec, pv[u]);
    store4<FULL>(m, i, whole, true, mv[u]);
    store4<FULL>(v, i, whole, true, vv[u]);
  }
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

// A double as the float that rounds to the same 8-bit value: cut off, with the lowest bit set where something was lost, so
// that the second rounding sees which side of a border the value lies on.
__device__ __forceinline__ float to_odd(double x) {
  const unsigned long long b = __double_as_longlong(x);
  unsigned lo = (unsigned)b;
  lo = (lo & 0xe0000000u) | ((lo & 0x1fffffffu) ? 0x20000000u : 0u);
  return (float)__longlong_as_double((long long)((b & 0xffffffff00000000ull) | lo));
}

// Four values of a 256-value block as e4m3 codes under the scale max / 448; the whole wave takes part.  The largest magnitude
// is found on the bits of the doubles (their order is the integers', and a NaN or infinity is above all others): the high
// words first, then the low words of those that share the highest.
template <bool POSITIVE>
__device__ __forceinline__ unsigned quantise4(const double (&x)[4], float& scale) {
  unsigned hi[4], lo[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned long long b = __double_as_longlong(x[j]);
    hi[j] = (unsigned)(b >> 32) & 0x7fffffffu;
    lo[j] = (unsigned)b;
  }
  const unsigned th = wave_max_u32(max(max(hi[0], hi[1]), max(hi[2], hi[3])));
  unsigned l = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) l = max(l, hi[j] == th ? lo[j] : 0u);
  const double top = __longlong_as_double((long long)((unsigned long long)th << 32 | wave_max_u32(l)));
  scale = (float)(top * (1.0 / 448.0));
  const double inv = scale > 0.f ? 1.0 / (double)scale : 0.0;
  float q[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) q[j] = __builtin_amdgcn_fmed3f(to_odd(x[j] * inv), -448.f, 448.f);
  int code = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  code = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], code, true);
  if (POSITIVE) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if ((hi[j] | lo[j]) != 0 && (code & (0xff << (8 * j))) == 0) code |= 1 << (8 * j);
  }
  if (th >= 0x7ff00000u) scale = __int_as_float(0x7fc00000);
  return (unsigned)code;
}

// sqrt in 64 bits to about 46: the hardware's reciprocal root and one step of Newton's method.
__device__ __forceinline__ double root64(double v) {
  const double y = __builtin_amdgcn_rsq(v), s = v * y;
  const double r = s + 0.5 * y * __builtin_fma(-s, s, v);
  return v > 0.0 && v < 1e300 ? r : v;        // zero, and what is not finite, as they are
}

// a / b: the hardware's reciprocal and one correction (within one unit of the last place); the division itself where an
// intermediate value could leave the range.
__device__ __forceinline__ float quotient(float a, float b) {
  const float y = __builtin_amdgcn_rcpf(b), q = a * y;
  float r = __builtin_fmaf(__builtin_fmaf(-q, b, a), y, q);
  if (!(b > 1e-30f && b < 1e30f && fabsf(q) < 1e30f)) r = a / b;
  return r;
}

template <bool FULL, typename P, typename G>
__device__ __forceinline__ void adam8_unit(const AdamUnit<P, G>& t, unsigned* ms, float* mscale, unsigned* rs, float* rscale,
                                           const AdamCoef& c) {
  const int n = t.n, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const float inv_root = 1.f / t.coef.y;
  float pv[4][4], gv[4][4], msc[4], rsc[4];
  unsigned mc[4], rc[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int b = (u * 4 + wave) * ADAM_BLOCK, i = b + lane * 4;   // uniform per wave: one block of values
    mc[u] = rc[u] = 0;
    msc[u] = rsc[u] = 0.f;
    if (FULL || b < n) {
      const size_t q = (t.state + i) / 4, sc = (t.state + b) / ADAM_BLOCK;
      load4<FULL>(t.p, i, n, t.vec, pv[u]);
      load4<FULL>(t.g, i, n, t.vec, gv[u]);
      mc[u] = ms[q];
      rc[u] = rs[q];
      msc[u] = mscale[sc];
      rsc[u] = rscale[sc];
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int b = (u * 4 + wave) * ADAM_BLOCK, i = b + lane * 4;
    if (!FULL && b >= n) break;
    float cm[4], cr[4];
    {
      const auto m0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc[u], false), m1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc[u], true);
      const auto r0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)rc[u], false), r1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)rc[u], true);
      cm[0] = m0[0], cm[1] = m0[1], cm[2] = m1[0], cm[3] = m1[1];
      cr[0] = r0[0], cr[1] = r0[1], cr[2] = r1[0], cr[3] = r1[1];
    }
    const double sm = (double)msc[u], sr = (double)rsc[u];
    const double fm = c.dbeta1 * sm, fr = c.dbeta2 * (sr * sr);
    double m[4], r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double gi = (double)(gv[u][j] * c.grad_scale);
      m[j] = __builtin_fma((double)cm[j], fm, c.domb1 * gi);
      r[j] = root64(__builtin_fma((double)(cr[j] * cr[j]), fr, c.domb2 * (gi * gi)));   // a code's square has 8 bits
      const float denom = (float)r[j] * inv_root + c.eps;
      pv[u][j] = pv[u][j] * c.decay - t.coef.x * quotient((float)m[j], denom);
    }
    store4<FULL>(t.p, i, n, t.vec, pv[u]);
    float nm, nr;
    const unsigned am = quantise4<false>(m, nm), ar = quantise4<true>(r, nr);
    const size_t q = (t.state + i) / 4, sc = (t.state + b) / ADAM_BLOCK;
    ms[q] = am;
    rs[q] = ar;
    if (lane == 0) {
      mscale[sc] = nm;
      rscale[sc] = nr;
    }
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
