// Decay attention: causal linear attention with one decay per head and a state a stream can carry,
//   S_t = exp(g) S_{t-1} + k_t (x) v_t,   o_t = scale q_t S_t,
// over clips in chunks, backwards, and for single tokens.
//
// Everything but the single token is ONE operator ("walk") on three token tensors a, k (width dk) and v (width dv),
//   X_p = lam X_{p-1} + s_kv k_p (x) v_p,   o_p = s_o a_p X_p,
// read in either direction of time:
//   forward  o   (a, k, v) = (q, k, v)   first token first, X = S,    s_o = scale
//   backward dq  (a, k, v) = (do, v, k)  first token first, X = S^T,  s_o = scale
//            dv  (a, k, v) = (k, q, do)  last token first,  X = dS,   s_kv = scale
//            dk  (a, k, v) = (v, do, q)  last token first,  X = dS^T, s_kv = scale
// The gradient of the final state meets the last token without a decay (`shift`).
//
// Chunks of C tokens with the state X before them:
//   o_i = s_o [ s_kv sum_{j<=i} lam^{i-j} (a_i . k_j) v_j + lam^{i+1} a_i X ],   X <- lam^C X + s_kv sum_j lam^{C-1-j} k_j (x) v_j
// i.e. four small matrix products per chunk.  A workgroup owns one (clip, head, segment of the token axis) and walks its
// chunks with X in registers.  Where clips and heads alone do not fill the GPU the token axis is cut into segments: one pass
// sums each segment's own contribution to the state, a scan turns them into the state before each segment, and the walk
// starts from those.
#include "token.h"
#include <type_traits>

namespace {

constexpr int DA_C = 32;   // tokens per chunk

struct Strides {
  long b, t, h;   // elements between clips, tokens and heads; the last axis has unit stride
};

struct WalkArgs {
  const void *a, *k, *v;
  void* o;
  Strides sa, sk, sv, so;
  const float* log_decay;   // [H]
  const int* lengths;       // [B] or null: T
  const float* x0;          // state before the first token, [B][H][dk][dv] (x0_tr: [dv][dk]) or null: zero
  float* x_end;             // state behind the last token, [B][H][dk][dv], or null
  float* seg;               // [B][H][nseg][dk][dv] workspace: sums of the segments, then the states before them
  float s_o, s_kv;
  int B, T, H, dk, dv, nseg, seg_len;
  int reverse, shift, end_decay, x0_tr;
  int seg_tr;               // seg holds the states of the walk with k and v swapped, [dv][dk] each: nothing to sum
  int va, vk, vv, vo;       // rows allow 16-byte accesses
};

// Walks of one shape that run side by side (blockIdx.y): one forward, three of the backward pass.
struct WalkSet {
  WalkArgs w[3];
};

__device__ __forceinline__ float decay_pow(float g2, int n) { return n <= 0 ? 1.f : exp2f(g2 * (float)n); }

using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
using u32x2 = __attribute__((ext_vector_type(2))) unsigned;

// Rows of a chunk as a buffer: accesses behind its end read zero and store nothing, so that neither the clip's last chunk nor
// columns behind the head need a branch.  `rows` of them (at most zero: none), `stride` >= `width` elements of `esize` bytes apart,
// `width` elements each.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t chunk_rows(const void* first, int rows, long stride, int width, int esize) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)first, 0, max((rows - 1) * (int)stride + width, 0) * esize, 0x00020000);
}
// A byte offset into such a buffer; one before its start, or of a column that does not exist, lands far behind its end.
__device__ __forceinline__ int chunk_offset(int off, bool exists) { return (int)min((unsigned)(exists ? off : -1), 0x80000000u); }

// A v that is not finite may reach no earlier token: its weight there is zero, but zero times it is not.  Such rows are rare, so
// they cost the walk a test as they come in, and where a chunk holds one behind its first token it ends before it.  The first
// of them goes through LDS (`cut`, one per chunk in flight); CUT_NONE: there is none.
constexpr int CUT_NONE = 1 << 30;

// fp32 arithmetic throughout (v_mfma_f32_16x16x4_f32).  P: dk and dv padded to 16, 32, 64 or 128; P / 16 waves up to four,
// each owning 16 NT of the P state columns.  The contraction index of an MFMA may be permuted as long as both operands agree:
// lane quarter q takes elements 4q..4q+3 of a 16-wide block over four consecutive instructions, so row-major operands are
// 16-byte LDS reads and an accumulator tile (row 4q + r in register r) is the next product's operand as it lies: the state
// never leaves its registers.  Weights and outputs are computed transposed, so that a lane holds four neighbours of a row.  Only
// the C x C weights pass through LDS (each wave computes a share of them).
// VEC: rows of a, k, v and o allow 16-byte accesses; otherwise elements go one by one, through the same buffers.
template <int P, bool STATE_ONLY, bool VEC>
__global__ __launch_bounds__(P >= 64 ? 256 : P * 4, 2) void walk_f32_kernel(WalkSet set) {
  const WalkArgs& w = set.w[blockIdx.y];
  constexpr int NW = P >= 64 ? 4 : P / 16, NT = P / 16 / NW, KT = P / 16, NTHR = NW * 64;
  constexpr int LD = P + 4, LDP = DA_C + 4, SLOTS = DA_C * P / 4 / NTHR, RS = NTHR / (P / 4);
  __shared__ __attribute__((aligned(16))) float sa[STATE_ONLY ? 4 : DA_C * LD];
  __shared__ __attribute__((aligned(16))) float sk[DA_C * LD], sv[DA_C * LD];
  __shared__ __attribute__((aligned(16))) float sp[STATE_ONLY ? 4 : DA_C * LDP];
  __shared__ float pw[DA_C + 1];                             // lam^i
  __shared__ float pv[2 * DA_C];                             // s_kv lam^{31-i}; a chunk of n tokens starts at 32 - n
  __shared__ float pp[DA_C + 16];                            // [15 + i - j]: s_o s_kv lam^{i-j}
  __shared__ int cut[2];
  const int tid = threadIdx.x, wave = NW == 1 ? 0 : tid >> 6, lane = tid & 63, q = lane >> 4, l16 = lane & 15;
  const int bh = blockIdx.x % (w.B * w.H), seg = blockIdx.x / (w.B * w.H);
  const int b = bh / w.H, h = bh % w.H;
  const int len = w.lengths ? min(max(w.lengths[b], 0), w.T) : w.T;
  const int p0 = seg * w.seg_len, p1 = min(p0 + w.seg_len, len);
  const int last_seg = len > 0 ? (len - 1) / w.seg_len : 0;
  float* ob = (float*)w.o + (size_t)b * w.so.b + (size_t)h * w.so.h;
  if (!STATE_ONLY) {
    // rows behind the clip's end are zero
    const int t0 = max(len, p0), t1 = min(p0 + w.seg_len, w.T);
    for (long i = (long)tid; i < (long)(t1 - t0) * w.dv; i += NTHR) ob[(t0 + i / w.dv) * w.so.t + i % w.dv] = 0.f;
  }
  if (STATE_ONLY ? seg >= last_seg : seg > last_seg) return;
  const float g2 = w.log_decay[h] * 1.44269504088896341f;
  for (int i = tid; i < 2 * DA_C; i += NTHR) {
    if (i <= DA_C) pw[i] = decay_pow(g2, i);
    if (i < DA_C + 16) pp[i] = w.s_o * w.s_kv * decay_pow(g2, i - 15);
    pv[i] = w.s_kv * decay_pow(g2, DA_C - 1 - i);
  }
  const float* ab = (const float*)w.a + (size_t)b * w.sa.b + (size_t)h * w.sa.h;
  const float* kb = (const float*)w.k + (size_t)b * w.sk.b + (size_t)h * w.sk.h;
  const float* vb = (const float*)w.v + (size_t)b * w.sv.b + (size_t)h * w.sv.h;

  // ---- state before the segment: X[kt][nt][r] = row kt 16 + 4q + r, column (wave NT + nt) 16 + l
  f32x4 X[KT][NT];
  const size_t mat = (size_t)w.dk * w.dv;
  {
    const bool from_seg = !STATE_ONLY && seg > 0;
    const float* src = STATE_ONLY ? nullptr : from_seg ? w.seg + ((size_t)bh * w.nseg + seg) * mat : w.x0 ? w.x0 + (size_t)bh * mat : nullptr;
    const bool tr = from_seg ? w.seg_tr : w.x0_tr;
    const int sr = tr ? 1 : w.dv, sc = tr ? w.dk : 1;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = kt * 16 + 4 * q + r, col = (wave * NT + nt) * 16 + l16;
          X[kt][nt][r] = src && row < w.dk && col < w.dv ? src[(size_t)row * sr + (size_t)col * sc] : 0.f;
        }
  }

  // arguments of the loop stay in registers: loading one again there waits for every LDS read under way (with a chunk's code in
  // one block, 64 clips of 1001 tokens, 8 heads: fp32 heads of 16 51 -> 44 us forward, of 64 133 -> 127)
  float s_o = w.s_o;
  int reverse = w.reverse, dk = w.dk, dv = w.dv, sa_t = (int)w.sa.t, sk_t = (int)w.sk.t, sv_t = (int)w.sv.t, so_t = (int)w.so.t;
  asm("" : "+s"(s_o), "+s"(reverse), "+s"(dk), "+s"(dv), "+s"(sa_t), "+s"(sk_t), "+s"(sv_t), "+s"(so_t));
  // a thread's SLOTS pieces of a tile are RS rows apart, in the same column
  const int i0 = tid / (P / 4), cc = tid % (P / 4) * 4;
  const int dir = reverse ? -1 : 1;
  f32x4 ra[STATE_ONLY ? 1 : SLOTS], rk[SLOTS], rv[SLOTS];
  auto rows4 = [&](const float* base, int st, int width, int c0, f32x4 (&out)[SLOTS]) {
    const int n = min(DA_C, p1 - c0);                       // none or fewer behind the last chunk
    const auto rs = chunk_rows(base + (reverse ? len - c0 - n : c0) * (long)st, n, st, width, 4);
    const int step = dir * RS * 4 * st;
    int off = (reverse ? n - 1 - i0 : i0) * 4 * st + 4 * cc;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s, off += step) {
      if (VEC) {
        out[s] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, chunk_offset(off, cc < width), 0, 0));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          out[s][e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, chunk_offset(off < 0 ? off : off + 4 * e, cc + e < width), 0, 0));
      }
    }
  };
  auto fetch = [&](int c0) {
    if constexpr (!STATE_ONLY) rows4(ab, sa_t, dk, c0, ra);
    rows4(kb, sk_t, dk, c0, rk);
    rows4(vb, sv_t, dv, c0, rv);
  };
  // returns the first row behind the chunk's first whose v is not finite, among this thread's
  auto put = [&]() {
    int bad = CUT_NONE;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int at = (i0 + s * RS) * LD + cc;
      if constexpr (!STATE_ONLY) *(f32x4*)(sa + at) = ra[s];
      *(f32x4*)(sk + at) = rk[s];
      *(f32x4*)(sv + at) = rv[s];
      if constexpr (!STATE_ONLY) {
        float z = 0.f;                                      // stays zero over finite values
#pragma unroll
        for (int e = 0; e < 4; ++e) z = __builtin_fmaf(rv[s][e], 0.f, z);
        const int row = i0 + s * RS;
        bad = z != 0.f && row > 0 ? min(bad, row) : bad;
      }
    }
    return bad;
  };
  if (p0 < p1) {
    if (!STATE_ONLY && tid < 2) cut[tid] = CUT_NONE;
    fetch(p0);
    const int bad = put();
    if constexpr (!STATE_ONLY) {
      __syncthreads();
      if (bad < CUT_NONE) atomicMin(&cut[0], bad);
    }
  }
  int turn = 0;
  for (int c0 = p0, n; c0 < p1; c0 += n, turn ^= 1) {
    n = min(DA_C, p1 - c0);                                 // tokens in this chunk
    const int shift = w.shift && c0 == 0 ? 1 : 0;
    __syncthreads();
    const int first_bad = STATE_ONLY ? CUT_NONE : cut[turn];
    fetch(c0 + DA_C);                                       // behind the last chunk: zeros, without an access
    if constexpr (!STATE_ONLY) {
      if (__builtin_amdgcn_readfirstlane(first_bad) < CUT_NONE) {
        n = __builtin_amdgcn_readfirstlane(first_bad);
        for (int i = n * LD + tid; i < DA_C * LD; i += NTHR) sk[i] = sv[i] = 0.f;
        fetch(c0 + n);
        __syncthreads();
        if (tid == 0) cut[turn] = CUT_NONE;                 // read by all; next written behind the next barrier
      }
    }
    f32x4 O[2][NT];
    if (!STATE_ONLY) {
      // ---- weights lam^{i-j} (a_i . k_j), transposed: a lane holds four neighbouring j of one i.  One 16 x 16 tile per wave and
      // turn; the tile above the diagonal is never read
#pragma unroll
      for (int u = 0; u < 4 / NW; ++u) {
        const int mt = (u * NW + wave) >> 1, jt = (u * NW + wave) & 1;
        if (jt > mt) continue;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const f32x4 x = *(const f32x4*)(sa + (mt * 16 + l16) * LD + kt * 16 + 4 * q);
          const f32x4 y = *(const f32x4*)(sk + (jt * 16 + l16) * LD + kt * 16 + 4 * q);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(y[r], x[r], acc, 0, 0, 0);
        }
        const int i = mt * 16 + l16, j = jt * 16 + 4 * q;
        float f[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) f[r] = pp[15 + i - j - r];
        // all four are read, whether they count or not: a branch around each would wait for each
        asm("" : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3]));
        const int last = mt == jt ? l16 - 4 * q : 4;
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = r <= last ? acc[r] * f[r] : 0.f;
        *(f32x4*)(sp + i * LDP + j) = acc;
      }
      // ---- what the state contributes, transposed: rows are the wave's columns, columns the tokens
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) O[mt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const f32x4 x = *(const f32x4*)(sa + (mt * 16 + l16) * LD + kt * 16 + 4 * q);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 4; ++r) O[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x4f32(X[kt][nt][r], x[r], O[mt][nt], 0, 0, 0);
        }
        const float f = s_o * pw[mt * 16 + l16 + 1 - shift];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) O[mt][nt] *= f;
      }
    }
    // ---- X = lam^n X + K^T V'
    const float f = pw[n - shift];
    f32x4 V[2][NT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) X[kt][nt] *= f;
#pragma unroll
    for (int jt = 0; jt < 2; ++jt) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) V[jt][nt][r] = sv[(jt * 16 + 4 * q + r) * LD + (wave * NT + nt) * 16 + l16];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float g = pv[DA_C - n + jt * 16 + 4 * q + r];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const float x = sk[(jt * 16 + 4 * q + r) * LD + kt * 16 + l16];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) X[kt][nt] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, V[jt][nt][r] * g, X[kt][nt], 0, 0, 0);
        }
      }
    }
    // every wave is done with the tiles and has left its weights: the next chunk's tiles may be written from here on, its
    // weights only behind the next barrier, i.e. when all have read these
    __syncthreads();
    if (!STATE_ONLY) {
      // ---- O += P V
#pragma unroll
      for (int jt = 0; jt < 2; ++jt)
#pragma unroll
        for (int mt = jt; mt < 2; ++mt) {
          const f32x4 x = *(const f32x4*)(sp + (mt * 16 + l16) * LDP + jt * 16 + 4 * q);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 4; ++r) O[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x4f32(V[jt][nt][r], x[r], O[mt][nt], 0, 0, 0);
        }
    }
    // the next tiles go in before this chunk's rows go out: waiting for loads that are older than a store is not waiting for the
    // store (memory operations are counted in order)
    const int bad = put();
    if (!STATE_ONLY) {
      const auto rs = chunk_rows(ob + (reverse ? len - c0 - n : c0) * (long)so_t, n, so_t, dv, 4);
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int i = mt * 16 + l16, off = (reverse ? n - 1 - i : i) * 4 * so_t;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int col = (wave * NT + nt) * 16 + 4 * q;
          if (VEC) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, O[mt][nt]), rs, chunk_offset(off + 4 * col, i < n && col < dv), 0, 0);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(O[mt][nt][e]), rs, chunk_offset(off + 4 * (col + e), i < n && col + e < dv), 0, 0);
          }
        }
      }
      if (bad < CUT_NONE) atomicMin(&cut[turn ^ 1], bad);
    }
  }
  // ---- state behind the segment
  float* dst = STATE_ONLY ? w.seg + ((size_t)bh * w.nseg + seg) * mat : seg == last_seg && w.x_end ? w.x_end + (size_t)bh * mat : nullptr;
  if (!dst) return;
  const float f = !STATE_ONLY && w.end_decay && len > 0 ? pw[1] : 1.f;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = kt * 16 + 4 * q + r, col = (wave * NT + nt) * 16 + l16;
        if (row < w.dk && col < w.dv) dst[(size_t)row * w.dv + col] = X[kt][nt][r] * f;
      }
}

// 16-bit tokens on the 16-bit matrix cores (v_mfma_f32_16x16x32_bf16 / _f16), 32 or 64 tokens per chunk, P / 16 waves that own 16
// state columns each.  What is rounded to 16 bits on its way into a product, and what is not:
//   * the weights lam^{i-j} (a_i . k_j) and the state as it meets a_i go in as two terms of the type each (2^-15 in bf16, 2^-22 in fp16
//     is left over), so that the output's own rounding is the only one that counts: with one term each its error was 1.41 times that
//     on long clips and up to 2.3 times on single tokens.  The weights' second term costs nothing; the state's, in us before and
//     after: heads of 64, 64 clips of 1001 tokens, 8 heads 70 and 70, one workgroup per CU (256 pairs of 2048 tokens) 80 and 87; heads
//     of 128, 192 pairs 129 and 132, where instruction issue bounds them (8 clips of 4096, 16 heads) 207 and 217 forward, 398 and
//     463 backward;
//   * lam^{n-1-j} v_j on its way into the state is split into three terms of the type (24 bits), since the state is fp32,
//     carried over any number of chunks and returned: X keeps fp32 accuracy at three products per term.
// fp16 has the fraction for that but not the range, so those three operands go in scaled by powers of two that bounds give
// (dk max|a| max|k| for the weights, max|v| for the split values, and for the state the recurrence of the bound itself); X is
// kept in the units of the last chunk's values, or in those in which it stays finite.  The bounds may be far too large: fp16
// stays normal over 2^29.
// Operands: lane (q = lane / 16, l = lane % 16) of an MFMA takes eight contraction indices 8q..8q+7 of row l, and an
// accumulator tile holds rows 4q + r of column l.  Two state tiles whose rows are dealt as 8q + 4s + r (s = tile) together
// are the eight indices the next product wants, so the state stays in registers.  Contractions over tokens read K and V
// through ds_read_b64_tr_b16, which hands a lane four tokens of one column; K's columns lie in LDS as those tiles want
// them (of every 32, the 4-element halves s = 0 first), so that a transposing read takes 32 contiguous bytes of four rows, and
// rows are padded by 32 bytes, so that it touches every bank once.
// Bound: HBM in the end, but first the latency of the chain load - weights - products of a chunk: 16 columns per wave (not
// 32) halve the registers of a wave and put four waves on a SIMD, at twice the LDS reads of a and K.
constexpr int DB_C = 64;

template <typename T>
using x8 = __attribute__((ext_vector_type(8))) T;
template <typename T>
using x2 = __attribute__((ext_vector_type(2))) T;
using u16x2 = __attribute__((ext_vector_type(2))) unsigned short;
using s16x4 = __attribute__((ext_vector_type(4))) short;

template <typename T>
__device__ __forceinline__ u32x4 row8(const T* base, bool live, int c, int width, bool vec) {
  u32x4 r = {0u, 0u, 0u, 0u};
  if (!live) return r;
  if (vec && c + 8 <= width) return *reinterpret_cast<const u32x4*>(base + c);
  x8<T> t;
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = c + i < width ? base[c + i] : (T)0.f;
  return __builtin_bit_cast(u32x4, t);
}

// Eight tokens (rows 8q .. 8q + 7 behind `tile`) of column l of the 16 columns that start there.
template <int LD, typename T>
__device__ __forceinline__ x8<T> read_tokens(const T* tile, int q, int l16) {
  using lds4 = __attribute__((address_space(3))) s16x4;
  const T* p = tile + (8 * q + l16 / 4) * LD + l16 % 4 * 4;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 4 * LD));
  return __builtin_bit_cast(x8<T>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// The two halves of a register as floats, two floats rounded into one, and the product.
template <typename T>
__device__ __forceinline__ float low16(unsigned u) {
  if constexpr (__is_same(T, bf16_t)) return __uint_as_float(u << 16);
  else return (float)__builtin_bit_cast(x2<f16_t>, u)[0];
}
template <typename T>
__device__ __forceinline__ float high16(unsigned u) {
  if constexpr (__is_same(T, bf16_t)) return __uint_as_float(u & 0xffff0000u);
  else return (float)__builtin_bit_cast(x2<f16_t>, u)[1];
}
template <typename T>
__device__ __forceinline__ unsigned pack16(float a, float b) {
  const x2<T> v = {(T)a, (T)b};
  return __builtin_bit_cast(unsigned, v);
}
// The leading term of two floats, and in their place what it leaves of them (exactly).  bf16 cuts: three terms are the whole float.
template <typename T>
__device__ __forceinline__ unsigned split16(float& a, float& b) {
  if constexpr (__is_same(T, bf16_t)) {
    const unsigned ua = __float_as_uint(a), ub = __float_as_uint(b), c = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
    a -= __uint_as_float(ua & 0xffff0000u);
    b -= __uint_as_float(ub & 0xffff0000u);
    return c;
  } else {
    // fixed before and after they are rounded: the compiler would round them once more, each by itself, where a rest is formed, or
    // round the product that leads to a there, and not a, and the terms would not add up
    asm("" : "+v"(a), "+v"(b));
    unsigned c = pack16<T>(a, b);
    asm("" : "+v"(c));
    a -= low16<T>(c);
    b -= high16<T>(c);
    return c;
  }
}
__device__ __forceinline__ f32x4 mfma16(x8<bf16_t> a, x8<bf16_t> b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma16(x8<f16_t> a, x8<f16_t> b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Largest magnitude among the fp16 values of a register, as bits (their order is the integers').
__device__ __forceinline__ u16x2 abs_max16(u16x2 m, unsigned u) { return __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, u & 0x7fff7fffu)); }
__device__ __forceinline__ float pow2(int e) { return ldexpf(1.f, e); }
// The exponent that brings a bound below 2^top, at most 60; a bound of zero, infinity or NaN gives a harmless one.
__device__ __forceinline__ int scale_for(float bound, int top) { return min(top - __builtin_amdgcn_frexp_expf(bound), 60); }

// VEC: rows of a, k, v and o allow 16-byte accesses.
template <typename T, int P, int CC, bool STATE_ONLY, bool VEC>
__global__ __launch_bounds__(P * 4, P == 128 ? 4 : 3) void walk_16_kernel(WalkSet set) {
  const WalkArgs& w = set.w[blockIdx.y];
  constexpr bool F16 = __is_same(T, f16_t);
  constexpr int C = CC, NI = C / 16, TILES = NI * (NI + 1) / 2;
  constexpr int NTHR = P * 4, NW = P / 16, KP = P / 32;      // KP: pairs of state row tiles
  constexpr int LD = P + 16, LDP = C + 8, SLOTS = C * P / 8 / NTHR;
  __shared__ __attribute__((aligned(16))) T sa[STATE_ONLY ? 8 : C * LD];
  __shared__ __attribute__((aligned(16))) T sk[C * LD], sv[C * LD];
  __shared__ __attribute__((aligned(16))) T sp[2][STATE_ONLY ? 8 : C * LDP];   // weights, in two terms
  __shared__ float pw[C + 1];                             // lam^i
  __shared__ float pv[2 * C];                             // s_kv lam^{C-1-i}; a chunk of n tokens starts at C - n
  __shared__ float pp[C + 16];                            // [15 + i - j]: s_o s_kv lam^{i-j}
  __shared__ unsigned top[F16 ? 3 * NW : 1];                 // largest finite a, k, v of the waves' pieces, as bits
  __shared__ int cut[2];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, q = lane >> 4, l16 = lane & 15;
  const int bh = blockIdx.x % (w.B * w.H), seg = blockIdx.x / (w.B * w.H);
  const int b = bh / w.H, h = bh % w.H;
  const int len = w.lengths ? min(max(w.lengths[b], 0), w.T) : w.T;
  const int p0 = seg * w.seg_len, p1 = min(p0 + w.seg_len, len);
  const int last_seg = len > 0 ? (len - 1) / w.seg_len : 0;
  T* ob = (T*)w.o + (size_t)b * w.so.b + (size_t)h * w.so.h;
  if (!STATE_ONLY) {
    // rows behind the clip's end are zero
    const int t0 = max(len, p0), t1 = min(p0 + w.seg_len, w.T);
    for (long i = (long)tid; i < (long)(t1 - t0) * w.dv; i += NTHR) ob[(t0 + i / w.dv) * w.so.t + i % w.dv] = (T)0.f;
  }
  if (STATE_ONLY ? seg >= last_seg : seg > last_seg) return;
  const float g2 = w.log_decay[h] * 1.44269504088896341f;
  for (int i = tid; i < 2 * C; i += NTHR) {
    if (i <= C) pw[i] = decay_pow(g2, i);
    if (i < C + 16) pp[i] = w.s_o * w.s_kv * decay_pow(g2, i - 15);
    pv[i] = w.s_kv * decay_pow(g2, C - 1 - i);
  }
  if (!STATE_ONLY) {
    // the weight tiles (0, 1) and (2, 3) lie above the diagonal but in a pair that is read: they stay zero
    for (int i = tid; i < C / 32 * 256; i += NTHR) {
      const int half = i >> 8, r = i >> 4 & 15, c = i & 15;
      sp[0][(half * 32 + r) * LDP + half * 32 + 16 + c] = sp[1][(half * 32 + r) * LDP + half * 32 + 16 + c] = (T)0.f;
    }
  }
  const T* ab = (const T*)w.a + (size_t)b * w.sa.b + (size_t)h * w.sa.h;
  const T* kb = (const T*)w.k + (size_t)b * w.sk.b + (size_t)h * w.sk.h;
  const T* vb = (const T*)w.v + (size_t)b * w.sv.b + (size_t)h * w.sv.h;
  const int col0 = wave * 16;                                // the wave's state columns

  // X[kp][s][r]: row kp 32 + 8q + 4s + r, column col0 + l
  f32x4 X[KP][2];
  const size_t mat = (size_t)w.dk * w.dv;
  const int xcol = col0 + l16;
  {
    const bool from_seg = !STATE_ONLY && seg > 0;
    const float* src = STATE_ONLY ? nullptr : from_seg ? w.seg + ((size_t)bh * w.nseg + seg) * mat : w.x0 ? w.x0 + (size_t)bh * mat : nullptr;
    const bool tr = from_seg ? w.seg_tr : w.x0_tr;
    const int sr = tr ? 1 : w.dv, sc = tr ? w.dk : 1;
#pragma unroll
    for (int kp = 0; kp < KP; ++kp)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = kp * 32 + 8 * q + 4 * s + r;
          X[kp][s][r] = src && row < w.dk && xcol < w.dv ? src[(size_t)row * sr + (size_t)xcol * sc] : 0.f;
        }
  }

  int E = 0;            // fp16: X is held times 2^E
  float bound = 0.f;    // fp16: no element of X is larger
  if constexpr (F16) {
#pragma unroll
    for (int kp = 0; kp < KP; ++kp)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int r = 0; r < 4; ++r) bound = fmaxf(bound, fabsf(X[kp][s][r]) < INFINITY ? fabsf(X[kp][s][r]) : 0.f);
    bound = wave_reduce_max(bound);
  }

  // as in the fp32 kernel: in registers for the loop
  float s_o = w.s_o;
  int reverse = w.reverse, dk = w.dk, dv = w.dv, sa_t = (int)w.sa.t, sk_t = (int)w.sk.t, sv_t = (int)w.sv.t, so_t = (int)w.so.t;
  asm("" : "+s"(s_o), "+s"(reverse), "+s"(dk), "+s"(dv), "+s"(sa_t), "+s"(sk_t), "+s"(sv_t), "+s"(so_t));
  // a thread's SLOTS pieces of a tile are RS rows apart, in the same column
  constexpr int RS = NTHR / (P / 8);
  const int i0 = tid / (P / 8), cc = tid % (P / 8) * 8;
  const int dir = reverse ? -1 : 1;
  u32x4 ra[STATE_ONLY ? 1 : SLOTS], rk[SLOTS], rv[SLOTS];
  auto rows8 = [&](const T* base, int st, int width, bool vec, int c0, u32x4 (&out)[SLOTS]) {
    const int n = min(C, p1 - c0);                       // none or fewer behind the last chunk
    if (VEC) {
      const auto rs = chunk_rows(base + (reverse ? len - c0 - n : c0) * (long)st, n, st, width, 2);
      const int step = dir * RS * 2 * st;
      int off = (reverse ? n - 1 - i0 : i0) * 2 * st + 2 * cc;
#pragma unroll
      for (int s = 0; s < SLOTS; ++s, off += step)
        out[s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, chunk_offset(off, cc < width), 0, 0));
    } else {
#pragma unroll
      for (int s = 0; s < SLOTS; ++s) {
        const int p = c0 + i0 + s * RS;
        const bool live = p < p1;
        out[s] = row8(base + (live ? (reverse ? len - 1 - p : p) : 0) * (long)st, live, cc, width, vec);
      }
    }
  };
  auto fetch = [&](int c0) {
    if constexpr (!STATE_ONLY) rows8(ab, sa_t, dk, w.va, c0, ra);
    rows8(kb, sk_t, dk, w.vk, c0, rk);
    rows8(vb, sv_t, dv, w.vv, c0, rv);
  };
  // returns the first row behind the chunk's first whose v is not finite, among this thread's
  auto put = [&]() {
    int bad = CUT_NONE;
    u16x2 m[3] = {};                                        // largest a, k, v
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int at = (i0 + s * RS) * LD + cc;
      if (!STATE_ONLY) *(u32x4*)(sa + at) = ra[s];
      T* kd = sk + (i0 + s * RS) * LD + cc / 32 * 32 + cc % 32 / 2;
      *(uint2*)kd = make_uint2(rk[s][0], rk[s][1]);
      *(uint2*)(kd + 16) = make_uint2(rk[s][2], rk[s][3]);
      *(u32x4*)(sv + at) = rv[s];
      u16x2 mv = {};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (F16 && !STATE_ONLY) m[0] = abs_max16(m[0], ra[s][e]);
        if constexpr (F16) m[1] = abs_max16(m[1], rk[s][e]);
        if constexpr (F16 || !STATE_ONLY) mv = abs_max16(mv, rv[s][e]);
      }
      if constexpr (F16) m[2] = __builtin_elementwise_max(m[2], mv);
      if constexpr (!STATE_ONLY) {
        const int row = i0 + s * RS;
        bad = max(mv[0], mv[1]) >= (F16 ? 0x7c00 : 0x7f80) && row > 0 ? min(bad, row) : bad;
      }
    }
    if constexpr (F16) {
#pragma unroll
      for (int z = STATE_ONLY ? 1 : 0; z < 3; ++z) {
        unsigned u = max(m[z][0], m[z][1]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) u = max(u, (unsigned)__shfl_xor((int)u, o, 64));
        if (u >= 0x7c00) {                                  // (the whole wave) a value that is not finite says nothing about the others
          u = 0;
          for (int s = 0; s < SLOTS; ++s)
            for (int e = 0; e < 8; ++e) {
              const unsigned x = (z == 0 ? ra[STATE_ONLY ? 0 : s] : z == 1 ? rk[s] : rv[s])[e >> 1] >> (e & 1) * 16 & 0x7fff;
              u = max(u, x < 0x7c00 ? x : 0u);
            }
          for (int o = 32; o > 0; o >>= 1) u = max(u, (unsigned)__shfl_xor((int)u, o, 64));
        }
        if (lane == 0) top[z * NW + wave] = u;
      }
    }
    return bad;
  };
  if (p0 < p1) {
    if (!STATE_ONLY && tid < 2) cut[tid] = CUT_NONE;
    fetch(p0);
    const int bad = put();
    if constexpr (!STATE_ONLY) {
      __syncthreads();
      if (bad < CUT_NONE) atomicMin(&cut[0], bad);
    }
  }
  int turn = 0;
  for (int c0 = p0, n; c0 < p1; c0 += n, turn ^= 1) {
    n = min(C, p1 - c0);                                 // tokens in this chunk
    const int shift = w.shift && c0 == 0 ? 1 : 0;
    __syncthreads();
    const int first_bad = STATE_ONLY ? CUT_NONE : cut[turn];
    if (P < 128 || STATE_ONLY || c0 + C < p1) fetch(c0 + C);   // behind the last chunk: zeros, without an access
    if constexpr (!STATE_ONLY) {
      if (__builtin_amdgcn_readfirstlane(first_bad) < CUT_NONE) {
        n = __builtin_amdgcn_readfirstlane(first_bad);
        for (int i = n * LD + tid; i < C * LD; i += NTHR) sk[i] = sv[i] = (T)0.f;
        fetch(c0 + n);
        __syncthreads();
        if (tid == 0) cut[turn] = CUT_NONE;                 // read by all; next written behind the next barrier
      }
    }
    float unit_p = 1.f, unit_x = 1.f, back = 1.f, unit_v = 1.f, carry = 1.f, largest = 0.f;
    if constexpr (F16) {
      float big[3];
#pragma unroll
      for (int z = 0; z < 3; ++z) {
        unsigned u = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) u = max(u, STATE_ONLY && z == 0 ? 0u : top[z * NW + i]);
        big[z] = (float)__builtin_bit_cast(f16_t, (unsigned short)u);
      }
      largest = fabsf(w.s_kv) * big[1] * big[2] * (float)n;
      // a state near fp32's end takes the exponents down, so that X 2^ev and the units of X's product stay finite: for |X| up to
      // 2^e the split values lose what lies below 2^(e - 150) and the weights what lies below 2^(e - 165)
      const int ex = scale_for(bound, 14);
      const int ep = min(scale_for((float)P * fabsf(s_o * w.s_kv) * big[0] * big[1], 15), 126 + ex);
      const int ev = min(scale_for(fabsf(w.s_kv) * big[2], 15), 126 - __builtin_amdgcn_frexp_expf(fminf(bound + largest, 3e38f)));
      unit_p = pow2(ep);                // weights
      unit_x = pow2(ex - E);            // X as an operand
      back = pow2(ep - ex);             // its product, in the weights' units
      unit_v = pow2(ev);                // values on their way into X
      carry = pow2(ev - E);
      E = ev;
    }
    const float decay = pw[n - shift] * carry;
    f32x4 O[STATE_ONLY ? 1 : NI];
    if (!STATE_ONLY) {
      // ---- weights, transposed tile by tile (rows j, columns i) so that a lane holds four neighbouring j of one i: the
      // 16 x 16 tiles on and below the diagonal, in the order (0,0) (1,0) (1,1) (2,0) ..., are dealt over the waves
#pragma unroll P == 128 ? 1 : 5   // eight waves have two tiles at most, and no registers for both at once
      for (int u = 0; u * NW < TILES; ++u) {
        const int tile = u * NW + wave;
        if ((u + 1) * NW > TILES && tile >= TILES) break;
        const int it = 0xffa94 >> (2 * tile) & 3, jt = tile - it * (it + 1) / 2;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kp = 0; kp < KP; ++kp) {
          const T* kr = sk + (jt * 16 + l16) * LD + kp * 32 + 4 * q;
          const uint2 k0 = *(const uint2*)kr, k1 = *(const uint2*)(kr + 16);
          const x8<T> x = __builtin_bit_cast(x8<T>, u32x4{k0.x, k0.y, k1.x, k1.y});
          const x8<T> y = *(const x8<T>*)(sa + (it * 16 + l16) * LD + kp * 32 + 8 * q);
          acc = mfma16(x, y, acc);
        }
        const int i = it * 16 + l16, j = jt * 16 + 4 * q;
        float f[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) f[r] = pp[15 + i - j - r];
        // all four are read, whether they count or not: a branch around each would wait for each
        asm("" : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3]));
        const int last = it == jt ? l16 - 4 * q : 4;
#pragma unroll
        for (int r = 0; r < 4; ++r) f[r] = r <= last ? acc[r] * (F16 ? unit_p * f[r] : f[r]) : 0.f;
        *(uint2*)(sp[0] + i * LDP + j) = make_uint2(split16<T>(f[0], f[1]), split16<T>(f[2], f[3]));
        *(uint2*)(sp[1] + i * LDP + j) = make_uint2(pack16<T>(f[0], f[1]), pack16<T>(f[2], f[3]));
      }
      // ---- what the state contributes, transposed: rows are the wave's columns, columns the tokens.  X goes on decayed; its old
      // registers are split where they lie
#pragma unroll
      for (int it = 0; it < NI; ++it) O[it] = f32x4{0.f, 0.f, 0.f, 0.f};
      // All of the first terms, then the second ones, which are formed while the products run; in wide heads they add to tiles of
      // their own, so that the two do not wait for each other (bf16), and where registers are short (LEAN: fp16, single values) each
      // pair of terms is used up at once (fp16, 8 clips of 2048 tokens, 16 heads of 100: 348 -> 297 us)
      constexpr bool LEAN = P == 128 && (F16 || !VEC), APART = P == 128 && !F16;   // APART: the same sums whatever VEC is
      u32x4 low[KP];
      x8<T> y[KP][NI];
      f32x4 R[NI];
#pragma unroll
      for (int it = 0; it < NI; ++it) R[it] = f32x4{0.f, 0.f, 0.f, 0.f};
      auto second = [&](int kp) {
#pragma unroll
        for (int it = 0; it < NI; ++it) {
          f32x4& to = APART ? R[it] : O[it];
          to = mfma16(__builtin_bit_cast(x8<T>, low[kp]), y[kp][it], to);
        }
      };
#pragma unroll
      for (int kp = 0; kp < KP; ++kp) {
        u32x4 high;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x0 = X[kp][e >> 1][2 * (e & 1)], x1 = X[kp][e >> 1][2 * (e & 1) + 1];
          if constexpr (F16) x0 *= unit_x, x1 *= unit_x;
          high[e] = split16<T>(x0, x1);
          low[kp][e] = pack16<T>(x0, x1);
        }
#pragma unroll
        for (int it = 0; it < NI; ++it) {
          y[kp][it] = *(const x8<T>*)(sa + (it * 16 + l16) * LD + kp * 32 + 8 * q);
          O[it] = mfma16(__builtin_bit_cast(x8<T>, high), y[kp][it], O[it]);
        }
        if constexpr (LEAN) second(kp);
      }
      if constexpr (!LEAN) {
#pragma unroll
        for (int kp = 0; kp < KP; ++kp) second(kp);
      }
      if constexpr (APART) {
#pragma unroll
        for (int it = 0; it < NI; ++it) O[it] += R[it];
      }
#pragma unroll
      for (int it = 0; it < NI; ++it) O[it] *= s_o * pw[it * 16 + l16 + 1 - shift] * back;
    }
    // ---- X = lam^n X + K^T V'
    x8<T> v[C / 32];
    if constexpr (F16) bound = fminf(bound * pw[n - shift] + largest, 3e38f);
#pragma unroll
    for (int kp = 0; kp < KP; ++kp)
#pragma unroll
      for (int s = 0; s < 2; ++s) X[kp][s] *= decay;
#pragma unroll
    for (int jj = 0; jj < C / 32; ++jj) {
      v[jj] = read_tokens<LD, T>(sv + jj * 32 * LD + col0, q, l16);
      u32x4 t[3];
      const float* f8 = pv + C - n + jj * 32 + 8 * q;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned u = __builtin_bit_cast(u32x4, v[jj])[e];
        float y0 = low16<T>(u) * (F16 ? unit_v * f8[2 * e] : f8[2 * e]), y1 = high16<T>(u) * (F16 ? unit_v * f8[2 * e + 1] : f8[2 * e + 1]);
#pragma unroll
        for (int z = 0; z < 2; ++z) t[z][e] = split16<T>(y0, y1);
        t[2][e] = pack16<T>(y0, y1);
      }
#pragma unroll
      for (int kp = 0; kp < KP; ++kp)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const x8<T> x = read_tokens<LD, T>(sk + jj * 32 * LD + kp * 32 + 16 * s, q, l16);
#pragma unroll
          for (int z = 2; z >= 0; --z) X[kp][s] = mfma16(x, __builtin_bit_cast(x8<T>, t[z]), X[kp][s]);
        }
    }
    // every wave is done with the tiles and has left its weights: the next chunk's tiles may be written from here on, its
    // weights only behind the next barrier, i.e. when all have read these
    __syncthreads();
    if (!STATE_ONLY) {
      // ---- O += P V
#pragma unroll
      for (int jj = 0; jj < C / 32; ++jj)
#pragma unroll
        for (int z = 1; z >= 0; --z)
#pragma unroll
          for (int it = 2 * jj; it < NI; ++it) {
            const x8<T> y = *(const x8<T>*)(sp[z] + (it * 16 + l16) * LDP + jj * 32 + 8 * q);
            O[it] = mfma16(v[jj], y, O[it]);
          }
    }
    // the next tiles go in before this chunk's rows go out: waiting for loads that are older than a store is not waiting for the
    // store (memory operations are counted in order).  Wide heads have no registers to hold both, and other waves to run.
    int bad = CUT_NONE;
    if constexpr (P < 128) bad = put();
    if (!STATE_ONLY) {
      const int col = col0 + 4 * q;
      const auto rs = chunk_rows(ob + (reverse ? len - c0 - n : c0) * (long)so_t, n, so_t, dv, 2);
#pragma unroll
      for (int it = 0; it < NI; ++it) {
        const int i = it * 16 + l16;
        if constexpr (F16) O[it] *= 1.f / unit_p;
        const u32x2 y = {pack16<T>(O[it][0], O[it][1]), pack16<T>(O[it][2], O[it][3])};
        const int row = reverse ? n - 1 - i : i;
        if (VEC) {
          __builtin_amdgcn_raw_buffer_store_b64(y, rs, chunk_offset(row * 2 * so_t + 2 * col, col < dv), 0, 0);
        } else if (i < n) {
          T* op = ob + ((reverse ? len - c0 - n : c0) + row) * (long)so_t + col;
          const auto z = __builtin_bit_cast(typename VecOf<T, 4>::type, y);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col + e < dv) op[e] = z[e];
        }
      }
    }
    if constexpr (P == 128) bad = put();
    if (!STATE_ONLY && bad < CUT_NONE) atomicMin(&cut[turn ^ 1], bad);
  }
  // ---- state behind the segment
  float* dst = STATE_ONLY ? w.seg + ((size_t)bh * w.nseg + seg) * mat : seg == last_seg && w.x_end ? w.x_end + (size_t)bh * mat : nullptr;
  if (!dst) return;
  const float f = (!STATE_ONLY && w.end_decay && len > 0 ? pw[1] : 1.f) * (F16 ? pow2(-E) : 1.f);
#pragma unroll
  for (int kp = 0; kp < KP; ++kp)
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = kp * 32 + 8 * q + 4 * s + r;
        if (row < w.dk && xcol < w.dv) dst[(size_t)row * w.dv + xcol] = X[kp][s][r] * f;
      }
}

// Sums of the segments -> states before the segments, in place: seg[s] = lam^{seg_len} seg[s-1] + sum[s-1], seg[0] = x0.  The
// shifted first decay of a reversed walk is that of segment 0.
__global__ __launch_bounds__(256) void walk_scan_kernel(WalkSet set) {
  const WalkArgs& w = set.w[blockIdx.z];
  const int mat = w.dk * w.dv;
  const int e = blockIdx.x * 256 + threadIdx.x;
  const int bh = blockIdx.y;
  if (e >= mat) return;
  const int b = bh / w.H, h = bh % w.H;
  const int len = w.lengths ? min(max(w.lengths[b], 0), w.T) : w.T;
  const int nseg = len > 0 ? (len - 1) / w.seg_len : 0;
  const float g2 = w.log_decay[h] * 1.44269504088896341f;
  const float f = decay_pow(g2, w.seg_len), f0 = w.shift ? decay_pow(g2, w.seg_len - 1) : f;
  float x = 0.f;
  if (w.x0) x = w.x0[(size_t)bh * mat + (w.x0_tr ? (size_t)(e % w.dv) * w.dk + e / w.dv : (size_t)e)];
  float* p = w.seg + (size_t)bh * w.nseg * mat + e;
  float sum = nseg > 0 ? p[0] : 0.f;
  for (int s = 1; s <= nseg; ++s) {
    const float next = s < nseg ? p[(size_t)s * mat] : 0.f;
    x = x * (s == 1 ? f0 : f) + sum;
    p[(size_t)s * mat] = x;
    sum = next;
  }
}

// One token per clip: the state is read and written once.  A workgroup owns one (clip, head); a thread owns four (or one)
// neighbouring columns of every RG-th row, the row groups meet in LDS for o.
template <typename T, int V>
__global__ __launch_bounds__(256) void step_kernel(const T* __restrict__ q, Strides sq, const T* __restrict__ k, Strides sk,
                                                   const T* __restrict__ v, Strides sv, const float* __restrict__ log_decay,
                                                   float* __restrict__ state, T* __restrict__ o, int H, int dk, int dv,
                                                   float scale) {
  __shared__ float red[256 * V];
  const int b = blockIdx.x / H, h = blockIdx.x % H;
  const int cols = (dv + V - 1) / V, groups = 256 / cols;     // dv <= 128 V
  const int c = threadIdx.x % cols * V, grp = threadIdx.x / cols;
  const float lam = decay_pow(log_decay[h] * 1.44269504088896341f, 1);
  const T* qp = q + (size_t)b * sq.b + (size_t)h * sq.h;
  const T* kp = k + (size_t)b * sk.b + (size_t)h * sk.h;
  const T* vp = v + (size_t)b * sv.b + (size_t)h * sv.h;
  float* sp = state + ((size_t)b * H + h) * dk * dv;
  float acc[V], vv[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    acc[i] = 0.f;
    vv[i] = (float)vp[c + i];
  }
  if (grp < groups) {
    // four rows requested before the first is worked on
    for (int r0 = grp; r0 < dk; r0 += 4 * groups) {
      float x[4][V], kr[4], qr[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = min(r0 + u * groups, dk - 1);
        load_vec<float, V>(sp + (size_t)r * dv + c, x[u]);
        kr[u] = (float)kp[r];
        qr[u] = (float)qp[r];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = r0 + u * groups;
        if (r >= dk) break;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[u][i] = x[u][i] * lam + kr[u] * vv[i];
          acc[i] += qr[u] * x[u][i];
        }
        store_vec<float, V>(sp + (size_t)r * dv + c, x[u]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) red[threadIdx.x * V + i] = acc[i];
  __syncthreads();
  if (grp == 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float t = 0.f;
      for (int j = 0; j < groups; ++j) t += red[(j * cols + threadIdx.x) * V + i];
      o[((size_t)b * H + h) * dv + c + i] = (T)(t * scale);
    }
  }
}

// Whether pieces of `v` elements of a row may be accessed as one: 16 bytes, and a row is a whole number of them.
bool rows_vec(const void* p, const Strides& s, int width, int v, int esize) {
  return ((uintptr_t)p % (v * esize)) == 0 && s.b % v == 0 && s.t % v == 0 && s.h % v == 0 && width % v == 0;
}
// Whether a chunk's rows make a buffer: rows apart, and offsets below 2^31 bytes.
bool rows_apart(const Strides& s, int width) { return s.t >= width && s.t < (1L << 22); }

// The passes of `n` walks of one shape: segment sums and scan for the first `sums` of them (the others reuse those), then the
// walks themselves.  vec: all rows of all walks allow 16-byte accesses.
template <typename Launch>
void walk_passes(const WalkSet& set, int n, int sums, hipStream_t st, Launch launch) {
  const WalkArgs& w = set.w[0];
  const dim3 grid((unsigned)w.B * w.H * w.nseg);
  if (w.nseg > 1) {
    launch(dim3(grid.x, sums), std::true_type());
    hipLaunchKernelGGL(walk_scan_kernel, dim3(noise_cdiv((long)w.dk * w.dv, 256), w.B * w.H, sums), dim3(256), 0, st, set);
  }
  launch(dim3(grid.x, n), std::false_type());
}

bool walk_vec(const WalkSet& set, int n) {
  bool vec = true;
  for (int i = 0; i < n; ++i) vec = vec && set.w[i].va && set.w[i].vk && set.w[i].vv && set.w[i].vo;
  return vec;
}

void walk_launch_f32(const WalkSet& set, int n, int sums, hipStream_t st) {
  const int d = set.w[0].dk > set.w[0].dv ? set.w[0].dk : set.w[0].dv;
  const bool vec = walk_vec(set, n);
  walk_passes(set, n, sums, st, [&](dim3 grid, auto only) {
    constexpr bool ONLY = decltype(only)::value;
#define GO(P)                                                                                                         \
  do {                                                                                                                \
    if (vec) hipLaunchKernelGGL((walk_f32_kernel<P, ONLY, true>), grid, dim3(P >= 64 ? 256 : P * 4), 0, st, set);     \
    else hipLaunchKernelGGL((walk_f32_kernel<P, ONLY, false>), grid, dim3(P >= 64 ? 256 : P * 4), 0, st, set);        \
  } while (0)
    if (d <= 16) GO(16);
    else if (d <= 32) GO(32);
    else if (d <= 64) GO(64);
    else GO(128);
#undef GO
  });
}

template <typename T>
void walk_launch_16(const WalkSet& set, int n, int sums, hipStream_t st) {
  const int d = set.w[0].dk > set.w[0].dv ? set.w[0].dk : set.w[0].dv;
  const bool vec = walk_vec(set, n);
  // tokens per chunk: 32 for heads of 128, where 64 spill registers (273 -> 251 us for 32 clips of 2048 tokens, 16 heads; at 32 the
  // kernels for rows of 16-byte pieces spill 3 in bf16 and none in fp16, those for single values 11 and 30), and for bf16
  // heads of up to 64, where 64 cost a workgroup per CU: heads of 64, 64 clips of 2048 tokens, 8 heads 139 -> 126 us (fp16: 150 ->
  // 163); heads of 16, 64 clips of 1001 forward 44 -> 39 us, backward 109 -> 97 (fp16: 66 -> 72 and 133 -> 109, so by direction
  // there).  One long clip, which has few workgroups anyway, loses by it: 60001 tokens with 16 heads of 32 283 -> 331 us
  // backward.  A pass that keeps only the state has the registers for 64 (60001 tokens, 16 heads of 128: 149 -> 134 us)
  constexpr int C64 = __is_same(T, bf16_t) ? 32 : 64;
  walk_passes(set, n, sums, st, [&](dim3 grid, auto only) {
    constexpr bool ONLY = decltype(only)::value;
#define GO(P, C)                                                                                       \
  do {                                                                                                 \
    if (vec) hipLaunchKernelGGL((walk_16_kernel<T, P, C, ONLY, true>), grid, dim3(P * 4), 0, st, set); \
    else hipLaunchKernelGGL((walk_16_kernel<T, P, C, ONLY, false>), grid, dim3(P * 4), 0, st, set);    \
  } while (0)
    if (d <= 32 && n > 1) GO(32, 32);
    else if (d <= 32) GO(32, C64);
    else if (d <= 64) GO(64, C64);
    else GO(128, (ONLY ? 64 : 32));
#undef GO
  });
}

int walk_launch(const WalkSet& set, int n, int sums, int dtype, hipStream_t st) {
  if (dtype == NOISE_F32) walk_launch_f32(set, n, sums, st);
  else if (dtype == NOISE_BF16) walk_launch_16<bf16_t>(set, n, sums, st);
  else walk_launch_16<f16_t>(set, n, sums, st);
  return 0;
}

// Segments of the token axis.  From `full` (clip, head) pairs on, clips and heads fill the GPU well enough that the second
// read of k and v costs more than it gives; below, the axis is cut until there are `target` workgroups.  A workgroup has one wave
// per 16 columns (fp32: at most four), so narrow heads need more of them; a backward pass has three walks per pair in flight and
// pays for segments with two sums, so it needs fewer.  Measured on 2048 tokens, us with 1 / 2 / 4 / 8 segments, forward:
//   bf16, heads of 16: 256 pairs 66 / 68 / 60 / 66, 128 pairs 66 / 62 / 43 / 39; of 64: 256 pairs 84 / 107 / 104 / 125, 192 pairs
//   83 / 100 / 83 / 94; of 128: 192 pairs 139 / 175 / 189 / 224, 128 pairs 130 / 124 / 126 / 150; fp16, heads of 16: 384 pairs
//   117 / 100 / 105 / 111; fp32, heads of 128: 192 pairs 433 / 483 / 431 / 461, 128 pairs 430 / 343 / 296 / 314
// backward: bf16, heads of 64: 128 pairs 107 / 131 / 127 / 142, 64 pairs 80 / 87 / 65 / 70; of 128: 96 pairs 213 / 241 / 238 / 274;
//   fp32, heads of 128: 128 pairs 693 / 728 / 718 / 763, 96 pairs 688 / 711 / 586 / 588.
// Of 96 cases of 16-bit heads the rule misses the best of the four by more than 6 % in 14, by up to 18 % (fp16 heads of up to 32
// backwards, 64 pairs: 62 us where 8 segments take 51).
// No segment is shorter than 64 tokens or than twice the head: its state is written, scanned and read again.
int walk_nseg(int B, int T, int H, int dk, int dv, int dtype, int backward) {
  static const int rule[3][2][4][2] = {   // {full, target} by type, direction and heads of up to 16, 32, 64, 128
      {{{384, 1024}, {512, 1024}, {256, 768}, {192, 512}}, {{192, 384}, {256, 512}, {128, 256}, {128, 256}}},    // fp32
      {{{256, 768}, {256, 768}, {256, 768}, {192, 512}}, {{128, 256}, {128, 256}, {128, 256}, {64, 256}}},       // bf16
      {{{512, 1024}, {512, 1024}, {384, 768}, {192, 512}}, {{192, 384}, {192, 384}, {128, 256}, {96, 256}}}};    // fp16
  const int d = dk > dv ? dk : dv;
  const int* f = rule[dtype][backward ? 1 : 0][d <= 16 ? 0 : d <= 32 ? 1 : d <= 64 ? 2 : 3];
  const long bh = (long)B * H;
  if (bh >= f[0]) return 1;
  const long want = (f[1] + bh - 1) / bh, most = T / (d <= 32 ? 64 : 2 * d);
  const long n = want < most ? want : most;
  return n < 1 ? 1 : (int)n;
}

const char* walk_check(int B, int T, int H, int dk, int dv, int dtype) {
  if (B < 1 || T < 1 || H < 1) return "empty shape";
  if (T > 1 << 30) return "more than 2^30 tokens";   // the token numbers of a segment's last chunk stay below 2^31
  if (dk < 1 || dk > 128 || dv < 1 || dv > 128) return "head sizes are 1..128";
  if ((long)B * H > (1L << 22)) return "more than 2^22 (clip, head) pairs in one call";   // a grid holds at most 2^32 threads
  if (dtype < NOISE_F32 || dtype > NOISE_F16) return "unknown element type";
  return nullptr;
}

}  // namespace

// Fills in what a walk derives from its shape; an error text, or null.
static const char* walk_plan(WalkArgs& w, int nseg, int dtype) {
  w.seg_len = (noise_cdiv(w.T, nseg) + DB_C - 1) / DB_C * DB_C;
  w.nseg = noise_cdiv(w.T, w.seg_len);
  if (w.nseg > 1 && !w.seg) return "this shape needs a workspace";
  if (!(rows_apart(w.sa, w.dk) && rows_apart(w.sk, w.dk) && rows_apart(w.sv, w.dv) && rows_apart(w.so, w.dv)))
    return "a token stride is below the row's width or not below 2^22 elements";
  const int piece = dtype == NOISE_F32 ? 4 : 8, es = dtype == NOISE_F32 ? 4 : 2;
  w.va = rows_vec(w.a, w.sa, w.dk, piece, es), w.vk = rows_vec(w.k, w.sk, w.dk, piece, es);
  w.vv = rows_vec(w.v, w.sv, w.dv, piece, es), w.vo = rows_vec(w.o, w.so, w.dv, piece, es);
  return nullptr;
}

// Whether two buffers of n floats share memory (null: no buffer).
static bool states_meet(const float* a, const float* b, size_t n) {
  return a && b && (uintptr_t)a < (uintptr_t)(b + n) && (uintptr_t)b < (uintptr_t)(a + n);
}

// Floats of workspace a forward (backward) pass of this shape needs.
NOISE_EXPORT long noise_decay_attn_workspace(int B, int T, int H, int dk, int dv, int dtype, int backward) {
  if (walk_check(B, T, H, dk, dv, dtype)) return 0;
  const int n = walk_nseg(B, T, H, dk, dv, dtype, backward);
  return n > 1 ? (long)B * H * n * dk * dv * (backward ? 2 : 1) : 0;
}

// strides: (clip, token, head) of q, k, v and o
NOISE_EXPORT int noise_decay_attn_fwd(const void* q, const void* k, const void* v, void* o, const long* strides,
                                      const float* log_decay, const int* lengths, const float* state, float* end,
                                      float* workspace, float scale, int B, int T, int H, int dk, int dv, int dtype, void* stream) {
  const char* why = walk_check(B, T, H, dk, dv, dtype);
  NOISE_REQUIRE(!why, "noise_decay_attn_fwd: %s (B %d, T %d, H %d, head sizes %d and %d)", why, B, T, H, dk, dv);
  NOISE_REQUIRE(q && k && v && o && strides && log_decay, "noise_decay_attn_fwd: null pointer");
  // the last segment's workgroup writes one while the first's reads the other
  NOISE_REQUIRE(!states_meet(state, end, (size_t)B * H * dk * dv), "noise_decay_attn_fwd: state and end share memory");
  const Strides* st = (const Strides*)strides;
  WalkSet set = {};
  WalkArgs& w = set.w[0];
  w.a = q, w.k = k, w.v = v, w.o = o, w.sa = st[0], w.sk = st[1], w.sv = st[2], w.so = st[3];
  w.log_decay = log_decay, w.lengths = lengths, w.x0 = state, w.x_end = end, w.seg = workspace, w.s_o = scale, w.s_kv = 1.f;
  w.B = B, w.T = T, w.H = H, w.dk = dk, w.dv = dv;
  why = walk_plan(w, walk_nseg(B, T, H, dk, dv, dtype, 0), dtype);
  NOISE_REQUIRE(!why, "noise_decay_attn_fwd: %s", why);
  walk_launch(set, 1, 1, dtype, (hipStream_t)stream);
  NOISE_CHECK_LAUNCH("noise_decay_attn_fwd");
  return 0;
}

// strides: (clip, token, head) of do, q, k, v, dq, dk, dv
NOISE_EXPORT int noise_decay_attn_bwd(const void* go, const void* q, const void* k, const void* v, void* dq, void* gk, void* gv,
                                      const long* strides, const float* log_decay, const int* lengths, const float* state,
                                      const float* d_end, float* d_state, float* workspace, float scale, int B, int T, int H,
                                      int dk, int dv, int dtype, void* stream) {
  const char* why = walk_check(B, T, H, dk, dv, dtype);
  NOISE_REQUIRE(!why, "noise_decay_attn_bwd: %s (B %d, T %d, H %d, head sizes %d and %d)", why, B, T, H, dk, dv);
  NOISE_REQUIRE(go && q && k && v && dq && gk && gv && strides && log_decay, "noise_decay_attn_bwd: null pointer");
  const Strides* st = (const Strides*)strides;
  const int nseg = walk_nseg(B, T, H, dk, dv, dtype, 1);
  float* ws2 = workspace ? workspace + (size_t)B * H * nseg * dk * dv : nullptr;
  WalkSet set = {};
  WalkArgs &x = set.w[0], &y = set.w[1], &z = set.w[2];
  // dq: first token first, X = S^T
  x.a = go, x.k = v, x.v = k, x.o = dq, x.sa = st[0], x.sk = st[3], x.sv = st[2], x.so = st[4];
  x.x0 = state, x.x0_tr = 1, x.seg = workspace, x.s_o = scale, x.s_kv = 1.f, x.dk = dv, x.dv = dk;
  // dv: last token first, X = dS
  y.a = k, y.k = q, y.v = go, y.o = gv, y.sa = st[2], y.sk = st[1], y.sv = st[0], y.so = st[6];
  y.x0 = d_end, y.x_end = d_state, y.seg = ws2, y.s_o = 1.f, y.s_kv = scale, y.dk = dk, y.dv = dv;
  // dk: the same with X transposed; it starts from the segments' states of dv
  z.a = v, z.k = go, z.v = q, z.o = gk, z.sa = st[3], z.sk = st[0], z.sv = st[1], z.so = st[5];
  z.x0 = d_end, z.x0_tr = 1, z.seg = ws2, z.seg_tr = 1, z.s_o = 1.f, z.s_kv = scale, z.dk = dv, z.dv = dk;
  for (int i = 0; i < 3; ++i) {
    WalkArgs& w = set.w[i];
    w.log_decay = log_decay, w.lengths = lengths, w.B = B, w.T = T, w.H = H;
    w.reverse = w.shift = w.end_decay = i > 0;
    why = walk_plan(w, nseg, dtype);
    NOISE_REQUIRE(!why, "noise_decay_attn_bwd: %s", why);
  }
  // the three walks run side by side: what one writes no other may read
  const size_t states = (size_t)B * H * dk * dv;
  NOISE_REQUIRE(!states_meet(state, d_state, states) && !states_meet(d_end, d_state, states), "noise_decay_attn_bwd: d_state shares memory with state or d_end");
  for (const void* in : {go, q, k, v})
    NOISE_REQUIRE(in != dq && in != gk && in != gv, "noise_decay_attn_bwd: a gradient is written over an input");
  walk_launch(set, 3, 2, dtype, (hipStream_t)stream);
  NOISE_CHECK_LAUNCH("noise_decay_attn_bwd");
  return 0;
}

NOISE_EXPORT int noise_decay_attn_step(const void* q, const void* k, const void* v, const long* strides, const float* log_decay,
                                       float* state, void* o, float scale, int B, int H, int dk, int dv, int dtype,
                                       void* stream) {
  NOISE_REQUIRE(q && k && v && strides && log_decay && state && o, "noise_decay_attn_step: null pointer");
  NOISE_REQUIRE(B > 0 && H > 0 && dk > 0 && dk <= 128 && dv > 0 && dv <= 128 && (long)B * H <= (1L << 23),
                "noise_decay_attn_step: head sizes are 1..128 and at most 2^23 (stream, head) pairs (B %d, H %d, %d and %d)", B, H, dk, dv);
  NOISE_REQUIRE(dtype >= NOISE_F32 && dtype <= NOISE_F16, "noise_decay_attn_step: unknown element type");
  // o may be q, k or v itself, packed (a workgroup reads its rows before it writes them), but no other part of what is read
  const int es = dtype == NOISE_F32 ? 4 : 2;
  const char *o0 = (const char*)o, *o1 = o0 + (size_t)B * H * dv * es, *s0 = (const char*)state;
  bool meets = o0 < s0 + (size_t)B * H * dk * dv * 4 && s0 < o1;
  const void* in[3] = {q, k, v};
  for (int i = 0; i < 3; ++i) {
    const long sb = B > 1 ? strides[2 * i] : 0, sh = H > 1 ? strides[2 * i + 1] : 0;
    const int width = i < 2 ? dk : dv;
    const char *t0 = (const char*)in[i], *t1 = t0 + ((B - 1) * sb + (H - 1) * sh + width) * es;
    const bool same = t0 == o0 && width == dv && (H == 1 || sh == dv) && (B == 1 || sb == (long)H * dv);
    meets = meets || (!same && o0 < t1 && t0 < o1);
  }
  NOISE_REQUIRE(!meets, "noise_decay_attn_step: o shares memory with the state or with a part of q, k or v");
  const Strides sq = {strides[0], 0, strides[1]}, sk = {strides[2], 0, strides[3]}, sv = {strides[4], 0, strides[5]};
  const bool vec = dv % 4 == 0 && ((uintptr_t)state & 15) == 0;
  hipStream_t st = (hipStream_t)stream;
#define GO(T, V) hipLaunchKernelGGL((step_kernel<T, V>), dim3(B * H), dim3(256), 0, st, (const T*)q, sq, (const T*)k, sk, (const T*)v, sv, log_decay, state, (T*)o, H, dk, dv, scale)
  if (dtype == NOISE_F32) { if (vec) GO(float, 4); else GO(float, 1); }
  else if (dtype == NOISE_BF16) { if (vec) GO(bf16_t, 4); else GO(bf16_t, 1); }
  else { if (vec) GO(f16_t, 4); else GO(f16_t, 1); }
#undef GO
  NOISE_CHECK_LAUNCH("noise_decay_attn_step");
  return 0;
}
