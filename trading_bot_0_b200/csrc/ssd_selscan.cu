// Selective scan with a decay per channel and state (the Mamba-1 form):
//     s_t = act(dt_t + dt_bias)          a_t[n] = exp(s_t A[n])          h_t[n] = a_t[n] h_{t-1}[n] + s_t x_t B_t[n]
//     y_t = (sum_n C_t[n] h_t[n] + D x_t) silu(z_t)
// per batch row and channel, B and C shared by the channels of a group; its gradients; and one step over many streams.
//
// The decays differ per channel and state, so there is no matrix form: every (token, channel, state) costs an exponential and a
// handful of fp32 operations, and the special-function units (16 exponentials per clock and SM) set the pace, not the memory
// (one bf16 token-channel is 8 bytes moved against dstate exponentials).  A thread holds eight states of one channel in registers
// (four in the backward, and where a channel has no more) and walks the tokens; neighbouring lanes make up a channel.  What is needed
// once per token and channel (softplus, s x, the gate) is computed once by one thread of the block, a tile of 16 tokens ahead, and
// handed over in shared memory.
#include <initializer_list>

#include "act.cuh"
#include "common.cuh"
#include "ssd_internal.h"
#include "umma.cuh"

namespace ssd {
namespace {

using umma::ex2;

constexpr int SEL_T = 16;             // tokens per tile
constexpr int SEL_C = 8;              // tokens between the states kept for the backward pass

struct SelGeo {
  int B, L, D, N, G, Dg, nb;          // nb = channel blocks per group
  int segs, seg_len;                  // the tokens in `segs` parts of seg_len (a multiple of SEL_T)
  int softplus, nc;                   // nc = states kept per channel and sequence
  int wide;                           // four channels of a row may be moved at once
  int par_row;                        // a block's sums of dA, dD and ddt_bias: D*NP + 2*D floats, up to a multiple of four
  long long xsb, xsl, dtsb, dtsl, bsb, bsl, csb, csl, zsb, zsl, ysb, ysl;
};

// Block shape for LPC lanes per channel with KS states each.  Two roles: the scan (thread = KS states of a channel), and tasks of a
// token and four neighbouring channels, in which everything that a token needs once per channel is loaded, computed and stored.
template <int KS_, int LPC_, int CHB_> struct Sh {
  static constexpr int KS = KS_, LPC = LPC_, CHB = CHB_;
  static constexpr int KP = KS / 2;                  // pairs of states
  static constexpr int NP = KS * LPC;                // states per channel, padded
  static constexpr int TH = CHB * LPC;               // threads
  static constexpr int W = TH / 32;
  static constexpr int CPW = 32 / LPC;               // channels per warp
  static constexpr int QR = CHB / 4;                 // tasks per token
  static constexpr int RS = TH / QR < SEL_T ? TH / QR : SEL_T;   // tokens between a thread's tasks
  static constexpr int IT = SEL_T / RS;              // tasks per thread
  static constexpr int BI = (SEL_T * NP + TH - 1) / TH;          // values of B (and of C) per thread
  static constexpr int COPIES = CPW < KS ? CPW : KS; // backward: orders of the states among a warp's lanes (see ChannelSum)
  static constexpr int BWD_FLOATS = SEL_T * CHB * 9 + 2 * COPIES * SEL_T * NP + W * SEL_T * 2 * NP + 2 * CHB + KS * TH;   // k_sel_bwd's shared memory ..
  template <typename T> static constexpr int bwd_smem() { return BWD_FLOATS * 4 + 3 * IT * TH * 4 * (int)sizeof(T); }    // .. with the raw values of its tasks
};

// softplus(v) = max(v, 0) + log(1 + exp(-|v|))
__device__ __forceinline__ float sel_step(float raw, float bias, int softplus) {
  const float v = raw + bias;
  return softplus ? softplusf_(v) : v;
}
// the same, and its derivative 1 / (1 + exp(-v)) from the same exponential
__device__ __forceinline__ float sel_step_d(float raw, float bias, int softplus, float& d) {
  const float v = raw + bias;
  if (!softplus) { d = 1.f; return v; }
  const float e = exp_neg(v);
  d = __fdividef(v >= 0.f ? 1.f : e, 1.f + e);
  return fmaxf(v, 0.f) + log1p01(e);
}
// relative error (4 + 1.2 |v|) 2^-23 (1e-6 at 5; 3e-6 at -20, where silu is 4e-8)
__device__ __forceinline__ float sig(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }
__device__ __forceinline__ float hsum(f32x2 v) { float a, b; unpack2(v, a, b); return a + b; }
__device__ __forceinline__ f32x2 dup2(float v) { return pack2(v, v); }
__device__ __forceinline__ f32x2 ex2_2(f32x2 v) { float a, b; unpack2(v, a, b); return pack2(ex2(a), ex2(b)); }
// exp(s A) for a pair of decays (A2 = A log2 e).  ex2.approx is 2e-8 low on average over the arguments that decays have (1.7e-8 to
// 2.6e-8 in every interval measured between -0.75 and -0.001; rms 4e-8); a state is a product of hundreds of them, where an offset
// adds up and scatter does not, so the argument is raised by 2e-8 log2 e.  (A step of 0 gives 1 exactly all the same.)
constexpr float DECAY_UP = 2.9e-8f;
__device__ __forceinline__ f32x2 decay2(f32x2 A2, f32x2 s2) { return ex2_2(fma2(A2, s2, pack2(DECAY_UP, DECAY_UP))); }

// The same once more (a value that the compiler does not keep from the first time).
__device__ __forceinline__ f32x2 decay2_again(f32x2 A2, f32x2 s2) {
  float a, b;
  unpack2(fma2(A2, s2, pack2(DECAY_UP, DECAY_UP)), a, b);
  asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
  return pack2(a, b);
}

// Four neighbouring values of a row as they lie in memory.
template <typename T> struct Raw4;
template <> struct Raw4<float> { float4 v; };
template <> struct Raw4<__nv_bfloat16> { uint2 v; };
// n values are there (at least one; where there are fewer than four the last one stands in for the rest)
__device__ __forceinline__ void load4(const float* p, bool wide, int n, Raw4<float>& r) {
  if (wide) r.v = *reinterpret_cast<const float4*>(p);
  else r.v = make_float4(p[0], p[n > 1 ? 1 : 0], p[n > 2 ? 2 : 0], p[n > 3 ? 3 : 0]);
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, bool wide, int n, Raw4<__nv_bfloat16>& r) {
  const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
  if (wide) r.v = *reinterpret_cast<const uint2*>(p);
  else r.v = make_uint2(q[0] | (uint32_t)q[n > 1 ? 1 : 0] << 16, q[n > 2 ? 2 : 0] | (uint32_t)q[n > 3 ? 3 : 0] << 16);
}
__device__ __forceinline__ void zero4(Raw4<float>& r) { r.v = make_float4(0.f, 0.f, 0.f, 0.f); }
__device__ __forceinline__ void zero4(Raw4<__nv_bfloat16>& r) { r.v = make_uint2(0, 0); }
__device__ __forceinline__ void values4(const Raw4<float>& r, float (&v)[4]) { v[0] = r.v.x; v[1] = r.v.y; v[2] = r.v.z; v[3] = r.v.w; }
__device__ __forceinline__ void values4(const Raw4<__nv_bfloat16>& r, float (&v)[4]) {
  v[0] = __uint_as_float(r.v.x << 16); v[1] = __uint_as_float(r.v.x & 0xffff0000u);
  v[2] = __uint_as_float(r.v.y << 16); v[3] = __uint_as_float(r.v.y & 0xffff0000u);
}
__device__ __forceinline__ void put4(float* p, bool wide, int n, const float (&v)[4]) {
  if (wide) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); return; }
#pragma unroll
  for (int i = 0; i < 4; ++i) if (i < n) p[i] = v[i];
}
__device__ __forceinline__ void put4(__nv_bfloat16* p, bool wide, int n, const float (&v)[4]) {
  if (wide) { *reinterpret_cast<uint2*>(p) = make_uint2(umma::pack_bf16(v[0], v[1]), umma::pack_bf16(v[2], v[3])); return; }
#pragma unroll
  for (int i = 0; i < 4; ++i) if (i < n) p[i] = __float2bfloat16_rn(v[i]);
}

struct Place { int b, seg, g, d, n; };               // batch row, part, group, first channel (of all), channels from there on (<= 0: none)
template <class S> __device__ __forceinline__ Place place(const SelGeo& q, int c) {
  const int nblk = q.G * q.nb;
  Place p;
  const int blk = blockIdx.x % nblk, rest = blockIdx.x / nblk;
  p.seg = rest % q.segs; p.b = rest / q.segs;
  p.g = blk / q.nb;
  const int cg = (blk - p.g * q.nb) * S::CHB + c;
  p.n = q.Dg - cg; p.d = p.g * q.Dg + (p.n > 0 ? cg : 0);
  return p;
}

// KS states of a [.., D, N] fp32 array (N not padded) at `p`, in the order (j ^ m).
template <class S> __device__ __forceinline__ void load_state(const float* p, int N, int nl, bool live, int m, f32x2 (&v)[S::KP]) {
  float f[S::KS];
#pragma unroll
  for (int j = 0; j < S::KS; ++j) {
    const int n = nl * S::KS + (j ^ m);
    f[j] = live && p && n < N ? p[n] : 0.f;
  }
#pragma unroll
  for (int k = 0; k < S::KP; ++k) v[k] = pack2(f[2 * k], f[2 * k + 1]);
}
template <class S> __device__ __forceinline__ void store_state(float* p, int N, int nl, bool live, int m, const f32x2 (&v)[S::KP]) {
#pragma unroll
  for (int k = 0; k < S::KP; ++k) {
    float f[2];
    unpack2(v[k], f[0], f[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int n = nl * S::KS + ((2 * k + i) ^ m);
      if (live && n < N) p[n] = f[i];
    }
  }
}
// KS states of a padded array of our own, natural order
template <class S> __device__ __forceinline__ void load_padded(const float* p, f32x2 (&v)[S::KP]) {
#pragma unroll
  for (int k = 0; k < S::KS / 4; ++k) {
    const float4 f = *reinterpret_cast<const float4*>(p + 4 * k);
    v[2 * k] = pack2(f.x, f.y); v[2 * k + 1] = pack2(f.z, f.w);
  }
}
template <class S> __device__ __forceinline__ void store_padded(float* p, const f32x2 (&v)[S::KP]) {
#pragma unroll
  for (int k = 0; k < S::KS / 4; ++k) {
    float4 f;
    unpack2(v[2 * k], f.x, f.y); unpack2(v[2 * k + 1], f.z, f.w);
    *reinterpret_cast<float4*>(p + 4 * k) = f;
  }
}
// natural order -> order (j ^ m), m uniform over nothing: one exchange of halves per bit
template <class S> __device__ __forceinline__ void permute(f32x2 (&v)[S::KP], int m) {
  float f[S::KS];
#pragma unroll
  for (int k = 0; k < S::KP; ++k) unpack2(v[k], f[2 * k], f[2 * k + 1]);
#pragma unroll
  for (int bit = 1; bit < S::KS; bit <<= 1) {
    const bool swap = m & bit;
#pragma unroll
    for (int j = 0; j < S::KS; ++j)
      if (!(j & bit)) {
        const float a = f[j], b = f[j | bit];
        f[j] = swap ? b : a; f[j | bit] = swap ? a : b;
      }
  }
#pragma unroll
  for (int k = 0; k < S::KP; ++k) v[k] = pack2(f[2 * k], f[2 * k + 1]);
}

struct SelFwd {
  const void *x, *dt, *Bm, *Cm, *z;
  const float *A, *D, *bias, *init;
  const int* lengths;
  void* y;
  float *fin, *ckpt;                  // ckpt [B][nc][D][NP]: the state before every SEL_C-th token
  float *segst, *segdt;               // [B][segs][D][NP] states of the parts from zero, [B][segs][D] their summed steps
};

// MODE 0: outputs (and the states kept for the backward); MODE 1: a part's own state from zero and its summed steps.
// Measured at 4 x 2048 x 1536 of 16 states, bf16, gated (events around each launch): 104 us, 82 us the parts' pass; at a quarter of
// the length issue slots are 52 % busy and special functions 50 % (64 % in the parts' pass).  Four blocks to an SM: with more, fewer
// registers, 134 to 146 us.
template <typename T, class S, int MODE>
__global__ void __launch_bounds__(S::TH, S::TH == 128 ? 4 : 1) k_sel_fwd(SelGeo q, SelFwd p) {
  constexpr int KS = S::KS, LPC = S::LPC, KP = S::KP, NP = S::NP, CHB = S::CHB, TH = S::TH, IT = S::IT, BI = S::BI;
  __shared__ __align__(16) float2 s_dt[SEL_T][CHB];  // step, step * x
  __shared__ __align__(16) float s_B[SEL_T][NP], s_C[SEL_T][NP], s_y[SEL_T][CHB];
  pdl_wait();
  const int tid = threadIdx.x, c = tid / LPC, nl = tid % LPC, qc = tid % S::QR * 4, r0 = tid / S::QR;
  const bool tasks = r0 < SEL_T;
  const Place me = place<S>(q, c), it = place<S>(q, qc);
  if (MODE == 1 && me.seg == q.segs - 1) return;
  const bool live = me.n > 0, wide = q.wide;
  const int len = p.lengths ? min(max(p.lengths[me.b], 0), q.L) : q.L;
  const int t_begin = me.seg * q.seg_len, t_end = min(t_begin + q.seg_len, q.L), t_live = min(t_end, len);
  const T* xp = (const T*)p.x + (long long)it.b * q.xsb + it.d;
  const T* dtp = (const T*)p.dt + (long long)it.b * q.dtsb + it.d;
  const T* zp = (const T*)p.z + (long long)it.b * q.zsb + it.d;
  const T* bp = (const T*)p.Bm + (long long)it.b * q.bsb + (long long)it.g * q.N;
  const T* cp = (const T*)p.Cm + (long long)it.b * q.csb + (long long)it.g * q.N;
  T* yp = (T*)p.y + (long long)it.b * q.ysb + it.d;
  const bool want_y = MODE == 0 && p.y, gated = want_y && p.z;
  float bias[4], Dv[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    bias[k] = p.bias && k < it.n ? p.bias[it.d + k] : 0.f;
    Dv[k] = p.D && k < it.n ? p.D[it.d + k] : 0.f;
  }

  f32x2 A[KP], h[KP];
  load_state<S>(p.A + (long long)me.d * q.N, q.N, nl, live, 0, A);
#pragma unroll
  for (int k = 0; k < KP; ++k) { A[k] = mul2(A[k], dup2(LOG2E)); h[k] = 0ull; }
  float dtsum = 0.f;
  if (MODE == 0) {
    load_state<S>(p.init ? p.init + ((long long)me.b * q.D + me.d) * q.N : nullptr, q.N, nl, live, 0, h);
    for (int s = 0; s < me.seg; ++s) {
      const long long at = ((long long)me.b * q.segs + s) * q.D + me.d;
      f32x2 v[KP];
      load_padded<S>(p.segst + at * NP + nl * KS, v);
      const f32x2 d2 = dup2(p.segdt[at]);
#pragma unroll
      for (int k = 0; k < KP; ++k) h[k] = fma2(decay2(A[k], d2), h[k], v[k]);
    }
  }

  Raw4<T> rx[IT], rd[IT], rz[IT];
  T rb[BI], rc[BI];
  auto request = [&](int t0) {                       // values of a tile into registers; nothing past the end is read
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int t = t0 + r0 + i * S::RS;
      zero4(rx[i]); zero4(rd[i]); zero4(rz[i]);
      if (tasks && it.n > 0 && t < t_live) {
        load4(xp + (long long)t * q.xsl, wide, it.n, rx[i]);
        load4(dtp + (long long)t * q.dtsl, wide, it.n, rd[i]);
        if (gated) load4(zp + (long long)t * q.zsl, wide, it.n, rz[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < BI; ++i) {
      const int e = tid + i * TH, n = e % NP, t = t0 + e / NP;
      rb[i] = rc[i] = T(0.f);
      if (n < q.N && t < t_live && e < SEL_T * NP) {
        rb[i] = bp[(long long)t * q.bsl + n];
        if (want_y) rc[i] = cp[(long long)t * q.csl + n];
      }
    }
  };
  request(t_begin);
  for (int t0 = t_begin; t0 < t_end; t0 += SEL_T) {
    float x[IT][4];
    Raw4<T> kz[IT];
    // hand over: step sizes, B and C of this tile
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = r0 + i * S::RS, t = t0 + r;
      float d[4], s[4];
      values4(rx[i], x[i]); values4(rd[i], d);
      kz[i] = rz[i];
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] = t < t_live ? sel_step(d[k], bias[k], q.softplus) : 0.f;
      if (tasks) {
        float4* w = reinterpret_cast<float4*>(&s_dt[r][qc]);
        w[0] = make_float4(s[0], s[0] * x[i][0], s[1], s[1] * x[i][1]);
        w[1] = make_float4(s[2], s[2] * x[i][2], s[3], s[3] * x[i][3]);
      }
    }
#pragma unroll
    for (int i = 0; i < BI; ++i) {
      const int e = tid + i * TH;
      if (e < SEL_T * NP) {
        s_B[e / NP][e % NP] = (float)rb[i];
        if (want_y) s_C[e / NP][e % NP] = (float)rc[i];
      }
    }
    __syncthreads();
    if (t0 + SEL_T < t_end) request(t0 + SEL_T);
    const bool work = t0 < len;
#pragma unroll
    for (int u = 0; u < SEL_T; u += LPC) {
      if (MODE == 0 && u % SEL_C == 0 && p.ckpt && live && t0 + u < t_end)
        store_padded<S>(p.ckpt + (((long long)me.b * q.nc + (t0 + u) / SEL_C) * q.D + me.d) * NP + nl * KS, h);
      if (!work) continue;
      float v[LPC];
#pragma unroll
      for (int i = 0; i < LPC; ++i) {
        const float2 sd = s_dt[u + i][c];
        const f32x2 s2 = dup2(sd.x), x2 = dup2(sd.y);
        f32x2 acc = 0ull;
#pragma unroll
        for (int k = 0; k < KP; k += 2) {
          const float4 b4 = *reinterpret_cast<const float4*>(&s_B[u + i][nl * KS + 2 * k]);
          h[k] = fma2(decay2(A[k], s2), h[k], mul2(pack2(b4.x, b4.y), x2));
          h[k + 1] = fma2(decay2(A[k + 1], s2), h[k + 1], mul2(pack2(b4.z, b4.w), x2));
          if (MODE == 0) {
            const float4 c4 = *reinterpret_cast<const float4*>(&s_C[u + i][nl * KS + 2 * k]);
            acc = k ? fma2(pack2(c4.x, c4.y), h[k], acc) : mul2(pack2(c4.x, c4.y), h[k]);
            acc = fma2(pack2(c4.z, c4.w), h[k + 1], acc);
          }
        }
        if (MODE == 1) dtsum += sd.x;
        v[i] = hsum(acc);
      }
      if (want_y) {
        int k;
        const float sum = fold_rows<LPC, LPC>(v, nl, k);
        s_y[u + k][c] = sum;
      }
    }
    __syncthreads();
    if (want_y && tasks && it.n > 0) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int r = r0 + i * S::RS, t = t0 + r;
        if (t >= t_end) continue;
        float o[4] = {0.f, 0.f, 0.f, 0.f};
        if (t < len) {
          const float4 y4 = *reinterpret_cast<const float4*>(&s_y[r][qc]);
          o[0] = fmaf(Dv[0], x[i][0], y4.x); o[1] = fmaf(Dv[1], x[i][1], y4.y);
          o[2] = fmaf(Dv[2], x[i][2], y4.z); o[3] = fmaf(Dv[3], x[i][3], y4.w);
          if (gated) {
            float z[4];
            values4(kz[i], z);
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] *= z[k] * sig(z[k]);
          }
        }
        put4(yp + (long long)t * q.ysl, wide, it.n, o);
      }
    }
  }
  if (MODE == 1) {
    const long long at = ((long long)me.b * q.segs + me.seg) * q.D + me.d;
    if (live) {
      store_padded<S>(p.segst + at * NP + nl * KS, h);
      if (nl == 0) p.segdt[at] = dtsum;
    }
  } else if (p.fin && me.seg == q.segs - 1) {
    store_state<S>(p.fin + ((long long)me.b * q.D + me.d) * q.N, q.N, nl, live, 0, h);
  }
}

// ---------------------------------------------------------------------------------------------
// Backward, with g_t = dL/dh_t = C_t dy'_t + a_{t+1} g_{t+1} and dy' = dy silu(z):
//     dB_t = sum_d g_t s x,   dC_t = sum_d dy' h_t,   dx = s (g.B) + D dy',   ds = x (g.B) + sum_n g_t a_t h_{t-1} A,
//     dA = sum_t g_t a_t h_{t-1} s.
// Eight tokens at a time the states and decays are computed again from the state kept before them and stay in registers (an
// exponential is computed once here, as in the forward), then the eight are walked backwards.  Sums over the states go over the lanes
// of a channel, sums over the channels over the lanes and warps of a block; blocks leave partial sums of dB and dC which a second
// kernel adds in order.
struct SelBwd {
  const void *x, *dt, *Bm, *Cm, *z, *dy;
  const float *A, *D, *bias, *dfin, *ckpt;
  const int* lengths;
  void *dx, *ddt, *dz;
  float *dinit, *part_bc, *part_par;  // [G*nb][B*L][2*NP]; [B*segs][par_row]
  float *segst, *segdt;               // [B][segs][D][NP]: gradient that a part passes to the state before it, with nothing coming in
};

// A part's own gradient of the state before it, from zero.
template <typename T, class S>
__global__ void __launch_bounds__(S::TH) k_sel_bwd_part(SelGeo q, SelBwd p) {
  constexpr int KS = S::KS, LPC = S::LPC, KP = S::KP, NP = S::NP, CHB = S::CHB, TH = S::TH, IT = S::IT, BI = S::BI;
  __shared__ __align__(16) float2 s_dt[SEL_T][CHB];  // step, dy'
  __shared__ __align__(16) float s_C[SEL_T][NP];
  pdl_wait();
  const int tid = threadIdx.x, c = tid / LPC, nl = tid % LPC, qc = tid % S::QR * 4, r0 = tid / S::QR;
  const bool tasks = r0 < SEL_T;
  const Place me = place<S>(q, c), it = place<S>(q, qc);
  if (me.seg == 0) return;
  const bool live = me.n > 0, wide = q.wide;
  const int len = p.lengths ? min(max(p.lengths[me.b], 0), q.L) : q.L;
  const int t_begin = me.seg * q.seg_len, t_end = min(t_begin + q.seg_len, q.L), t_live = min(t_end, len);
  const T* dtp = (const T*)p.dt + (long long)it.b * q.dtsb + it.d;
  const T* zp = (const T*)p.z + (long long)it.b * q.zsb + it.d;
  const T* dyp = (const T*)p.dy + (long long)it.b * q.ysb + it.d;
  const T* cp = (const T*)p.Cm + (long long)it.b * q.csb + (long long)it.g * q.N;
  float bias[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) bias[k] = p.bias && k < it.n ? p.bias[it.d + k] : 0.f;
  f32x2 A[KP], g[KP];
  load_state<S>(p.A + (long long)me.d * q.N, q.N, nl, live, 0, A);
#pragma unroll
  for (int k = 0; k < KP; ++k) { A[k] = mul2(A[k], dup2(LOG2E)); g[k] = 0ull; }
  float dtsum = 0.f;
  Raw4<T> rd[IT], ry[IT], rz[IT];
  T rc[BI];
  auto request = [&](int t0) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int t = t0 + r0 + i * S::RS;
      zero4(rd[i]); zero4(ry[i]); zero4(rz[i]);
      if (tasks && it.n > 0 && t < t_live) {
        load4(dtp + (long long)t * q.dtsl, wide, it.n, rd[i]);
        load4(dyp + (long long)t * q.ysl, wide, it.n, ry[i]);
        if (p.z) load4(zp + (long long)t * q.zsl, wide, it.n, rz[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < BI; ++i) {
      const int e = tid + i * TH, n = e % NP, t = t0 + e / NP;
      rc[i] = T(0.f);
      if (n < q.N && t < t_live && e < SEL_T * NP) rc[i] = cp[(long long)t * q.csl + n];
    }
  };
  const int t_last = t_begin + (t_end - t_begin - 1) / SEL_T * SEL_T;
  request(t_last);
  for (int t0 = t_last; t0 >= t_begin; t0 -= SEL_T) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = r0 + i * S::RS, t = t0 + r;
      float d[4], y[4], z[4];
      values4(rd[i], d); values4(ry[i], y); values4(rz[i], z);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        d[k] = t < t_live ? sel_step(d[k], bias[k], q.softplus) : 0.f;
        if (p.z) y[k] *= z[k] * sig(z[k]);
      }
      if (tasks) {
        float4* w = reinterpret_cast<float4*>(&s_dt[r][qc]);
        w[0] = make_float4(d[0], y[0], d[1], y[1]);
        w[1] = make_float4(d[2], y[2], d[3], y[3]);
      }
    }
#pragma unroll
    for (int i = 0; i < BI; ++i) {
      const int e = tid + i * TH;
      if (e < SEL_T * NP) s_C[e / NP][e % NP] = (float)rc[i];
    }
    __syncthreads();
    if (t0 > t_begin) request(t0 - SEL_T);
    if (t0 < len) {
#pragma unroll
      for (int r = SEL_T - 1; r >= 0; --r) {
        const float2 sd = s_dt[r][c];
        const f32x2 s2 = dup2(sd.x), y2 = dup2(sd.y);
#pragma unroll
        for (int k = 0; k < KP; k += 2) {
          const float4 c4 = *reinterpret_cast<const float4*>(&s_C[r][nl * KS + 2 * k]);
          g[k] = mul2(decay2(A[k], s2), fma2(pack2(c4.x, c4.y), y2, g[k]));
          g[k + 1] = mul2(decay2(A[k + 1], s2), fma2(pack2(c4.z, c4.w), y2, g[k + 1]));
        }
        dtsum += sd.x;
      }
    }
    __syncthreads();
  }
  const long long at = ((long long)me.b * q.segs + me.seg) * q.D + me.d;
  if (live) {
    store_padded<S>(p.segst + at * NP + nl * KS, g);
    if (nl == 0) p.segdt[at] = dtsum;
  }
}

// Sums over the channels of a warp (lane = channel * LPC + nl) of a token's contributions to dB and dC, KS states each.  Every
// exchange folds two values into one: the lanes of a pair keep one half of the states each and give the other.  Which half a lane
// keeps follows from a bit of its channel; its registers hold the states in the order (j ^ m), m the lane's bits, so that the half to
// keep is the same registers in every lane and no selects are needed (they were a quarter of the backward's instructions).
// A lane ends up with V values: state v ^ m of dB and of dC, or, with one value, that of `kind`.
template <class S> struct ChannelSum {
  static constexpr int CPW = S::CPW, KS = S::KS;
  static constexpr int V = CPW >= KS ? 1 : KS / CPW;             // states left per kind
  static constexpr bool ONE = CPW >= 2 * KS;                     // and one kind
  __device__ static __forceinline__ int order(int lane) {        // m
    int m = 0, o = 16;
#pragma unroll
    for (int h = KS / 2; h > 0 && o >= S::LPC; h >>= 1, o >>= 1) if (lane & o) m |= h;
    return m;
  }
  // b, c: the 2 KS values; afterwards b[0..V-1], c[0..V-1] (ONE: b[0], kind returned)
  __device__ static __forceinline__ int run(float (&b)[KS], float (&c)[KS], int lane) {
    int o = 16;
#pragma unroll
    for (int h = KS / 2; h > 0 && o >= S::LPC; h >>= 1, o >>= 1) {
#pragma unroll
      for (int j = 0; j < h; ++j) {
        b[j] += __shfl_xor_sync(0xffffffffu, b[j + h], o);
        c[j] += __shfl_xor_sync(0xffffffffu, c[j + h], o);
      }
    }
    int kind = 0;
    if (ONE) {
      const bool up = lane & o;
      const float keep = up ? c[0] : b[0], give = up ? b[0] : c[0];
      b[0] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      kind = up;
#pragma unroll
      for (o >>= 1; o >= S::LPC; o >>= 1) b[0] += __shfl_xor_sync(0xffffffffu, b[0], o);
    }
    return kind;
  }
};

// Four blocks to an SM, so 128 registers, with 56 bytes of spills for 16 states in bf16, gated (12 to 84 for the other shapes of 128 threads).
// 4 x 2048 x 1536 of 16 states, bf16, gated: 322 us; three blocks 360; when it took 343, five spilled more and took 418.  From 33 states on
// the shared memory leaves room for two blocks, and the bound costs 320 to 588 bytes of spills for nothing (fp32 of 8 states: for three).  Keeping eight tokens' decays beside their states took 383 where recomputing them took 358, eight states a thread 424 to 491.
// At a quarter of the length: issue slots 52 % busy, the shared-memory path 63 %, special functions 31 %.
template <typename T, class S, bool GATED>
__global__ void __launch_bounds__(S::TH, S::TH == 128 ? 4 : 1) k_sel_bwd(SelGeo q, SelBwd p) {
  constexpr int KS = S::KS, LPC = S::LPC, KP = S::KP, NP = S::NP, CHB = S::CHB, TH = S::TH, IT = S::IT, BI = S::BI, W = S::W, CO = S::COPIES;
  extern __shared__ __align__(16) float sel_smem[];                   // (registers are short here: what a tile needs once lies in it)
  float2 (*s_a)[CHB] = reinterpret_cast<float2 (*)[CHB]>(sel_smem);    // step, step * x
  float (*s_y)[CHB] = reinterpret_cast<float (*)[CHB]>(sel_smem + 2 * SEL_T * CHB);               // dy'
  float (*s_ds)[CHB] = s_y + SEL_T;                                    // d step / d raw
  float (*s_1)[CHB] = s_ds + SEL_T, (*s_2)[CHB] = s_1 + SEL_T, (*s_3)[CHB] = s_2 + SEL_T;         // g.B, sum of g a h A, C.h
  float (*s_dD)[CHB] = s_3 + SEL_T, (*s_db)[CHB] = s_dD + SEL_T, *s_bias = s_db[SEL_T], *s_D = s_bias + CHB;
  float (*s_B)[SEL_T][NP] = reinterpret_cast<float (*)[SEL_T][NP]>(s_D + CHB);                    // [order][token][states]
  float (*s_C)[SEL_T][NP] = s_B + CO;
  float (*s_bc)[SEL_T][2 * NP] = reinterpret_cast<float (*)[SEL_T][2 * NP]>(s_C + CO);            // [warp][token][dB | dC]
  float4* s_dA = reinterpret_cast<float4*>(s_bc + W);                  // [KS / 4][thread]
  Raw4<T>* s_raw = reinterpret_cast<Raw4<T>*>(s_dA + KS / 4 * TH);     // [x, dy, z][task][thread]
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = tid / LPC, nl = tid % LPC, qc = tid % S::QR * 4, r0 = tid / S::QR;
  const bool tasks = r0 < SEL_T;
  const Place me = place<S>(q, c), it = place<S>(q, qc);
  const bool live = me.n > 0, wide = q.wide;
  const int len = p.lengths ? min(max(p.lengths[me.b], 0), q.L) : q.L;
  const int t_begin = me.seg * q.seg_len, t_end = min(t_begin + q.seg_len, q.L), t_live = min(t_end, len);
  const T* xp = (const T*)p.x + (long long)it.b * q.xsb + it.d;
  const T* dtp = (const T*)p.dt + (long long)it.b * q.dtsb + it.d;
  const T* zp = (const T*)p.z + (long long)it.b * q.zsb + it.d;
  const T* dyp = (const T*)p.dy + (long long)it.b * q.ysb + it.d;
  const T* bp = (const T*)p.Bm + (long long)it.b * q.bsb + (long long)it.g * q.N;
  const T* cp = (const T*)p.Cm + (long long)it.b * q.csb + (long long)it.g * q.N;
  const long long out0 = (long long)it.b * q.L * q.D + it.d;
  float* bc0 = p.part_bc + ((long long)(blockIdx.x % (q.G * q.nb)) * q.B + me.b) * q.L * (2 * NP);
  for (int e = tid; e < CHB; e += TH) {
    const Place at = place<S>(q, e);
    s_bias[e] = p.bias && at.n > 0 ? p.bias[at.d] : 0.f;
    s_D[e] = p.D && at.n > 0 ? p.D[at.d] : 0.f;
  }
  if (tasks)
#pragma unroll
    for (int k = 0; k < 4; ++k) s_dD[r0][qc + k] = s_db[r0][qc + k] = 0.f;
  __syncthreads();
  const int m = ChannelSum<S>::order(lane);

  f32x2 A[KP], g[KP];                                // g: a_{t+1} g_{t+1}
  load_state<S>(p.A + (long long)me.d * q.N, q.N, nl, live, m, A);
  load_state<S>(p.dfin ? p.dfin + ((long long)me.b * q.D + me.d) * q.N : nullptr, q.N, nl, live, m, g);
#pragma unroll
  for (int k = 0; k < KP; ++k) A[k] = mul2(A[k], dup2(LOG2E));
#pragma unroll
  for (int k = 0; k < KS / 4; ++k) s_dA[k * TH + tid] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = q.segs - 1; s > me.seg; --s) {
    const long long at = ((long long)me.b * q.segs + s) * q.D + me.d;
    f32x2 v[KP];
    load_padded<S>(p.segst + at * NP + nl * KS, v);
    permute<S>(v, m);
    const f32x2 d2 = dup2(p.segdt[at]);
#pragma unroll
    for (int k = 0; k < KP; ++k) g[k] = fma2(decay2(A[k], d2), g[k], v[k]);
  }

  Raw4<T> rx[IT], rd[IT], ry[IT], rz[IT];
  T rb[BI], rc[BI];
  // Values of a tile into registers, for a tile that has tokens.  Every address is one that may be read (a row past the end becomes
  // the last one before it) and nothing is chosen among before the values are used: a select would wait for the load (4 x 2048 x 1536:
  // 343 us with loads under a condition, 321 so; in the forward the clamping costs more than it gives, 104 against 121).
  const int have = max(it.n, 1);
  auto request = [&](int t0) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const long long t = min(t0 + r0 + i * S::RS, t_live - 1);
      load4(xp + t * q.xsl, wide, have, rx[i]);
      load4(dtp + t * q.dtsl, wide, have, rd[i]);
      load4(dyp + t * q.ysl, wide, have, ry[i]);
      if (GATED) load4(zp + t * q.zsl, wide, have, rz[i]);
    }
#pragma unroll
    for (int i = 0; i < BI; ++i) {
      const int e = tid + i * TH, n = min(e % NP, q.N - 1);
      const long long t = min(t0 + e / NP, t_live - 1);
      rb[i] = bp[t * q.bsl + n];
      rc[i] = cp[t * q.csl + n];
    }
  };
  // the state before token t (of channels and tokens that are not there: of others; nothing comes of it)
  const float* ck0 = p.ckpt + ((long long)me.b * q.nc * q.D + me.d) * NP + nl * KS;
  auto kept = [&](int t, f32x2 (&v)[KP]) { load_padded<S>(ck0 + (long long)min(t / SEL_C, q.nc - 1) * q.D * NP, v); };
  const int t_last = t_begin + (t_end - t_begin - 1) / SEL_T * SEL_T;
  if (t_last < t_live) request(t_last);
  f32x2 first[KP];                                   // the state before the next eight tokens to be walked
  kept(t_last + SEL_C, first);
  for (int t0 = t_last; t0 >= t_begin; t0 -= SEL_T) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = r0 + i * S::RS, t = t0 + r;
      float x[4], d[4], y[4], z[4], s[4], ds[4];
      s_raw[(0 * IT + i) * TH + tid] = rx[i]; s_raw[(1 * IT + i) * TH + tid] = ry[i];
      if (GATED) s_raw[(2 * IT + i) * TH + tid] = rz[i];
      values4(rx[i], x); values4(rd[i], d); values4(ry[i], y); values4(rz[i], z);
      const float4 b4 = *reinterpret_cast<const float4*>(s_bias + qc);
      const float bias[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s[k] = ds[k] = 0.f;
        const bool ok = t < t_live && k < it.n;
        if (ok) s[k] = sel_step_d(d[k], bias[k], q.softplus, ds[k]);
        if (GATED) y[k] *= z[k] * sig(z[k]);
        y[k] = ok ? y[k] : 0.f;
        x[k] = ok ? x[k] : 0.f;
      }
      if (tasks) {
        float4* w = reinterpret_cast<float4*>(&s_a[r][qc]);
        w[0] = make_float4(s[0], s[0] * x[0], s[1], s[1] * x[1]);
        w[1] = make_float4(s[2], s[2] * x[2], s[3], s[3] * x[3]);
        *reinterpret_cast<float4*>(&s_y[r][qc]) = make_float4(y[0], y[1], y[2], y[3]);
        *reinterpret_cast<float4*>(&s_ds[r][qc]) = make_float4(ds[0], ds[1], ds[2], ds[3]);
      }
    }
#pragma unroll
    for (int i = 0; i < BI; ++i) {
      const int e = tid + i * TH;
      if (e < SEL_T * NP) {
        const int r = e / NP, n = e % NP;
        const bool ok = n < q.N && t0 + r < t_live;
        const float fb = ok ? (float)rb[i] : 0.f, fc = ok ? (float)rc[i] : 0.f;
#pragma unroll
        for (int o = 0; o < CO; ++o) { const int oo = o * (KS / CO); s_B[o][r][n ^ oo] = fb; s_C[o][r][n ^ oo] = fc; }
      }
    }
    f32x2 tA[KP] = {};                               // a tile's share of dA: sums of 16, then sums of tiles
    __syncthreads();
    if (t0 > t_begin && t0 - SEL_T < t_live) request(t0 - SEL_T);
    if (t0 >= len) {
      if (t0 > t_begin) kept(t0 - SEL_C, first);
    } else {
      const int co = m / (KS / CO);
#pragma unroll 1
      for (int half = 1; half >= 0; --half) {
        f32x2 h[SEL_C + 1][KP];
        permute<S>(first, m);
#pragma unroll
        for (int k = 0; k < KP; ++k) h[0][k] = first[k];
        if (half) kept(t0, first);
        else if (t0 > t_begin) kept(t0 - SEL_C, first);
#pragma unroll
        for (int i = 0; i < SEL_C; ++i) {
          const int r = half * SEL_C + i;
          const float2 v = s_a[r][c];
          const f32x2 s2 = dup2(v.x), x2 = dup2(v.y);
#pragma unroll
          for (int k = 0; k < KP; k += 2) {
            const float4 b4 = *reinterpret_cast<const float4*>(&s_B[co][r][nl * KS + 2 * k]);
            h[i + 1][k] = fma2(decay2(A[k], s2), h[i][k], mul2(pack2(b4.x, b4.y), x2));
            h[i + 1][k + 1] = fma2(decay2(A[k + 1], s2), h[i][k + 1], mul2(pack2(b4.z, b4.w), x2));
          }
        }
        constexpr int FR = LPC < SEL_C ? LPC : SEL_C;  // tokens whose sums over the states are folded together
#pragma unroll
        for (int u = SEL_C - FR; u >= 0; u -= FR) {
          float v1[FR], v2[FR], v3[FR];
#pragma unroll
          for (int f = FR - 1; f >= 0; --f) {
            const int i = u + f, r = half * SEL_C + i;
            const float2 v = s_a[r][c];
            const f32x2 s2 = dup2(v.x), x2 = dup2(v.y), y2 = dup2(s_y[r][c]);
            f32x2 a1 = 0ull, a2 = 0ull, a3 = 0ull;
            float wb[KS], wc[KS];
#pragma unroll
            for (int k2 = 0; k2 < KP; k2 += 2) {
              const float4 b4 = *reinterpret_cast<const float4*>(&s_B[co][r][nl * KS + 2 * k2]);
              const float4 c4 = *reinterpret_cast<const float4*>(&s_C[co][r][nl * KS + 2 * k2]);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int k = k2 + e;
                const f32x2 Bk = e ? pack2(b4.z, b4.w) : pack2(b4.x, b4.y), Ck = e ? pack2(c4.z, c4.w) : pack2(c4.x, c4.y);
                g[k] = fma2(Ck, y2, g[k]);
                unpack2(mul2(g[k], x2), wb[2 * k], wb[2 * k + 1]);
                unpack2(mul2(h[i + 1][k], y2), wc[2 * k], wc[2 * k + 1]);
                a1 = k ? fma2(Bk, g[k], a1) : mul2(Bk, g[k]);
                if (GATED) a3 = k ? fma2(Ck, h[i + 1][k], a3) : mul2(Ck, h[i + 1][k]);
                g[k] = mul2(g[k], decay2_again(A[k], s2));
                const f32x2 qk = mul2(g[k], h[i][k]);
                a2 = k ? fma2(A[k], qk, a2) : mul2(A[k], qk);
                tA[k] = fma2(qk, s2, tA[k]);
              }
            }
            v1[f] = hsum(a1); v2[f] = hsum(a2);
            if (GATED) v3[f] = hsum(a3);
            typedef ChannelSum<S> CS;
            const int kind = CS::run(wb, wc, lane);
            float* o = &s_bc[warp][r][nl * KS];
            if (CS::ONE) o[kind * NP + m] = wb[0];
            else
#pragma unroll
              for (int j = 0; j < CS::V; ++j) { o[j ^ m] = wb[j]; o[NP + (j ^ m)] = wc[j]; }
          }
          int k;
          const float f1 = fold_rows<LPC, FR>(v1, nl, k);
          const int r = half * SEL_C + u + k;
          s_1[r][c] = f1;
          s_2[r][c] = fold_rows<LPC, FR>(v2, nl, k);
          if (GATED) s_3[r][c] = fold_rows<LPC, FR>(v3, nl, k);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < KS / 4; ++k) {
      const float4 f = s_dA[k * TH + tid];
      float t[4];
      unpack2(tA[2 * k], t[0], t[1]); unpack2(tA[2 * k + 1], t[2], t[3]);
      s_dA[k * TH + tid] = make_float4(f.x + t[0], f.y + t[1], f.z + t[2], f.w + t[3]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = r0 + i * S::RS, t = t0 + r;
      if (!tasks || it.n <= 0 || t >= t_end) continue;
      float dx[4] = {}, dd[4] = {}, dz[4] = {};
      if (t < len) {
        float x[4], y[4], z[4];
        values4(s_raw[(0 * IT + i) * TH + tid], x); values4(s_raw[(1 * IT + i) * TH + tid], y);
        if (GATED) values4(s_raw[(2 * IT + i) * TH + tid], z);
        const float4 y4 = *reinterpret_cast<const float4*>(&s_y[r][qc]), ds4 = *reinterpret_cast<const float4*>(&s_ds[r][qc]);
        const float dy0[4] = {y4.x, y4.y, y4.z, y4.w}, ds[4] = {ds4.x, ds4.y, ds4.z, ds4.w};
        const float4 f1 = *reinterpret_cast<const float4*>(&s_1[r][qc]), f2 = *reinterpret_cast<const float4*>(&s_2[r][qc]);
        const float4 f3 = GATED ? *reinterpret_cast<const float4*>(&s_3[r][qc]) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float4 D4 = *reinterpret_cast<const float4*>(s_D + qc);
        float4 aD = *reinterpret_cast<const float4*>(&s_dD[r0][qc]), ab = *reinterpret_cast<const float4*>(&s_db[r0][qc]);
        float dD[4] = {aD.x, aD.y, aD.z, aD.w}, dbias[4] = {ab.x, ab.y, ab.z, ab.w};
        const float Dv[4] = {D4.x, D4.y, D4.z, D4.w}, gB[4] = {f1.x, f1.y, f1.z, f1.w}, qA[4] = {f2.x, f2.y, f2.z, f2.w}, hC[4] = {f3.x, f3.y, f3.z, f3.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (GATED) {
            const float sg = sig(z[k]);
            dz[k] = y[k] * fmaf(Dv[k], x[k], hC[k]) * sg * fmaf(z[k], 1.f - sg, 1.f);
          }
          dx[k] = fmaf(s_a[r][qc + k].x, gB[k], Dv[k] * dy0[k]);
          dd[k] = fmaf(x[k], gB[k], qA[k] * LN2) * ds[k];
          dD[k] = fmaf(dy0[k], x[k], dD[k]);
          dbias[k] += dd[k];
        }
        *reinterpret_cast<float4*>(&s_dD[r0][qc]) = make_float4(dD[0], dD[1], dD[2], dD[3]);
        *reinterpret_cast<float4*>(&s_db[r0][qc]) = make_float4(dbias[0], dbias[1], dbias[2], dbias[3]);
      }
      const long long o = out0 + (long long)t * q.D;
      put4((T*)p.dx + o, wide, it.n, dx); put4((T*)p.ddt + o, wide, it.n, dd);
      if (GATED) put4((T*)p.dz + o, wide, it.n, dz);
    }
    for (int e = tid; e < SEL_T * 2 * NP / 4; e += TH) {
      const int r = e / (NP / 2), n = e % (NP / 2) * 4, t = t0 + r;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (t < len)
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float4 f = *reinterpret_cast<const float4*>(&s_bc[w][r][n]);
          v.x += f.x; v.y += f.y; v.z += f.z; v.w += f.w;
        }
      if (t < t_end) *reinterpret_cast<float4*>(bc0 + (long long)t * (2 * NP) + n) = v;
    }
    __syncthreads();
  }
  if (p.dinit && me.seg == 0) store_state<S>(p.dinit + ((long long)me.b * q.D + me.d) * q.N, q.N, nl, live, m, g);
  float* par = p.part_par + ((long long)me.b * q.segs + me.seg) * q.par_row;
  f32x2 dA[KP];
#pragma unroll
  for (int k = 0; k < KS / 4; ++k) {
    const float4 f = s_dA[k * TH + tid];
    dA[2 * k] = pack2(f.x, f.y); dA[2 * k + 1] = pack2(f.z, f.w);
  }
  permute<S>(dA, m);                                 // (its own inverse)
  if (live) store_padded<S>(par + (long long)me.d * NP + nl * KS, dA);
  __syncthreads();                                   // the threads of four channels, in order
  for (int e = tid; e < CHB; e += TH) {
    const Place at = place<S>(q, e);
    if (at.n <= 0) continue;
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int r = 0; r < S::RS; ++r) { a += s_dD[r][e]; b += s_db[r][e]; }
    par[(long long)q.D * NP + at.d] = a;
    par[(long long)q.D * (NP + 1) + at.d] = b;
  }
}

// dB, dC of a token and group: the channel blocks' shares.  64 times four values to a block; four threads take every fourth share each,
// and their sums are added in order.
template <typename T>
__global__ void __launch_bounds__(256) k_sel_sum_bc(SelGeo q, int NP, const float* __restrict__ part, T* __restrict__ dB, T* __restrict__ dC) {
  __shared__ float4 sum[3][64];
  pdl_wait();
  const int V = NP / 2, lane = threadIdx.x & 63, r = threadIdx.x >> 6;   // V fours per token: dB, then dC
  const long long BL = (long long)q.B * q.L, n = BL * V, i = (long long)blockIdx.x * 64 + lane;
  const int g = blockIdx.y;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (i < n) {
    const float4* p = reinterpret_cast<const float4*>(part) + (long long)g * q.nb * n + i;
#pragma unroll 8
    for (int j = r; j < q.nb; j += 4) {
      const float4 f = __ldg(p + j * n);
      a.x += f.x; a.y += f.y; a.z += f.z; a.w += f.w;
    }
  }
  if (r) sum[r - 1][lane] = a;
  __syncthreads();
  if (r || i >= n) return;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const float4 f = sum[k][lane];
    a.x += f.x; a.y += f.y; a.z += f.z; a.w += f.w;
  }
  const long long bl = i / V;
  const int v = (int)(i - bl * V) * 4, s = v % NP;
  T* o = (v < NP ? dB : dC) + (bl * q.G + g) * q.N + s;
  const float f[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) if (s + k < q.N) stf(o + k, f[k]);
}

// dA, dD, ddt_bias: the batch rows' (and parts') shares; eight threads per value, in a fixed order.
__global__ void __launch_bounds__(256) k_sel_sum_par(SelGeo q, int NP, const float* __restrict__ part, float* __restrict__ dA,
                                                     float* __restrict__ dD, float* __restrict__ dbias) {
  __shared__ float s[8][32];
  pdl_wait();
  const long long i = (long long)blockIdx.x * 32 + threadIdx.x, row = (long long)q.D * (NP + 2);
  const int rows = q.B * q.segs;
  float a = 0.f;
  if (i < row)
    for (int r = threadIdx.y; r < rows; r += 8) a += part[(long long)r * q.par_row + i];
  s[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.y || i >= row) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) a += s[k][threadIdx.x];
  if (i < (long long)q.D * NP) {
    const int n = (int)(i % NP);
    if (n < q.N) dA[i / NP * q.N + n] = a;
  } else if (i < (long long)q.D * (NP + 1)) {
    if (dD) dD[i - (long long)q.D * NP] = a;
  } else if (dbias) {
    dbias[i - (long long)q.D * (NP + 1)] = a;
  }
}

// ---------------------------------------------------------------------------------------------
// One step over many streams, in place on the state: the state is read and written once, everything else is small beside it.
// 8192 streams of 256 x 16: 58 us, 4.8 TB/s, issue slots 62 % busy.
// Four states per thread, dstate / 4 lanes per channel; a thread takes U streams `groups` apart, whose states it asks for together, and
// reads what belongs to the channel once.
struct SelStep {
  int S, D, N, G, Dg, softplus, groups, nx;          // nx = blocks of 256 threads over the channels' lanes
  long long xs, dts, bs, cs, zs, ys;
};
template <typename T, int LPC, bool VEC, int U>
__global__ void __launch_bounds__(256) k_sel_step(SelStep q, SsdStepPtrs p) {
  pdl_wait();
  const int s0 = blockIdx.x / q.nx, unit = (blockIdx.x - s0 * q.nx) * 256 + threadIdx.x;
  const bool live = unit / LPC < q.D;
  const int d = live ? unit / LPC : q.D - 1, nl = unit % LPC, n0 = nl * 4, g = d / q.Dg;
  // everything that the U streams need is asked for before any of it is used (a stream past the last reads the first one's)
  float h[U][4];
  T rx[U], rd[U], rz[U];
  Raw4<T> rb[U], rc[U];
  const int have = min(q.N - n0, 4);                 // states of this thread that are there
  const long long at = (long long)g * q.N + (have > 0 ? n0 : 0);
  float* const hp = p.state + ((long long)s0 * q.D + d) * q.N + n0;
  const T *xp = (const T*)p.x + s0 * q.xs + d, *dtp = (const T*)p.dt + s0 * q.dts + d, *zp = (const T*)p.z + s0 * q.zs + d;
  const T *bp = (const T*)p.Bm + s0 * q.bs + at, *cp = (const T*)p.Cm + s0 * q.cs + at;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long k = s0 + u * q.groups < q.S ? (long long)u * q.groups : 0;
    const float* hu = hp + k * q.D * q.N;
    if (VEC) {
      const float4 v = *reinterpret_cast<const float4*>(hu);
      h[u][0] = v.x; h[u][1] = v.y; h[u][2] = v.z; h[u][3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) h[u][j] = j < have ? hu[j] : 0.f;
    }
    rx[u] = xp[k * q.xs];
    rd[u] = dtp[k * q.dts];
    if (p.z) rz[u] = zp[k * q.zs];
    load4(bp + k * q.bs, VEC, have > 0 ? have : 1, rb[u]);
    load4(cp + k * q.cs, VEC, have > 0 ? have : 1, rc[u]);
  }
  float a[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) a[j] = j < have ? __ldg(p.A + (long long)d * q.N + n0 + j) * LOG2E : 0.f;
  const float bias = p.dt_bias ? __ldg(p.dt_bias + d) : 0.f, Dv = p.D ? __ldg(p.D + d) : 0.f;
  // a channel's lanes share out the softplus of its streams
  float step[U];
  if (U > 1 && LPC >= U) {
    float mine = (float)rd[0];
#pragma unroll
    for (int u = 1; u < U; ++u) mine = nl % U == u ? (float)rd[u] : mine;
    mine = sel_step(mine, bias, q.softplus);
#pragma unroll
    for (int u = 0; u < U; ++u) step[u] = __shfl_sync(0xffffffffu, mine, u, LPC);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) step[u] = sel_step((float)rd[u], bias, q.softplus);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool mine = live && s0 + u * q.groups < q.S;
    float b[4], c[4], y = 0.f;
    values4(rb[u], b); values4(rc[u], c);
    const float x = (float)rx[u], sx = step[u] * x;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!VEC && j >= have) b[j] = c[j] = 0.f;
      h[u][j] = fmaf(ex2(fmaf(step[u], a[j], DECAY_UP)), h[u][j], sx * b[j]);
      y = fmaf(c[j], h[u][j], y);
    }
    if (mine) {
      float* hu = hp + (long long)u * q.groups * q.D * q.N;
      if (VEC) *reinterpret_cast<float4*>(hu) = make_float4(h[u][0], h[u][1], h[u][2], h[u][3]);
      else
#pragma unroll
        for (int j = 0; j < 4; ++j) if (j < have) hu[j] = h[u][j];
    }
#pragma unroll
    for (int o = LPC / 2; o; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (mine && nl == 0) {
      y = fmaf(Dv, x, y);
      if (p.z) { const float z = (float)rz[u]; y *= z * sig(z); }
      stf((T*)p.y + (s0 + (long long)u * q.groups) * q.ys + d, y);
    }
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------
// Block shapes by the number of states (padded to 4, 8, 16, 32, 64): eight states per thread where there are as many, since what a
// thread does per token and channel, the sums over lanes and the reads of B and C, is shared by its states.
typedef Sh<4, 1, 64> Sh4;
typedef Sh<8, 1, 64> Sh8;
typedef Sh<8, 2, 64> Sh16;
typedef Sh<8, 4, 32> Sh32;
typedef Sh<8, 8, 16> Sh64;
typedef Sh<4, 1, 64> Bh4;
typedef Sh<4, 2, 64> Bh8;
typedef Sh<4, 4, 32> Bh16;
typedef Sh<4, 8, 16> Bh32;
typedef Sh<8, 8, 16> Bh64;
int block_channels_bwd(int NP) { return NP == 4 ? Bh4::CHB : NP == 8 ? Bh8::CHB : NP == 16 ? Bh16::CHB : NP == 32 ? Bh32::CHB : Bh64::CHB; }
int padded_states(int N) { return N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }
int block_channels(int NP) { return NP <= 16 ? 64 : NP == 32 ? 32 : 16; }
int lanes_for(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }   // single step: four states per thread
size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

int check_common(const char* what, int channels, int dstate, int ngroups, int dtype, int device) {
  if (channels <= 0 || dstate <= 0 || ngroups <= 0) {
    set_error("%s: channels, dstate and ngroups must be positive (got %d %d %d)", what, channels, dstate, ngroups);
    return SSD_ERR_BAD_SHAPE;
  }
  if (channels % ngroups) { set_error("%s: channels (%d) must be a multiple of ngroups (%d)", what, channels, ngroups); return SSD_ERR_BAD_SHAPE; }
  if (dstate > 64) { set_error("%s: dstate (%d) must be <= 64", what, dstate); return SSD_ERR_UNSUPPORTED; }
  if (dtype != SSD_F32 && dtype != SSD_BF16) { set_error("%s: unknown dtype %d", what, dtype); return SSD_ERR_UNSUPPORTED; }
  if (device >= 0) {
    int cur = -1;
    if (cudaGetDevice(&cur) != cudaSuccess || cur != device) {
      set_error("%s: current CUDA device is %d but dims.device is %d (the library never switches devices)", what, cur, device);
      return SSD_ERR_CUDA;
    }
  }
  return SSD_OK;
}

struct SelPlan {
  SelGeo q;
  int NP, nb_bwd, segs_fwd, segs_bwd;
  size_t ckpt, segst, segdt, part_bc, part_par, fwd_bytes, bwd_bytes;   // offsets and totals
};

// Parts of the sequence.  n blocks walk the tokens one after the other; where they are few the SMs mostly wait, and the sequence is cut into
// parts, which costs a pass over the steps for the states (or gradients) that the parts begin with: about eight blocks to an SM in all, as
// far as a part keeps `least_tiles` tiles.  Measured (us of the call, L2 flushed; parts, the rule's choice in brackets), 16 states, bf16, gated:
//   forward    1 x 4096 x 1536 (24 blocks)  1: 621, 12: 114, 24: 93, [43: 95], 64: 108     12 x 1024 x 1024 (192)  1: 188, 4: 165, [6: 158], 8: 162
//              4 x 2048 x 1536 (96)         1: 316, 4: 197, [12: 167], 24: 169             14 x 1024 x 1024 (224)  1: 188, 4: 190, [5: 184]
//              2 x 512 x 768 (24)           1: 84, 4: 42, 8: 32, [16: 26]                  16 x 1024 x 1024 (256)  [1: 188], 4: 201; 8 x 4096 x 2048 (256)  [1: 727], 4: 758
//   backward   1 x 4096 x 1536 (48 blocks)  1: 1183, 8: 270, [24: 223], 48: 231            12 x 1024 x 1024 (384)  1: 427, 2: 486, [3: 396], 4: 407
//              4 x 2048 x 1536 (192)        1: 707, 3: 417, 4: 485, [6: 406], 16: 417      14 x 1024 x 1024 (448)  [1: 483], 2: 513, 4: 496
//              2 x 512 x 768 (48)           1: 159, 4: 67, [8: 47], 16: 48                 64 x 512 x 512 (1024)   [1: 474], 2: 502, 4: 513
// so one part from 1.7 blocks to an SM on in the forward and from 2.8 in the backward.
int choose_parts(long long n, int L, long long below, int least_tiles) {
  const int tiles = cdiv(L, SEL_T);
  if (n >= below) return 1;
  long long s = 8 * 148 / n;
  if (s > tiles / least_tiles) s = tiles / least_tiles;
  if (s < 2) return 1;
  return cdiv(tiles, cdiv(tiles, (int)s));
}
void set_parts(SelGeo& q, int segs) {
  q.segs = segs;
  q.seg_len = cdiv(cdiv(q.L, SEL_T), segs) * SEL_T;
}

int make_sel_plan(const SsdSelDims* d, SelPlan* o) {
  if (!d) { set_error("selscan: dims is NULL"); return SSD_ERR_NULL_POINTER; }
  if (d->batch <= 0 || d->seqlen <= 0) { set_error("selscan: batch and seqlen must be positive (got %d %d)", d->batch, d->seqlen); return SSD_ERR_BAD_SHAPE; }
  const int rc = check_common("selscan", d->channels, d->dstate, d->ngroups, d->dtype, -1);
  if (rc) return rc;
  SelGeo& q = o->q;
  q.B = d->batch; q.L = d->seqlen; q.D = d->channels; q.N = d->dstate; q.G = d->ngroups; q.Dg = q.D / q.G;
  q.softplus = d->dt_softplus != 0;
  o->NP = padded_states(q.N);
  q.nb = cdiv(q.Dg, block_channels(o->NP));
  o->nb_bwd = cdiv(q.Dg, block_channels_bwd(o->NP));
  q.nc = cdiv(q.L, SEL_C);
  q.wide = 0;
  if (q.G > 65535 || (long long)q.B * q.L * (o->NP / 2) / 64 >= 0x7fffffffLL) { set_error("selscan: too many groups or tokens for one grid"); return SSD_ERR_UNSUPPORTED; }
  if ((long long)q.D * (o->NP + 2) > 0x7ffffff0LL) { set_error("selscan: too many channels (%d)", q.D); return SSD_ERR_UNSUPPORTED; }
  q.par_row = (q.D * (o->NP + 2) + 3) / 4 * 4;
  const long long GN = (long long)q.G * q.N;
  auto pick = [](long long v, long long dflt) { return v ? v : dflt; };
  q.xsl = pick(d->x_stride_l, q.D); q.xsb = pick(d->x_stride_b, (long long)q.D * q.L);
  q.dtsl = pick(d->dt_stride_l, q.D); q.dtsb = pick(d->dt_stride_b, (long long)q.D * q.L);
  q.bsl = pick(d->b_stride_l, GN); q.bsb = pick(d->b_stride_b, GN * q.L);
  q.csl = pick(d->c_stride_l, GN); q.csb = pick(d->c_stride_b, GN * q.L);
  q.zsl = pick(d->z_stride_l, q.D); q.zsb = pick(d->z_stride_b, (long long)q.D * q.L);
  q.ysl = pick(d->y_stride_l, q.D); q.ysb = pick(d->y_stride_b, (long long)q.D * q.L);
  if (q.xsl < q.D || q.dtsl < q.D || q.zsl < q.D || q.ysl < q.D || q.bsl < GN || q.csl < GN) {
    set_error("selscan: sequence strides must be at least the dense row size");
    return SSD_ERR_BAD_SHAPE;
  }
  const long long nf = (long long)q.B * q.G * q.nb, nb = (long long)q.B * q.G * o->nb_bwd;
  o->segs_fwd = choose_parts(nf, q.L, 246, 2);
  o->segs_bwd = choose_parts(nb, q.L, 414, 4);
  if (nf * o->segs_fwd > 0x7fffffffLL || nb * o->segs_bwd > 0x7fffffffLL) { set_error("selscan: too many blocks for one grid"); return SSD_ERR_UNSUPPORTED; }
  q.segs = 1; q.seg_len = 0;
  const int most = o->segs_fwd > o->segs_bwd ? o->segs_fwd : o->segs_bwd;
  const size_t st = (size_t)q.B * most * q.D * sizeof(float);
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t r = at; at += up256(bytes); return r; };
  o->segst = take(st * o->NP); o->segdt = take(st);
  o->fwd_bytes = at + 256;
  o->ckpt = take((size_t)q.B * q.nc * q.D * o->NP * sizeof(float));
  o->part_bc = take((size_t)q.G * o->nb_bwd * q.B * q.L * 2 * o->NP * sizeof(float));
  o->part_par = take((size_t)q.B * o->segs_bwd * q.par_row * sizeof(float));
  o->bwd_bytes = at + 256;
  return SSD_OK;
}
int need_device(const SsdSelDims* d) { return check_common("selscan", d->channels, d->dstate, d->ngroups, d->dtype, d->device); }

#define SEL_SHAPE(F) \
  switch (pl.NP) { case 4: F(Sh4); break; case 8: F(Sh8); break; case 16: F(Sh16); break; case 32: F(Sh32); break; default: F(Sh64); }

#define SEL_SHAPE_BWD(F) \
  switch (pl.NP) { case 4: F(Bh4); break; case 8: F(Bh8); break; case 16: F(Bh16); break; case 32: F(Bh32); break; default: F(Bh64); }

// Whether four channels of a row can be moved at once (8 bytes of bf16, 16 of fp32): every row of every tensor starts there.
bool rows_fit(const SelGeo& q, int es, std::initializer_list<const void*> ps, std::initializer_list<long long> strides) {
  uintptr_t low = (uintptr_t)(q.Dg * es);
  for (const void* p : ps) low |= (uintptr_t)p;
  for (long long v : strides) low |= (uintptr_t)(v * es);
  return low % (4 * es) == 0;
}
template <typename T> int sel_forward(SelPlan pl, const SelFwd& p, cudaStream_t s) {
  SelGeo& q = pl.q;
  set_parts(q, pl.segs_fwd);
  q.wide = rows_fit(q, sizeof(T), {p.x, p.dt, p.z, p.y}, {q.xsb, q.xsl, q.dtsb, q.dtsl, p.z ? q.zsb : 0, p.z ? q.zsl : 0, p.y ? q.ysb : 0, p.y ? q.ysl : 0});
  const unsigned grid = (unsigned)((long long)q.B * q.segs * q.G * q.nb);
  if (q.segs > 1) {
#define SEL_RUN(S) launch<k_sel_fwd<T, S, 1>>(grid, S::TH, 0, s, q, p)
    SEL_SHAPE(SEL_RUN)
#undef SEL_RUN
    SSD_CUDA_CHECK_LAUNCH("selscan_parts");
  }
#define SEL_RUN(S) launch<k_sel_fwd<T, S, 0>>(grid, S::TH, 0, s, q, p)
  SEL_SHAPE(SEL_RUN)
#undef SEL_RUN
  SSD_CUDA_CHECK_LAUNCH("selscan_fwd");
  return SSD_OK;
}

template <typename T> int sel_backward(SelPlan pl, const SelBwd& p, const SsdSelBwdPtrs& u, cudaStream_t s) {
  SelGeo& q = pl.q;
  q.nb = pl.nb_bwd;
  set_parts(q, pl.segs_bwd);
  q.wide = rows_fit(q, sizeof(T), {p.x, p.dt, p.z, p.dy, p.dx, p.ddt, p.dz}, {q.xsb, q.xsl, q.dtsb, q.dtsl, p.z ? q.zsb : 0, p.z ? q.zsl : 0, q.ysb, q.ysl});
  const unsigned grid = (unsigned)((long long)q.B * q.segs * q.G * q.nb);
  if (q.segs > 1) {
#define SEL_RUN(S) launch<k_sel_bwd_part<T, S>>(grid, S::TH, 0, s, q, p)
    SEL_SHAPE_BWD(SEL_RUN)
#undef SEL_RUN
    SSD_CUDA_CHECK_LAUNCH("selscan_bwd_parts");
  }
#define SEL_RUN(S) do { \
    if (p.z) launch<k_sel_bwd<T, S, true>>(grid, S::TH, S::bwd_smem<T>(), s, q, p); \
    else launch<k_sel_bwd<T, S, false>>(grid, S::TH, S::bwd_smem<T>(), s, q, p); } while (0)
  SEL_SHAPE_BWD(SEL_RUN)
#undef SEL_RUN
  SSD_CUDA_CHECK_LAUNCH("selscan_bwd");
  launch<k_sel_sum_bc<T>>(dim3((unsigned)(((long long)q.B * q.L * (pl.NP / 2) + 63) / 64), (unsigned)q.G), 256, 0, s, q, pl.NP, p.part_bc, (T*)u.dB, (T*)u.dC);
  SSD_CUDA_CHECK_LAUNCH("selscan_sum_bc");
  launch<k_sel_sum_par>((unsigned)(((long long)q.D * (pl.NP + 2) + 31) / 32), dim3(32, 8), 0, s, q, pl.NP, p.part_par, u.dA, u.dD, u.ddt_bias);
  SSD_CUDA_CHECK_LAUNCH("selscan_sum_par");
  return SSD_OK;
}

char* aligned_base(void* ws) { return (char*)(((uintptr_t)ws + 255) & ~(uintptr_t)255); }
int check_ws(const void* ws, size_t have, size_t need) {
  if (!ws) { set_error("selscan: workspace is NULL"); return SSD_ERR_NULL_POINTER; }
  if (have < need) { set_error("selscan: workspace too small: %zu < %zu", have, need); return SSD_ERR_WORKSPACE_TOO_SMALL; }
  return SSD_OK;
}

}  // namespace
}  // namespace ssd

using namespace ssd;

extern "C" {

size_t ssd_selscan_workspace_bytes(const SsdSelDims* dims, int32_t pass) {
  clear_error();
  SelPlan pl;
  if (make_sel_plan(dims, &pl)) return 0;
  return pass == SSD_PASS_BWD ? pl.bwd_bytes : pl.fwd_bytes;
}

int32_t ssd_selscan_forward(const SsdSelDims* dims, const SsdSelFwdPtrs* p, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  clear_error();
  SelPlan pl;
  int rc = make_sel_plan(dims, &pl);
  if (rc || (rc = need_device(dims))) return rc;
  if (!p || !p->x || !p->dt || !p->A || !p->Bm || !p->Cm || !p->y) { set_error("selscan: x, dt, A, B, C and y must be non-NULL"); return SSD_ERR_NULL_POINTER; }
  if ((rc = check_ws(workspace, workspace_bytes, pl.fwd_bytes))) return rc;
  char* ws = aligned_base(workspace);
  SelFwd f{p->x, p->dt, p->Bm, p->Cm, p->z, p->A, p->D, p->dt_bias, p->init_state, p->lengths, p->y, p->final_state,
           workspace_bytes >= pl.bwd_bytes ? (float*)(ws + pl.ckpt) : nullptr, (float*)(ws + pl.segst), (float*)(ws + pl.segdt)};
  cudaStream_t s = (cudaStream_t)cuda_stream;
  return dims->dtype == SSD_BF16 ? sel_forward<__nv_bfloat16>(pl, f, s) : sel_forward<float>(pl, f, s);
}

int32_t ssd_selscan_backward(const SsdSelDims* dims, const SsdSelBwdPtrs* p, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  clear_error();
  SelPlan pl;
  int rc = make_sel_plan(dims, &pl);
  if (rc || (rc = need_device(dims))) return rc;
  if (!p || !p->x || !p->dt || !p->A || !p->Bm || !p->Cm || !p->dy || !p->dx || !p->ddt || !p->dA || !p->dB || !p->dC) {
    set_error("selscan backward: a required pointer is NULL");
    return SSD_ERR_NULL_POINTER;
  }
  if ((p->z != nullptr) != (p->dz != nullptr) || (p->D && !p->dD) || (p->dt_bias && !p->ddt_bias)) {
    set_error("selscan backward: dz, dD and ddt_bias go with z, D and dt_bias");
    return SSD_ERR_NULL_POINTER;
  }
  if ((rc = check_ws(workspace, workspace_bytes, pl.bwd_bytes))) return rc;
  char* ws = aligned_base(workspace);
  cudaStream_t s = (cudaStream_t)cuda_stream;
  const bool bf = dims->dtype == SSD_BF16;
  if (!p->fwd_saved) {   // the states at the tiles' starts again
    SelFwd f{p->x, p->dt, p->Bm, p->Cm, nullptr, p->A, nullptr, p->dt_bias, p->init_state, p->lengths, nullptr, nullptr,
             (float*)(ws + pl.ckpt), (float*)(ws + pl.segst), (float*)(ws + pl.segdt)};
    rc = bf ? sel_forward<__nv_bfloat16>(pl, f, s) : sel_forward<float>(pl, f, s);
    if (rc) return rc;
  }
  SelBwd b{p->x, p->dt, p->Bm, p->Cm, p->z, p->dy, p->A, p->D, p->dt_bias, p->dfinal_state, (const float*)(ws + pl.ckpt), p->lengths,
           p->dx, p->ddt, p->dz, p->dinit_state, (float*)(ws + pl.part_bc), (float*)(ws + pl.part_par), (float*)(ws + pl.segst),
           (float*)(ws + pl.segdt)};
  return bf ? sel_backward<__nv_bfloat16>(pl, b, *p, s) : sel_backward<float>(pl, b, *p, s);
}

int32_t ssd_selscan_step(const SsdSelStepDims* d, const SsdStepPtrs* p, void* cuda_stream) {
  clear_error();
  if (!d || !p) { set_error("selscan step: dims or pointers are NULL"); return SSD_ERR_NULL_POINTER; }
  if (d->streams <= 0) { set_error("selscan step: streams must be positive (got %d)", d->streams); return SSD_ERR_BAD_SHAPE; }
  const int rc = check_common("selscan step", d->channels, d->dstate, d->ngroups, d->dtype, d->device);
  if (rc) return rc;
  if (!p->state || !p->x || !p->dt || !p->A || !p->Bm || !p->Cm || !p->y) {
    set_error("selscan step: state, x, dt, A, B, C and y must be non-NULL");
    return SSD_ERR_NULL_POINTER;
  }
  SelStep q;
  q.S = d->streams; q.D = d->channels; q.N = d->dstate; q.G = d->ngroups; q.Dg = q.D / q.G; q.softplus = d->dt_softplus != 0;
  const long long GN = (long long)q.G * q.N;
  auto pick = [](long long v, long long dflt) { return v ? v : dflt; };
  q.xs = pick(d->x_stride_s, q.D); q.dts = pick(d->dt_stride_s, q.D); q.bs = pick(d->b_stride_s, GN); q.cs = pick(d->c_stride_s, GN);
  q.zs = pick(d->z_stride_s, q.D); q.ys = pick(d->y_stride_s, q.D);
  if (q.xs < q.D || q.dts < q.D || q.zs < q.D || q.ys < q.D || q.bs < GN || q.cs < GN) {
    set_error("selscan step: strides must be at least the dense row size");
    return SSD_ERR_BAD_SHAPE;
  }
  // what a thread writes is read by no other: y may be x, dt or z itself (a channel's lanes have read theirs by then), nothing else shared
  const int es = d->dtype == SSD_BF16 ? 2 : 4;
  auto of_streams = [&](const void* p, long long stride, long long width) { return Rows{p, q.S, stride * es, width * es}; };
  const Rows state{p->state, 1, 0, (long long)q.S * q.D * q.N * 4}, y = of_streams(p->y, q.ys, q.D);
  const Rows ins[] = {of_streams(p->x, q.xs, q.D), of_streams(p->dt, q.dts, q.D), of_streams(p->z, q.zs, q.D), of_streams(p->Bm, q.bs, GN),
                      of_streams(p->Cm, q.cs, GN), {p->A, 1, 0, (long long)q.D * q.N * 4}, {p->D, 1, 0, q.D * 4LL}, {p->dt_bias, 1, 0, q.D * 4LL}};
  if (rows_share(state, y)) { set_error("selscan step: state and y share memory"); return SSD_ERR_BAD_SHAPE; }
  for (int i = 0; i < 8; ++i) {
    const bool itself = i < 3 && ins[i].p == y.p && (q.S == 1 || ins[i].stride == y.stride);
    if (rows_share(state, ins[i]) || (!itself && rows_share(y, ins[i]))) {
      static const char* const names[] = {"x", "dt", "z", "B", "C", "A", "D", "dt_bias"};
      set_error("selscan step: %s shares memory with the state or, without being it, with y", names[i]);
      return SSD_ERR_BAD_SHAPE;
    }
  }
  const int lpc = lanes_for(q.N);
  if ((long long)q.D * lpc > 0x7fffff00LL) { set_error("selscan step: too many channels (%d)", q.D); return SSD_ERR_UNSUPPORTED; }
  q.nx = (q.D * lpc + 255) / 256;
  const bool four = (long long)q.S * q.nx >= 4LL * 148 * 8;   // four streams per thread where the SMs stay full
  q.groups = four ? (q.S + 3) / 4 : q.S;
  const long long blocks = (long long)q.groups * q.nx;
  if (blocks > 0x7fffffffLL) { set_error("selscan step: too many blocks for one grid (%lld)", blocks); return SSD_ERR_UNSUPPORTED; }
  // four states, and four values of B and C, at a time
  const bool vec = q.N == 4 * lpc && ((uintptr_t)p->state & 15) == 0 && (((uintptr_t)p->Bm | (uintptr_t)p->Cm) & (4 * es - 1)) == 0 && q.bs % 4 == 0 && q.cs % 4 == 0;
  cudaStream_t s = (cudaStream_t)cuda_stream;
#define SEL_GO(T, LPC, VEC) do { \
    if (four) launch<k_sel_step<T, LPC, VEC, 4>>((unsigned)blocks, 256, 0, s, q, *p); \
    else launch<k_sel_step<T, LPC, VEC, 1>>((unsigned)blocks, 256, 0, s, q, *p); } while (0)
#define SEL_RUN(LPC) do { \
    if (d->dtype == SSD_BF16) { if (vec) SEL_GO(__nv_bfloat16, LPC, true); else SEL_GO(__nv_bfloat16, LPC, false); } \
    else { if (vec) SEL_GO(float, LPC, true); else SEL_GO(float, LPC, false); } } while (0)
  switch (lpc) { case 1: SEL_RUN(1); break; case 2: SEL_RUN(2); break; case 4: SEL_RUN(4); break; case 8: SEL_RUN(8); break; default: SEL_RUN(16); }
#undef SEL_RUN
#undef SEL_GO
  SSD_CUDA_CHECK_LAUNCH("selscan_step");
  return SSD_OK;
}

}  // extern "C"
