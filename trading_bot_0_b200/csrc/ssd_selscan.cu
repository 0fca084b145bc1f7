// Selective scan with a decay per channel and state (the Mamba-1 form):
//     s_t = act(dt_t + dt_bias)          a_t[n] = exp(s_t A[n])          h_t[n] = a_t[n] h_{t-1}[n] + s_t x_t B_t[n]
//     y_t = (sum_n C_t[n] h_t[n] + D x_t) silu(z_t)
// per batch row and channel, B and C shared by the channels of a group; its gradients; and one step over many streams.
//
// The decays differ per channel and state, so there is no matrix form: every (token, channel, state) costs an exponential and a
// handful of fp32 operations, and the special-function units (16 exponentials per clock and SM) set the pace, not the memory
// (one bf16 token-channel is 8 bytes moved against dstate exponentials).  A thread holds four states of one channel in registers
// and walks the tokens; dstate / 4 neighbouring lanes make up a channel.  What is needed once per token and channel (softplus, s x,
// the gate) is computed once by one thread of the block, a tile of 16 tokens ahead, and handed over in shared memory.
#include "common.cuh"
#include "ssd_internal.h"
#include "umma.cuh"

namespace ssd {
namespace {

using umma::ex2;

constexpr int SEL_T = 16;             // tokens per tile, and between the states kept for the backward pass
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct SelGeo {
  int B, L, D, N, G, Dg, nb;          // nb = channel blocks per group
  int segs, seg_len;                  // the tokens in `segs` parts of seg_len (a multiple of SEL_T)
  int softplus, nt;                   // nt = tiles of the whole sequence
  int par_row;                        // a block's sums of dA, dD and ddt_bias: D*NP + 2*D floats, up to a multiple of four
  long long xsb, xsl, dtsb, dtsl, bsb, bsl, csb, csl, zsb, zsl, ysb, ysl;
};

// Lanes per channel -> block shape.
template <int LPC> struct Sh {
  static constexpr int NP = 4 * LPC;                 // states per channel, padded
  static constexpr int CHB = LPC <= 8 ? 32 : 16;     // channels per block
  static constexpr int TH = CHB * LPC;               // threads
  static constexpr int IT = SEL_T * CHB / TH;        // (token, channel) items per thread
  static constexpr int RS = TH / CHB;                // tokens between a thread's items
  static constexpr int BI = SEL_T * NP / TH;         // values of B (and of C) per thread
  static constexpr int W = TH / 32;
  static constexpr int BWD_SMEM = SEL_T * CHB * 16 + W * SEL_T * 2 * NP * 4;   // backward: a tile's values per channel, the warps' shares of dB and dC
};

// log(1 + e) for e in [0, 1]: e P(e) with P the least-maximum fit of log1p(e) / e of degree 8 (relative error 3e-8, 1.7e-7 as
// evaluated), so that small step sizes keep their digits where log(1 + e) would lose them.
__device__ __forceinline__ float log1p01(float e) {
  float p = 0.00523267664f;
  p = fmaf(p, e, -0.0295051682f);
  p = fmaf(p, e, 0.0782258369f);
  p = fmaf(p, e, -0.13663236f);
  p = fmaf(p, e, 0.191060022f);
  p = fmaf(p, e, -0.24842981f);
  p = fmaf(p, e, 0.333190967f);
  p = fmaf(p, e, -0.499994931f);
  p = fmaf(p, e, 0.99999997f);
  return p * e;
}
// softplus(v) = max(v, 0) + log(1 + exp(-|v|))
__device__ __forceinline__ float sel_step(float raw, float bias, int softplus) {
  const float v = raw + bias;
  return softplus ? fmaxf(v, 0.f) + log1p01(expf(-fabsf(v))) : v;
}
// d step / d raw
__device__ __forceinline__ float sel_dstep(float raw, float bias, int softplus) {
  return softplus ? 1.f / (1.f + __expf(-(raw + bias))) : 1.f;
}
__device__ __forceinline__ float sig(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float hsum(f32x2 v) { float a, b; unpack2(v, a, b); return a + b; }
__device__ __forceinline__ f32x2 dup2(float v) { return pack2(v, v); }
__device__ __forceinline__ f32x2 ex2_2(f32x2 v) { float a, b; unpack2(v, a, b); return pack2(ex2(a), ex2(b)); }
// exp(s A) for a pair of decays (A2 = A log2 e).  ex2.approx is 2e-8 low on average over the arguments that decays have (1.7e-8 to
// 2.6e-8 in every interval measured between -0.75 and -0.001; rms 4e-8); a state is a product of hundreds of them, where an offset
// adds up and scatter does not, so the argument is raised by 2e-8 log2 e.
__device__ __forceinline__ f32x2 decay2(f32x2 A2, f32x2 s2) { return ex2_2(fma2(A2, s2, pack2(2.9e-8f, 2.9e-8f))); }

struct Place { int b, seg, g, d, c; bool live; };    // batch row, part, group, channel (of all), channel of the block
template <int LPC> __device__ __forceinline__ Place place(const SelGeo& q, int c) {
  const int nblk = q.G * q.nb;
  Place p;
  const int blk = blockIdx.x % nblk, rest = blockIdx.x / nblk;
  p.seg = rest % q.segs; p.b = rest / q.segs;
  p.g = blk / q.nb;
  const int cg = (blk - p.g * q.nb) * Sh<LPC>::CHB + c;
  p.c = c; p.live = cg < q.Dg; p.d = p.g * q.Dg + (p.live ? cg : 0);
  return p;
}

// Four states of a [.., D, N] fp32 array (N not padded).
template <int LPC> __device__ __forceinline__ void load_state(const float* p, int N, int nl, bool live, float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = live && p && nl * 4 + j < N ? p[nl * 4 + j] : 0.f;
}
template <int LPC> __device__ __forceinline__ void store_state(float* p, int N, int nl, bool live, const float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) if (live && nl * 4 + j < N) p[nl * 4 + j] = v[j];
}

struct SelFwd {
  const void *x, *dt, *Bm, *Cm, *z;
  const float *A, *D, *bias, *init;
  const int* lengths;
  void* y;
  float *fin, *ckpt;                  // ckpt [B][nt][D][NP]: the state entering every tile
  float *segst, *segdt;               // [B][segs][D][NP] states of the parts from zero, [B][segs][D] their summed steps
};

// MODE 0: outputs (and the states kept for the backward); MODE 1: a part's own state from zero and its summed steps.
template <typename T, int LPC, int MODE>
__global__ void __launch_bounds__(Sh<LPC>::TH) k_sel_fwd(SelGeo q, SelFwd p) {
  using S = Sh<LPC>;
  constexpr int NP = S::NP, CHB = S::CHB, TH = S::TH, IT = S::IT, BI = S::BI;
  __shared__ float2 s_dt[2][SEL_T][CHB];             // step, step * x
  __shared__ __align__(16) float s_B[2][SEL_T][NP], s_C[2][SEL_T][NP];
  __shared__ float s_y[SEL_T][CHB];
  pdl_wait();
  const int tid = threadIdx.x, c = tid / LPC, nl = tid % LPC;
  const Place me = place<LPC>(q, c), it = place<LPC>(q, tid % CHB);   // roles: states of a channel; (token, channel) items
  if (MODE == 1 && me.seg == q.segs - 1) return;
  const int len = p.lengths ? min(max(p.lengths[me.b], 0), q.L) : q.L;
  const int t_begin = me.seg * q.seg_len, t_end = min(t_begin + q.seg_len, q.L);
  const int r0 = tid / CHB;
  const T* xp = (const T*)p.x + (long long)it.b * q.xsb + it.d;
  const T* dtp = (const T*)p.dt + (long long)it.b * q.dtsb + it.d;
  const T* zp = (const T*)p.z + (long long)it.b * q.zsb + it.d;
  const T* bp = (const T*)p.Bm + (long long)it.b * q.bsb + (long long)it.g * q.N;
  const T* cp = (const T*)p.Cm + (long long)it.b * q.csb + (long long)it.g * q.N;
  T* yp = (T*)p.y + (long long)it.b * q.ysb + it.d;
  const float bias = p.bias ? p.bias[it.d] : 0.f, Dv = p.D ? p.D[it.d] : 0.f;
  const bool want_y = MODE == 0 && p.y;

  float A4[4], h4[4];
  load_state<LPC>(p.A + (long long)me.d * q.N, q.N, nl, me.live, A4);
  const f32x2 A01 = pack2(A4[0] * LOG2E, A4[1] * LOG2E), A23 = pack2(A4[2] * LOG2E, A4[3] * LOG2E);
  f32x2 h01 = 0ull, h23 = 0ull;
  float dtsum = 0.f;
  if (MODE == 0) {
    load_state<LPC>(p.init ? p.init + ((long long)me.b * q.D + me.d) * q.N : nullptr, q.N, nl, me.live, h4);
    h01 = pack2(h4[0], h4[1]); h23 = pack2(h4[2], h4[3]);
    for (int s = 0; s < me.seg; ++s) {
      const long long at = ((long long)me.b * q.segs + s) * q.D + me.d;
      const float4 v = *reinterpret_cast<const float4*>(p.segst + at * NP + nl * 4);
      const f32x2 d2 = dup2(p.segdt[at]);
      h01 = fma2(decay2(A01, d2), h01, pack2(v.x, v.y));
      h23 = fma2(decay2(A23, d2), h23, pack2(v.z, v.w));
    }
  }

  T rx[IT], rd[IT], rz[IT], rb[BI], rc[BI];
  auto request = [&](int t0) {                       // values of a tile into registers; nothing past the end is read
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int t = t0 + r0 + i * S::RS;
      const bool ok = it.live && t < len && t < t_end;
      rx[i] = rd[i] = rz[i] = T(0.f);
      if (ok) {
        rx[i] = xp[(long long)t * q.xsl]; rd[i] = dtp[(long long)t * q.dtsl];
        if (want_y && p.z) rz[i] = zp[(long long)t * q.zsl];
      }
    }
#pragma unroll
    for (int i = 0; i < BI; ++i) {
      const int e = tid + i * TH, n = e % NP, t = t0 + e / NP;
      const bool ok = n < q.N && t < len && t < t_end;
      rb[i] = rc[i] = T(0.f);
      if (ok) {
        rb[i] = bp[(long long)t * q.bsl + n];
        if (want_y) rc[i] = cp[(long long)t * q.csl + n];
      }
    }
  };
  float kx[IT], kz[IT];
  auto hand_over = [&](int t0, int buf) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int t = t0 + r0 + i * S::RS;
      kx[i] = (float)rx[i]; kz[i] = (float)rz[i];
      const float s = it.live && t < len && t < t_end ? sel_step((float)rd[i], bias, q.softplus) : 0.f;
      s_dt[buf][r0 + i * S::RS][tid % CHB] = make_float2(s, s * kx[i]);
    }
#pragma unroll
    for (int i = 0; i < BI; ++i) {
      const int e = tid + i * TH;
      s_B[buf][e / NP][e % NP] = (float)rb[i];
      if (want_y) s_C[buf][e / NP][e % NP] = (float)rc[i];
    }
  };

  request(t_begin);
  hand_over(t_begin, 0);
  __syncthreads();
  int buf = 0;
  for (int t0 = t_begin; t0 < t_end; t0 += SEL_T, buf ^= 1) {
    const bool more = t0 + SEL_T < t_end;
    float ex[IT], ez[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) { ex[i] = kx[i]; ez[i] = kz[i]; }
    if (more) request(t0 + SEL_T);
    if (MODE == 0 && p.ckpt && me.live) {
      float4 v;
      unpack2(h01, v.x, v.y); unpack2(h23, v.z, v.w);
      *reinterpret_cast<float4*>(p.ckpt + (((long long)me.b * q.nt + t0 / SEL_T) * q.D + me.d) * NP + nl * 4) = v;
    }
    if (t0 < len) {
#pragma unroll
      for (int u = 0; u < SEL_T; u += LPC) {
        float v[LPC];
#pragma unroll
        for (int i = 0; i < LPC; ++i) {
          const float2 sd = s_dt[buf][u + i][c];
          const float4 b4 = *reinterpret_cast<const float4*>(&s_B[buf][u + i][nl * 4]);
          const f32x2 s2 = dup2(sd.x), x2 = dup2(sd.y);
          h01 = fma2(decay2(A01, s2), h01, mul2(pack2(b4.x, b4.y), x2));
          h23 = fma2(decay2(A23, s2), h23, mul2(pack2(b4.z, b4.w), x2));
          if (MODE == 1) dtsum += sd.x;
          if (MODE == 0) {
            const float4 c4 = *reinterpret_cast<const float4*>(&s_C[buf][u + i][nl * 4]);
            v[i] = hsum(fma2(pack2(c4.z, c4.w), h23, mul2(pack2(c4.x, c4.y), h01)));
          }
        }
        if (MODE == 0 && want_y) {
          int k;
          const float sum = fold_rows<LPC, LPC>(v, nl, k);
          s_y[u + k][c] = sum;
        }
      }
    }
    __syncthreads();
    if (want_y && it.live) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int r = r0 + i * S::RS, t = t0 + r;
        if (t < t_end) {
          float o = 0.f;
          if (t < len) {
            o = fmaf(Dv, ex[i], s_y[r][tid % CHB]);
            if (p.z) o *= ez[i] * sig(ez[i]);
          }
          stf(yp + (long long)t * q.ysl, o);
        }
      }
    }
    if (more) hand_over(t0 + SEL_T, buf ^ 1);
    __syncthreads();
  }
  unpack2(h01, h4[0], h4[1]); unpack2(h23, h4[2], h4[3]);
  if (MODE == 1) {
    const long long at = ((long long)me.b * q.segs + me.seg) * q.D + me.d;
    if (me.live) {
      *reinterpret_cast<float4*>(p.segst + at * NP + nl * 4) = make_float4(h4[0], h4[1], h4[2], h4[3]);
      if (nl == 0) p.segdt[at] = dtsum;
    }
  } else if (p.fin && me.seg == q.segs - 1) {
    store_state<LPC>(p.fin + ((long long)me.b * q.D + me.d) * q.N, q.N, nl, me.live, h4);
  }
}

// ---------------------------------------------------------------------------------------------
// Backward, with g_t = dL/dh_t = C_t dy'_t + a_{t+1} g_{t+1} and dy' = dy silu(z):
//     dB_t = sum_d g_t s x,   dC_t = sum_d dy' h_t,   dx = s (g.B) + D dy',   ds = x (g.B) + sum_n g_t a_t h_{t-1} A,
//     dA = sum_t g_t a_t h_{t-1} s.
// Per tile of 16 tokens the states and decays are computed again from the state kept at the tile's start and stay in registers
// (so an exponential is computed once here, as in the forward), then the tile is walked backwards.  Sums over the states go over the
// lanes of a channel, sums over the channels over the lanes and warps of a block; blocks leave partial sums of dB and dC which a
// second kernel adds in order.
struct SelBwd {
  const void *x, *dt, *Bm, *Cm, *z, *dy;
  const float *A, *D, *bias, *dfin, *ckpt;
  const int* lengths;
  void *dx, *ddt, *dz;
  float *dinit, *part_bc, *part_par;  // [G*nb][B*L][2*NP]; [B*segs][par_row]
  float *segst, *segdt;               // [B][segs][D][NP]: gradient that a part passes to the state before it, with nothing coming in
};

// A part's own gradient of the state before it, from zero.
template <typename T, int LPC>
__global__ void __launch_bounds__(Sh<LPC>::TH) k_sel_bwd_part(SelGeo q, SelBwd p) {
  using S = Sh<LPC>;
  constexpr int NP = S::NP, CHB = S::CHB, TH = S::TH, IT = S::IT, BI = S::BI;
  __shared__ float2 s_dt[SEL_T][CHB];                // step, dy'
  __shared__ __align__(16) float s_C[SEL_T][NP];
  pdl_wait();
  const int tid = threadIdx.x, c = tid / LPC, nl = tid % LPC;
  const Place me = place<LPC>(q, c), it = place<LPC>(q, tid % CHB);
  if (me.seg == 0) return;
  const int len = p.lengths ? min(max(p.lengths[me.b], 0), q.L) : q.L;
  const int t_begin = me.seg * q.seg_len, t_end = min(t_begin + q.seg_len, q.L);
  const int r0 = tid / CHB;
  const T* dtp = (const T*)p.dt + (long long)it.b * q.dtsb + it.d;
  const T* zp = (const T*)p.z + (long long)it.b * q.zsb + it.d;
  const T* dyp = (const T*)p.dy + (long long)it.b * q.ysb + it.d;
  const T* cp = (const T*)p.Cm + (long long)it.b * q.csb + (long long)it.g * q.N;
  const float bias = p.bias ? p.bias[it.d] : 0.f;
  float A4[4];
  load_state<LPC>(p.A + (long long)me.d * q.N, q.N, nl, me.live, A4);
  const f32x2 A01 = pack2(A4[0] * LOG2E, A4[1] * LOG2E), A23 = pack2(A4[2] * LOG2E, A4[3] * LOG2E);
  f32x2 g01 = 0ull, g23 = 0ull;
  float dtsum = 0.f;
  for (int t0 = t_begin + (t_end - t_begin - 1) / SEL_T * SEL_T; t0 >= t_begin; t0 -= SEL_T) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = r0 + i * S::RS, t = t0 + r;
      float s = 0.f, g = 0.f;
      if (it.live && t < len && t < t_end) {
        s = sel_step((float)dtp[(long long)t * q.dtsl], bias, q.softplus);
        g = (float)dyp[(long long)t * q.ysl];
        if (p.z) { const float z = (float)zp[(long long)t * q.zsl]; g *= z * sig(z); }
      }
      s_dt[r][tid % CHB] = make_float2(s, g);
    }
#pragma unroll
    for (int i = 0; i < BI; ++i) {
      const int e = tid + i * TH, n = e % NP, t = t0 + e / NP;
      s_C[e / NP][n] = n < q.N && t < len && t < t_end ? (float)cp[(long long)t * q.csl + n] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int r = SEL_T - 1; r >= 0; --r) {
      const float2 sd = s_dt[r][c];
      const float4 c4 = *reinterpret_cast<const float4*>(&s_C[r][nl * 4]);
      const f32x2 s2 = dup2(sd.x), y2 = dup2(sd.y);
      g01 = mul2(decay2(A01, s2), fma2(pack2(c4.x, c4.y), y2, g01));
      g23 = mul2(decay2(A23, s2), fma2(pack2(c4.z, c4.w), y2, g23));
      dtsum += sd.x;
    }
  }
  const long long at = ((long long)me.b * q.segs + me.seg) * q.D + me.d;
  if (me.live) {
    float4 v;
    unpack2(g01, v.x, v.y); unpack2(g23, v.z, v.w);
    *reinterpret_cast<float4*>(p.segst + at * NP + nl * 4) = v;
    if (nl == 0) p.segdt[at] = dtsum;
  }
}

// Sums of R values over the CPW lane groups of a warp that hold other channels (lane = channel * LPC + nl): every exchange folds
// two values into one; a lane ends up with the sums of `left` values, the first of them value `u`.
template <int LPC, int R> struct ChannelFold {
  static constexpr int CPW = 32 / LPC;
  static constexpr int left = R > CPW ? R / CPW : 1;
  __device__ static __forceinline__ void run(float (&v)[R], int lane, int& u) {
    u = 0;
    int o = 16;
#pragma unroll
    for (int n = R; n > 1; n >>= 1, o >>= 1) {
      if (o < LPC) break;
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < n / 2; ++i) {
        const float keep = up ? v[n / 2 + i] : v[i], give = up ? v[i] : v[n / 2 + i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
      u += up ? n / 2 : 0;
    }
#pragma unroll
    for (; o >= LPC && CPW > R; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  }
};

template <typename T, int LPC, bool GATED>
__global__ void __launch_bounds__(Sh<LPC>::TH) k_sel_bwd(SelGeo q, SelBwd p) {
  using S = Sh<LPC>;
  constexpr int NP = S::NP, CHB = S::CHB, TH = S::TH, IT = S::IT, BI = S::BI, W = S::W;
  __shared__ __align__(16) float s_B[SEL_T][NP], s_C[SEL_T][NP];
  __shared__ float s_1[SEL_T][CHB], s_2[SEL_T][CHB], s_3[GATED ? SEL_T : 1][CHB];
  extern __shared__ __align__(16) float4 sel_smem[];
  float4 (*s_v)[CHB] = reinterpret_cast<float4 (*)[CHB]>(sel_smem);    // step, step * x, dy', -
  float (*s_bc)[SEL_T][2 * NP] = reinterpret_cast<float (*)[SEL_T][2 * NP]>(sel_smem + SEL_T * CHB);
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = tid / LPC, nl = tid % LPC;
  const Place me = place<LPC>(q, c), it = place<LPC>(q, tid % CHB);
  const int len = p.lengths ? min(max(p.lengths[me.b], 0), q.L) : q.L;
  const int t_begin = me.seg * q.seg_len, t_end = min(t_begin + q.seg_len, q.L);
  const int r0 = tid / CHB, ic = tid % CHB;
  const T* xp = (const T*)p.x + (long long)it.b * q.xsb + it.d;
  const T* dtp = (const T*)p.dt + (long long)it.b * q.dtsb + it.d;
  const T* zp = (const T*)p.z + (long long)it.b * q.zsb + it.d;
  const T* dyp = (const T*)p.dy + (long long)it.b * q.ysb + it.d;
  const T* bp = (const T*)p.Bm + (long long)it.b * q.bsb + (long long)it.g * q.N;
  const T* cp = (const T*)p.Cm + (long long)it.b * q.csb + (long long)it.g * q.N;
  const long long out0 = (long long)it.b * q.L * q.D + it.d;
  const float bias = p.bias ? p.bias[it.d] : 0.f, Dv = p.D ? p.D[it.d] : 0.f;
  const int blk = blockIdx.x % (q.G * q.nb);

  float A4[4], g4[4];
  load_state<LPC>(p.A + (long long)me.d * q.N, q.N, nl, me.live, A4);
  const f32x2 A01 = pack2(A4[0] * LOG2E, A4[1] * LOG2E), A23 = pack2(A4[2] * LOG2E, A4[3] * LOG2E);
  load_state<LPC>(p.dfin ? p.dfin + ((long long)me.b * q.D + me.d) * q.N : nullptr, q.N, nl, me.live, g4);
  f32x2 g01 = pack2(g4[0], g4[1]), g23 = pack2(g4[2], g4[3]);    // a_{t+1} g_{t+1}
  for (int s = q.segs - 1; s > me.seg; --s) {
    const long long at = ((long long)me.b * q.segs + s) * q.D + me.d;
    const float4 v = *reinterpret_cast<const float4*>(p.segst + at * NP + nl * 4);
    const f32x2 d2 = dup2(p.segdt[at]);
    g01 = fma2(decay2(A01, d2), g01, pack2(v.x, v.y));
    g23 = fma2(decay2(A23, d2), g23, pack2(v.z, v.w));
  }
  f32x2 dA01 = 0ull, dA23 = 0ull;
  float dD = 0.f, dbias = 0.f;

  for (int t0 = t_begin + (t_end - t_begin - 1) / SEL_T * SEL_T; t0 >= t_begin; t0 -= SEL_T) {
    if (t0 >= len) {                                 // (uniform over the block) nothing here but zeros
      if (it.live)
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int t = t0 + r0 + i * S::RS;
          if (t < t_end) {
            const long long o = out0 + (long long)t * q.D;
            stf((T*)p.dx + o, 0.f); stf((T*)p.ddt + o, 0.f);
            if (GATED) stf((T*)p.dz + o, 0.f);
          }
        }
      for (int e = tid; e < SEL_T * 2 * NP; e += TH) {
        const int t = t0 + e / (2 * NP);
        if (t < t_end) p.part_bc[((long long)blk * q.B * q.L + (long long)me.b * q.L + t) * (2 * NP) + e % (2 * NP)] = 0.f;
      }
      continue;
    }
    float4 k4 = make_float4(0.f, 0.f, 0.f, 0.f);
    if (me.live) k4 = *reinterpret_cast<const float4*>(p.ckpt + (((long long)me.b * q.nt + t0 / SEL_T) * q.D + me.d) * NP + nl * 4);
    float vx[IT], vs[IT], vd[IT], vy[IT], vz[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int r = r0 + i * S::RS, t = t0 + r;
      vx[i] = vs[i] = vd[i] = vy[i] = vz[i] = 0.f;
      float dy0 = 0.f;
      if (it.live && t < len && t < t_end) {
        vx[i] = (float)xp[(long long)t * q.xsl];
        const float raw = (float)dtp[(long long)t * q.dtsl];
        vs[i] = sel_step(raw, bias, q.softplus);
        vd[i] = sel_dstep(raw, bias, q.softplus);
        dy0 = vy[i] = (float)dyp[(long long)t * q.ysl];
        if (GATED) { vz[i] = (float)zp[(long long)t * q.zsl]; dy0 *= vz[i] * sig(vz[i]); }
      }
      s_v[r][ic] = make_float4(vs[i], vs[i] * vx[i], dy0, 0.f);
    }
#pragma unroll
    for (int i = 0; i < BI; ++i) {
      const int e = tid + i * TH, n = e % NP, t = t0 + e / NP;
      const bool ok = n < q.N && t < len && t < t_end;
      s_B[e / NP][n] = ok ? (float)bp[(long long)t * q.bsl + n] : 0.f;
      s_C[e / NP][n] = ok ? (float)cp[(long long)t * q.csl + n] : 0.f;
    }
    __syncthreads();
    f32x2 a01[SEL_T], a23[SEL_T], h01[SEL_T + 1], h23[SEL_T + 1];
    h01[0] = pack2(k4.x, k4.y); h23[0] = pack2(k4.z, k4.w);
#pragma unroll
    for (int r = 0; r < SEL_T; ++r) {
      const float4 v = s_v[r][c];
      const float4 b4 = *reinterpret_cast<const float4*>(&s_B[r][nl * 4]);
      const f32x2 s2 = dup2(v.x), x2 = dup2(v.y);
      a01[r] = decay2(A01, s2); a23[r] = decay2(A23, s2);
      h01[r + 1] = fma2(a01[r], h01[r], mul2(pack2(b4.x, b4.y), x2));
      h23[r + 1] = fma2(a23[r], h23[r], mul2(pack2(b4.z, b4.w), x2));
    }
    f32x2 tA01 = 0ull, tA23 = 0ull;                  // a tile's share of dA: sums of 16, then sums of tiles
#pragma unroll
    for (int u = SEL_T - LPC; u >= 0; u -= LPC) {
      float v1[LPC], v2[LPC], v3[LPC];
#pragma unroll
      for (int i = LPC - 1; i >= 0; --i) {
        const int r = u + i;
        const float4 v = s_v[r][c];
        const float4 b4 = *reinterpret_cast<const float4*>(&s_B[r][nl * 4]), c4 = *reinterpret_cast<const float4*>(&s_C[r][nl * 4]);
        const f32x2 s2 = dup2(v.x), x2 = dup2(v.y), y2 = dup2(v.z);
        const f32x2 C01 = pack2(c4.x, c4.y), C23 = pack2(c4.z, c4.w);
        g01 = fma2(C01, y2, g01); g23 = fma2(C23, y2, g23);
        float w[8];
        const f32x2 e0 = mul2(g01, x2), e1 = mul2(g23, x2), e2 = mul2(h01[r + 1], y2), e3 = mul2(h23[r + 1], y2);
        unpack2(e0, w[0], w[1]); unpack2(e1, w[2], w[3]); unpack2(e2, w[4], w[5]); unpack2(e3, w[6], w[7]);
        v1[i] = hsum(fma2(pack2(b4.z, b4.w), g23, mul2(pack2(b4.x, b4.y), g01)));
        if (GATED) v3[i] = hsum(fma2(C23, h23[r + 1], mul2(C01, h01[r + 1])));
        g01 = mul2(g01, a01[r]); g23 = mul2(g23, a23[r]);
        const f32x2 q01 = mul2(g01, h01[r]), q23 = mul2(g23, h23[r]);
        v2[i] = hsum(fma2(A23, q23, mul2(A01, q01)));
        tA01 = fma2(q01, s2, tA01); tA23 = fma2(q23, s2, tA23);
        int k;
        using F = ChannelFold<LPC, 8>;
        F::run(w, lane, k);
#pragma unroll
        for (int j = 0; j < F::left; ++j) s_bc[warp][r][((k + j) >> 2) * NP + nl * 4 + ((k + j) & 3)] = w[j];
      }
      int k;
      const float a = fold_rows<LPC, LPC>(v1, nl, k);
      s_1[u + k][c] = a;
      const float b = fold_rows<LPC, LPC>(v2, nl, k);
      s_2[u + k][c] = b;
      if (GATED) {
        const float d = fold_rows<LPC, LPC>(v3, nl, k);
        s_3[u + k][c] = d;
      }
    }
    dA01 = add2(dA01, tA01); dA23 = add2(dA23, tA23);
    __syncthreads();
    float tD = 0.f, tb = 0.f;
    if (it.live)
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int r = r0 + i * S::RS, t = t0 + r;
        if (t < t_end) {
          const long long o = out0 + (long long)t * q.D;
          float dx = 0.f, ddt = 0.f, dz = 0.f;
          if (t < len) {
            const float gB = s_1[r][ic];
            float dy0 = vy[i];
            if (GATED) {
              const float sg = sig(vz[i]);
              dz = vy[i] * fmaf(Dv, vx[i], s_3[r][ic]) * sg * fmaf(vz[i], 1.f - sg, 1.f);
              dy0 *= vz[i] * sg;
            }
            dx = fmaf(vs[i], gB, Dv * dy0);
            ddt = fmaf(vx[i], gB, s_2[r][ic] * LN2) * vd[i];
            tD = fmaf(dy0, vx[i], tD); tb += ddt;
          }
          stf((T*)p.dx + o, dx); stf((T*)p.ddt + o, ddt);
          if (GATED) stf((T*)p.dz + o, dz);
        }
      }
    dD += tD; dbias += tb;
    for (int e = tid; e < SEL_T * 2 * NP; e += TH) {
      const int r = e / (2 * NP), t = t0 + r;
      float a = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) a += s_bc[w][r][e % (2 * NP)];
      if (t < t_end) p.part_bc[((long long)blk * q.B * q.L + (long long)me.b * q.L + t) * (2 * NP) + e % (2 * NP)] = a;
    }
    __syncthreads();
  }
  unpack2(g01, g4[0], g4[1]); unpack2(g23, g4[2], g4[3]);
  if (p.dinit && me.seg == 0) store_state<LPC>(p.dinit + ((long long)me.b * q.D + me.d) * q.N, q.N, nl, me.live, g4);
  float* par = p.part_par + ((long long)me.b * q.segs + me.seg) * q.par_row;
  if (me.live) {
    float4 v;
    unpack2(dA01, v.x, v.y); unpack2(dA23, v.z, v.w);
    *reinterpret_cast<float4*>(par + (long long)me.d * NP + nl * 4) = v;
  }
  s_1[r0][ic] = dD; s_2[r0][ic] = dbias;             // the block's threads of a channel, in order
  __syncthreads();
  if (tid < CHB && it.live) {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int r = 0; r < S::RS; ++r) { a += s_1[r][tid]; b += s_2[r][tid]; }
    par[(long long)q.D * NP + it.d] = a;
    par[(long long)q.D * (NP + 1) + it.d] = b;
  }
}

// dB, dC of a token and group: the channel blocks' shares in order.
template <typename T>
__global__ void __launch_bounds__(256) k_sel_sum_bc(SelGeo q, int NP, const float* __restrict__ part, T* __restrict__ dB, T* __restrict__ dC) {
  pdl_wait();
  const long long BL = (long long)q.B * q.L, n = BL * q.G * 2 * NP;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const int v = (int)(i % (2 * NP));
    const long long k = i / (2 * NP), bl = k % BL;
    const int g = (int)(k / BL), s = v % NP;
    if (s >= q.N) continue;
    float a = 0.f;
#pragma unroll 4
    for (int j = 0; j < q.nb; ++j) a += part[((long long)(g * q.nb + j) * BL + bl) * (2 * NP) + v];
    stf((v < NP ? dB : dC) + (bl * q.G + g) * q.N + s, a);
  }
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
// Four states per thread, dstate / 4 lanes per channel.
struct SelStep {
  int S, D, N, G, Dg, softplus;
  long long xs, dts, bs, cs, zs, ys;
};
template <typename T, int LPC, bool VEC>
__global__ void __launch_bounds__(256) k_sel_step(SelStep q, SsdStepPtrs p) {
  pdl_wait();
  const long long item = ((long long)blockIdx.x * 256 + threadIdx.x) / LPC, n = (long long)q.S * q.D;
  const int nl = threadIdx.x % LPC;
  const bool live = item < n;
  const long long i = live ? item : 0;
  const int s = (int)(i / q.D), d = (int)(i - (long long)s * q.D), g = d / q.Dg;
  float* hp = p.state + i * q.N + nl * 4;
  const float* ap = p.A + (long long)d * q.N + nl * 4;
  const T* bp = (const T*)p.Bm + s * q.bs + (long long)g * q.N + nl * 4;
  const T* cp = (const T*)p.Cm + s * q.cs + (long long)g * q.N + nl * 4;
  float h[4], a[4];
  if (VEC) {
    const float4 v = *reinterpret_cast<const float4*>(hp), w = __ldg(reinterpret_cast<const float4*>(ap));
    h[0] = v.x; h[1] = v.y; h[2] = v.z; h[3] = v.w;
    a[0] = w.x; a[1] = w.y; a[2] = w.z; a[3] = w.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool ok = nl * 4 + j < q.N;
      h[j] = ok ? hp[j] : 0.f; a[j] = ok ? __ldg(ap + j) : 0.f;
    }
  }
  const float x = (float)((const T*)p.x)[s * q.xs + d];
  const float st = sel_step((float)((const T*)p.dt)[s * q.dts + d], p.dt_bias ? __ldg(p.dt_bias + d) : 0.f, q.softplus);
  float y = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool ok = VEC || nl * 4 + j < q.N;
    const float b = ok ? (float)bp[j] : 0.f, c = ok ? (float)cp[j] : 0.f;
    h[j] = fmaf(ex2(st * (a[j] * LOG2E)), h[j], st * x * b);
    y = fmaf(c, h[j], y);
  }
  if (live) {
    if (VEC) *reinterpret_cast<float4*>(hp) = make_float4(h[0], h[1], h[2], h[3]);
    else
#pragma unroll
      for (int j = 0; j < 4; ++j) if (nl * 4 + j < q.N) hp[j] = h[j];
  }
#pragma unroll
  for (int o = LPC / 2; o; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
  if (live && nl == 0) {
    if (p.D) y = fmaf(__ldg(p.D + d), x, y);
    if (p.z) { const float z = (float)((const T*)p.z)[s * q.zs + d]; y *= z * sig(z); }
    stf((T*)p.y + s * q.ys + d, y);
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------
int lanes_for(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }
int chb_for(int lpc) { return lpc <= 8 ? 32 : 16; }
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
  int lpc, NP;
  size_t ckpt, segst, segdt, part_bc, part_par, fwd_bytes, bwd_bytes;   // offsets and totals
};

int make_sel_plan(const SsdSelDims* d, SelPlan* o) {
  if (!d) { set_error("selscan: dims is NULL"); return SSD_ERR_NULL_POINTER; }
  if (d->batch <= 0 || d->seqlen <= 0) { set_error("selscan: batch and seqlen must be positive (got %d %d)", d->batch, d->seqlen); return SSD_ERR_BAD_SHAPE; }
  const int rc = check_common("selscan", d->channels, d->dstate, d->ngroups, d->dtype, -1);
  if (rc) return rc;
  SelGeo& q = o->q;
  q.B = d->batch; q.L = d->seqlen; q.D = d->channels; q.N = d->dstate; q.G = d->ngroups; q.Dg = q.D / q.G;
  q.softplus = d->dt_softplus != 0;
  o->lpc = lanes_for(q.N); o->NP = 4 * o->lpc;
  q.nb = cdiv(q.Dg, chb_for(o->lpc));
  q.nt = cdiv(q.L, SEL_T);
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
  // Parts of the sequence (see below): one where the channel blocks of the batch fill the SMs.
  const long long n = (long long)q.B * q.G * q.nb;
  const int sms = 148;
  int segs = 1;
  if (n < sms) {
    segs = (int)((2LL * sms + n - 1) / n);
    if (segs > q.nt / 4) segs = q.nt / 4;
    if (segs < 3) segs = 1;
  }
  q.seg_len = cdiv(q.nt, segs) * SEL_T;
  q.segs = cdiv(q.L, q.seg_len);
  if (n * q.segs > 0x7fffffffLL) { set_error("selscan: too many blocks for one grid (%lld)", n * q.segs); return SSD_ERR_UNSUPPORTED; }
  const size_t st = (size_t)q.B * q.segs * q.D * sizeof(float);
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t r = at; at += up256(bytes); return r; };
  o->segst = take(st * o->NP); o->segdt = take(st);
  o->fwd_bytes = at + 256;
  o->ckpt = take((size_t)q.B * q.nt * q.D * o->NP * sizeof(float));
  o->part_bc = take((size_t)q.G * q.nb * q.B * q.L * 2 * o->NP * sizeof(float));
  o->part_par = take((size_t)q.B * q.segs * q.par_row * sizeof(float));
  o->bwd_bytes = at + 256;
  return SSD_OK;
}
int need_device(const SsdSelDims* d) { return check_common("selscan", d->channels, d->dstate, d->ngroups, d->dtype, d->device); }

#define SEL_LPC(F) \
  switch (lpc) { case 1: F(1); break; case 2: F(2); break; case 4: F(4); break; case 8: F(8); break; default: F(16); }

template <typename T> int sel_forward(const SelPlan& pl, const SelFwd& p, cudaStream_t s) {
  const SelGeo& q = pl.q;
  const int lpc = pl.lpc;
  const unsigned grid = (unsigned)((long long)q.B * q.segs * q.G * q.nb);
  if (q.segs > 1) {
#define SEL_RUN(LPC) launch<k_sel_fwd<T, LPC, 1>>(grid, Sh<LPC>::TH, 0, s, q, p)
    SEL_LPC(SEL_RUN)
#undef SEL_RUN
    SSD_CUDA_CHECK_LAUNCH("selscan_parts");
  }
#define SEL_RUN(LPC) launch<k_sel_fwd<T, LPC, 0>>(grid, Sh<LPC>::TH, 0, s, q, p)
  SEL_LPC(SEL_RUN)
#undef SEL_RUN
  SSD_CUDA_CHECK_LAUNCH("selscan_fwd");
  return SSD_OK;
}

template <typename T> int sel_backward(const SelPlan& pl, const SelBwd& p, const SsdSelBwdPtrs& u, cudaStream_t s) {
  const SelGeo& q = pl.q;
  const int lpc = pl.lpc;
  const unsigned grid = (unsigned)((long long)q.B * q.segs * q.G * q.nb);
  if (q.segs > 1) {
#define SEL_RUN(LPC) launch<k_sel_bwd_part<T, LPC>>(grid, Sh<LPC>::TH, 0, s, q, p)
    SEL_LPC(SEL_RUN)
#undef SEL_RUN
    SSD_CUDA_CHECK_LAUNCH("selscan_bwd_parts");
  }
#define SEL_RUN(LPC) do { \
    if (p.z) launch<k_sel_bwd<T, LPC, true>>(grid, Sh<LPC>::TH, Sh<LPC>::BWD_SMEM, s, q, p); \
    else launch<k_sel_bwd<T, LPC, false>>(grid, Sh<LPC>::TH, Sh<LPC>::BWD_SMEM, s, q, p); } while (0)
  SEL_LPC(SEL_RUN)
#undef SEL_RUN
  SSD_CUDA_CHECK_LAUNCH("selscan_bwd");
  const long long nbc = (long long)q.B * q.L * q.G * 2 * pl.NP;
  const long long most = (long long)sm_count() * 16;
  launch<k_sel_sum_bc<T>>((unsigned)((nbc + 255) / 256 < most ? (nbc + 255) / 256 : most), 256, 0, s, q, pl.NP, p.part_bc, (T*)u.dB, (T*)u.dC);
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
  const int lpc = lanes_for(q.N);
  const long long blocks = ((long long)q.S * q.D * lpc + 255) / 256;
  if (blocks > 0x7fffffffLL) { set_error("selscan step: too many blocks for one grid (%lld)", blocks); return SSD_ERR_UNSUPPORTED; }
  const bool vec = q.N == 4 * lpc && (((uintptr_t)p->state | (uintptr_t)p->A) & 15) == 0;
  cudaStream_t s = (cudaStream_t)cuda_stream;
#define SEL_RUN(LPC) do { \
    if (d->dtype == SSD_BF16) { if (vec) launch<k_sel_step<__nv_bfloat16, LPC, true>>((unsigned)blocks, 256, 0, s, q, *p); \
                                else launch<k_sel_step<__nv_bfloat16, LPC, false>>((unsigned)blocks, 256, 0, s, q, *p); } \
    else { if (vec) launch<k_sel_step<float, LPC, true>>((unsigned)blocks, 256, 0, s, q, *p); \
           else launch<k_sel_step<float, LPC, false>>((unsigned)blocks, 256, 0, s, q, *p); } } while (0)
  SEL_LPC(SEL_RUN)
#undef SEL_RUN
  SSD_CUDA_CHECK_LAUNCH("selscan_step");
  return SSD_OK;
}

}  // extern "C"
