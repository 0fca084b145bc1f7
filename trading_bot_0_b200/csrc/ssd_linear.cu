// A layer's projection with its epilogue:  out = act(x W^T + bias) + residual, and its gradients.
//
// k_mm2: bf16 on the tensor cores, pairs of CTAs on tiles of 256 x up to 256.
// k_mm: the general form, any sizes, strides and both storage types, fp32 products and sums on the CUDA cores.
#include <type_traits>

#include "act.cuh"
#include "common.cuh"
#include "ssd_internal.h"
#include "umma.cuh"

namespace ssd {
namespace {

__device__ __forceinline__ float relu(float v) { return v < 0.f ? 0.f : v; }   // (fmaxf would turn NaN into 0)
// The sigmoids' relative error is (4 + 1.2 |v|) 2^-23: 1e-6 at 5; 3e-6 at -20, where silu is 4e-8.
__device__ __forceinline__ float act_of(float v, int act) {
  if (act == SSD_ACT_SILU) return v * __fdividef(1.f, 1.f + __expf(-v));
  if (act == SSD_ACT_SOFTPLUS) return softplusf_(v);
  if (act == SSD_ACT_RELU2) { const float r = relu(v); return r * r; }
  return v;
}
__device__ __forceinline__ float dact_of(float v, int act) {
  if (act == SSD_ACT_SILU) { const float s = __fdividef(1.f, 1.f + __expf(-v)); return s * fmaf(v, 1.f - s, 1.f); }
  if (act == SSD_ACT_SOFTPLUS) return __fdividef(1.f, 1.f + __expf(-v));
  if (act == SSD_ACT_RELU2) return 2.f * relu(v);
  return 1.f;
}

// Values of a 16-byte piece (or a single one) as it lies in memory.
template <typename T> __device__ __forceinline__ void values_of(const T& r, float (&v)[1]) { v[0] = (float)r; }
__device__ __forceinline__ void values_of(const uint4& r, float (&v)[4]) {
  v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
}
__device__ __forceinline__ void values_of(const uint4& r, float (&v)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 f = umma::unpack_bf16(w[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
}
__device__ __forceinline__ void load_floats(const float* p, float (&v)[1]) { v[0] = *p; }
template <int V> __device__ __forceinline__ void load_floats(const float* p, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V / 4; ++i) *reinterpret_cast<float4*>(v + 4 * i) = *reinterpret_cast<const float4*>(p + 4 * i);
}
template <typename T> __device__ __forceinline__ void put_values(T* p, const float (&v)[1]) { stf(p, v[0]); }
__device__ __forceinline__ void put_values(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void put_values(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(umma::pack_bf16(v[0], v[1]), umma::pack_bf16(v[2], v[3]), umma::pack_bf16(v[4], v[5]), umma::pack_bf16(v[6], v[7]));
}

// out[m][n] = epilogue(sum_k P(m,k) Q(n,k)); element strides of P and Q along both dims.
struct MmArgs {
  const void *P, *Q, *bias, *residual;
  void* out;
  float* pre;
  long long M, N, K, psm, psk, qsn, qsk, os, rs;
  int act, splits;
  long long kper;
  float* part;                                      // splits > 1: [splits][M][N] sums, finished by k_join
  int* status;                                      // first kernel of a call: the workspace's status word, to be cleared; else null
};
// The status word is cleared once per call, by its first kernel (whichever path that is), and only ever set after that.
__device__ __forceinline__ void clear_status(int* status) {
  if (status && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0 && threadIdx.y == 0) *status = 0;
}
template <typename T> __device__ __forceinline__ void finish(const MmArgs& a, long long m, long long n, float v) {
  if (a.bias) v += ldf((const T*)a.bias + n);
  if (a.pre) a.pre[m * a.N + n] = v;
  v = act_of(v, a.act);
  if (a.residual) v += ldf((const T*)a.residual + m * a.rs + n);
  stf((T*)a.out + m * a.os + n, v);
}

// Block = 16 TM x 16 TM outputs, thread = TM x TM of them as packed pairs; 32 k at a time through shared memory, the next 32 in
// registers meanwhile.  Eight k by four rows per warp and request where k runs along memory: whole sectors, and no two lanes of a
// store on one bank.
template <typename T, int TM>
__global__ void __launch_bounds__(256) k_mm(MmArgs a) {
  constexpr int BM = 16 * TM, BK = 32, LD = BM + 4, IT = BM * BK / 256;
  __shared__ __align__(16) float sp[BK][LD], sq[BK][LD];
  pdl_wait();
  clear_status(a.status);
  const int tid = threadIdx.x, tm = tid / 16, tn = tid % 16;
  const long long nn = (a.N + BM - 1) / BM, nm = (a.M + BM - 1) / BM;
  const long long tile = blockIdx.x % (nn * nm), sp_i = blockIdx.x / (nn * nm);
  const long long m0 = tile / nn * BM, n0 = tile % nn * BM, kb = sp_i * a.kper, ke = min(kb + a.kper, a.K);
  const T *P = (const T*)a.P, *Q = (const T*)a.Q;
  auto where = [&](bool along_k, int i, int& k, int& r) {
    const int e = tid + i * 256;
    if (along_k) { const int w = e >> 5, l = e & 31; k = (w & 3) * 8 + (l & 7); r = (w >> 2) * 4 + (l >> 3); }
    else { k = e / BM; r = e % BM; }
  };
  const bool pk = a.psk == 1, qk = a.qsk == 1;
  // a thread's values of a block of k, as addresses that step by 32 k (rows past the end stand on the last one)
  const T *pp[IT], *qp[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    int k, r;
    where(pk, i, k, r);
    pp[i] = P + min(m0 + r, a.M - 1) * a.psm + (kb + k) * a.psk;
    where(qk, i, k, r);
    qp[i] = Q + min(n0 + r, a.N - 1) * a.qsn + (kb + k) * a.qsk;
  }
  const long long pstep = BK * a.psk, qstep = BK * a.qsk;
  float rp[IT], rq[IT];
  auto request = [&](int left) {                     // `left`: k from here to the end of the split
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      int k, r;
      where(pk, i, k, r);
      rp[i] = k < left ? ldf(pp[i]) : 0.f;
      pp[i] += pstep;
      where(qk, i, k, r);
      rq[i] = k < left ? ldf(qp[i]) : 0.f;
      qp[i] += qstep;
    }
  };
  f32x2 acc[TM][TM / 2] = {};
  request((int)min(ke - kb, (long long)BK));
  for (long long k0 = kb; k0 < ke; k0 += BK) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      int k, r;
      where(pk, i, k, r); sp[k][r] = rp[i];
      where(qk, i, k, r); sq[k][r] = rq[i];
    }
    __syncthreads();
    if (k0 + BK < ke) request((int)min(ke - k0 - BK, (long long)BK));
#pragma unroll 8
    for (int k = 0; k < BK; ++k) {
      float x[TM];
      f32x2 y[TM / 2];
#pragma unroll
      for (int h = 0; h < TM / 4; ++h) {
        const float4 v = *reinterpret_cast<const float4*>(&sp[k][h * 64 + tm * 4]), w = *reinterpret_cast<const float4*>(&sq[k][h * 64 + tn * 4]);
        x[4 * h] = v.x; x[4 * h + 1] = v.y; x[4 * h + 2] = v.z; x[4 * h + 3] = v.w;
        y[2 * h] = pack2(w.x, w.y); y[2 * h + 1] = pack2(w.z, w.w);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const f32x2 xx = pack2(x[i], x[i]);
#pragma unroll
        for (int j = 0; j < TM / 2; ++j) acc[i][j] = fma2(xx, y[j], acc[i][j]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const long long m = m0 + (i / 4) * 64 + tm * 4 + i % 4;
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const long long n = n0 + (j / 4) * 64 + tn * 4 + j % 4;
      if (n >= a.N) continue;
      float lo, hi;
      unpack2(acc[i][j / 2], lo, hi);
      const float v = j % 2 ? hi : lo;
      if (a.splits > 1) a.part[(sp_i * a.M + m) * a.N + n] = v;
      else finish<T>(a, m, n, v);
    }
  }
}
// The splits' sums in order, then the epilogue.  Thread = one value; neighbouring threads neighbouring columns.
template <typename T>
__global__ void __launch_bounds__(256) k_join(MmArgs a) {
  pdl_wait();
  const long long n = a.M * a.N;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    float v = 0.f;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) v += a.part[s * n + i];
    const long long m = i / a.N;
    finish<T>(a, m, i - m * a.N, v);
  }
}

// Few rows (up to eight tokens): bound by one reading of the weights and, below some megabytes, by latency, so one launch and every
// load of a weight row in flight at once.  Warp = F output features and all tokens, lane = 16 bytes of k at a time; x comes out of
// the L1, F features share a reading of it.  4 x 1536 x 768: 5.5 us, a launch and one latency.
template <typename T, int RM, int F>
__global__ void __launch_bounds__(256) k_mm_few(MmArgs a) {
  constexpr int V = 16 / (int)sizeof(T);
  pdl_wait();
  clear_status(a.status);
  const int lane = threadIdx.x & 31;
  const long long n0 = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * F;
  if (n0 >= a.N) return;
  const T *P = (const T*)a.P, *Q = (const T*)a.Q;
  float acc[F][RM] = {};
#pragma unroll (RM * F > 8 ? 2 : 4)
  for (long long k = lane * V; k < a.K; k += 32 * V) {
    float w[F][V], x[V];
#pragma unroll
    for (int f = 0; f < F; ++f) values_of(__ldg(reinterpret_cast<const uint4*>(Q + min(n0 + f, a.N - 1) * a.qsn + k)), w[f]);
#pragma unroll
    for (int m = 0; m < RM; ++m) {
      values_of(__ldg(reinterpret_cast<const uint4*>(P + min((long long)m, a.M - 1) * a.psm + k)), x);
#pragma unroll
      for (int f = 0; f < F; ++f)
#pragma unroll
        for (int v = 0; v < V; ++v) acc[f][m] = fmaf(x[v], w[f][v], acc[f][m]);
    }
  }
#pragma unroll
  for (int f = 0; f < F; ++f) {
    int m;
    const float v = fold_rows<32, RM>(acc[f], lane, m);
    if ((lane & (32 / RM - 1)) == 0 && m < a.M && n0 + f < a.N) finish<T>(a, m, n0 + f, v);
  }
}

// ---------------------------------------------------------------------------------------------
// out[m][n] = epilogue(sum_k P(m,k) Q(n,k)) for bf16 operands that a tensor map can describe.
//
// A pair of CTAs computes tiles of 256 x bn: every CTA loads 128 rows of P and bn/2 rows of Q per block of 64 k (32 KB at bn = 256,
// where a CTA on its own would load 48 KB for the same work per SM).  Warp 0 of each CTA issues the loads (five stages), warp 1 of the
// leader the MMAs, eight warps per CTA read the accumulators (two of them in TMEM, so that a tile's epilogue runs beside the next
// tile's products).  Pairs walk the units (split of k, tile row, tile column) with a fixed stride; with splits > 1 a unit leaves fp32
// sums in the workspace and k_mm2_join adds them in order.  Every wait is bounded: when one runs out a code goes to the status word, the
// outputs become NaN, and a later product of the same call waits for nothing and gives NaN.
//
// Measured with cuBLAS beside it in one run, bare calls after an L2 flush (one after the other, as a layer makes them, the second takes 86
// to 89): 8192^3 694 us = 1.58 PFLOP/s (647), 16384 x 768 x 3352 76 (72), 4096 x 2048 x 2048 45 (41),
// 512 x 768 x 1536 14 (8).  8192^3 before and after on one board: 785 us with loads and MMAs issued by `lane == 0`, 677 by an elected
// lane, whatever the tile's width; four stages are as fast as five, three 10 % slower;
// both accumulators as one tile of 256 x 512, which loads a quarter less, 670 us, but 103 against 77 us at 16384 x 768 x 3352, where
// its epilogue is not hidden.
namespace u = umma;
constexpr int MM_BM = 256, MM_EPI = 8, MM_THREADS = 32 * (4 + MM_EPI);
constexpr int MM_SLOT = 4096;                      // output staging of a warp: a box of 32 x 32 fp32, or two of bf16
constexpr int MM_ROWS = 8;                         // tile rows walked side by side: the pairs at work share operands in the L2
constexpr int MM_STAGES = 5, MM_STAGE = 32768;      // 128 rows of P, up to 128 of Q
constexpr size_t MM_SMEM = (size_t)MM_STAGES * MM_STAGE + MM_EPI * MM_SLOT + 1024;

struct Mm2 {
  long long M, N;                                  // of the tiles: rows of P, rows of Q
  int kb, kper, splits, bn, rt, ct, units;         // blocks of 64 k, per split; tile rows and columns
  int trans;                                       // the tiles' rows are the output's columns (few tokens: the weights are P)
  int act, vec;                                    // vec: tensor maps fit out, pre and residual (with splits: the sums)
  long long os, rs;
  const __nv_bfloat16 *bias, *residual;
  __nv_bfloat16* out;
  float *pre, *part;                                     // [splits][out rows][out columns]
  int* status;
  int first;                                       // the call's first kernel: clears the status word
};

// unit -> split, tile row, tile column; columns of a group of MM_ROWS tile rows one after the other
__device__ __forceinline__ void unit_at(const Mm2& a, int un, int& sp, int& r, int& c) {
  const int tiles = a.rt * a.ct;
  sp = un / tiles;
  const int t = un - sp * tiles, g = t / (MM_ROWS * a.ct), r0 = g * MM_ROWS, n = min(MM_ROWS, a.rt - r0), w = t - g * MM_ROWS * a.ct;
  c = w / n; r = r0 + w - c * n;
}
// One value of the result at output row m and column n.
__device__ __forceinline__ void finish_one(const Mm2& a, long long cols, long long m, long long n, float v) {
  if (a.bias) v += __bfloat162float(a.bias[n]);
  if (a.pre) a.pre[m * cols + n] = v;
  v = act_of(v, a.act);
  if (a.residual) v += __bfloat162float(a.residual[m * a.rs + n]);
  a.out[m * a.os + n] = __float2bfloat16_rn(v);
}

// Output through shared memory and TMA stores (a thread holds a row: stored from registers, the lanes of a warp write 16 or 32 bytes
// each at the rows' distance, 2.3 times the tensor cores' time at 16384 x 768 x 3352).
__device__ __forceinline__ void stage_bf16(uint32_t box, int lane, const float (&v)[32]) {   // 64-byte rows, 64-byte swizzle
#pragma unroll
  for (int i = 0; i < 4; ++i)
    u::st_shared_v4(box + lane * 64 + ((i ^ (lane >> 1)) & 3) * 16, u::pack_bf16(v[8 * i], v[8 * i + 1]), u::pack_bf16(v[8 * i + 2], v[8 * i + 3]),
                    u::pack_bf16(v[8 * i + 4], v[8 * i + 5]), u::pack_bf16(v[8 * i + 6], v[8 * i + 7]));
}
__device__ __forceinline__ void stage_f32(uint32_t box, int lane, const float (&v)[32]) {    // 128-byte rows, 128-byte swizzle
#pragma unroll
  for (int i = 0; i < 8; ++i)
    u::st_shared_v4(box + lane * 128 + ((i ^ lane) & 7) * 16, __float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                    __float_as_uint(v[4 * i + 3]));
}

template <bool PMN, bool QMN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MM_THREADS, 1)
k_mm2(const __grid_constant__ CUtensorMap tp, const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tout,
      const __grid_constant__ CUtensorMap tpre, const __grid_constant__ Mm2 a) {
  extern __shared__ unsigned char mm_raw[];
  __shared__ __align__(8) uint64_t full[MM_STAGES], empty[MM_STAGES], tfull[2], tempty[2];
  __shared__ uint32_t slot;
  __shared__ int dead;
  __shared__ __align__(16) __nv_bfloat16 s_bias[2][256];
  unsigned char* st = mm_raw + (1024 - (u::smem_u32(mm_raw) & 1023)) % 1024;   // the same offset in both CTAs
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = u::cluster_rank();
  if (tid == 0) {
    dead = 0;
    for (int i = 0; i < MM_STAGES; ++i) { u::mbar_init(&full[i], 1); u::mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { u::mbar_init(&tfull[i], 1); u::mbar_init(&tempty[i], 2 * MM_EPI); }
    u::mbar_fence_init();
  }
  if (warp == 2) u::tmem_alloc_pair(&slot, 512);
  u::tc_fence_before();
  __syncthreads();
  u::cluster_sync();
  u::tc_fence_after();
  const uint32_t tmem = slot;
  pdl_wait();
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  volatile int* is_dead = &dead;
  if (a.first) clear_status(a.status);
  else if (*(volatile int*)a.status) *is_dead = 1;   // an earlier kernel gave up
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    if (*is_dead) return false;
    if (u::mbar_wait(bar, parity)) return true;
    *is_dead = 1;
    *a.status = code;
    return false;
  };
  auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) { return __all_sync(0xffffffffu, wait(bar, parity, code)) != 0; };   // a warp goes on or gives up as one
  const int half = a.bn / 2;
  if (warp == 0) {
    const int qbox = QMN ? (half + 63) / 64 : 1;
    const uint32_t bytes = 2u * (16384u + (QMN ? qbox * 8192u : half * 128u));
    int s = 0;
    uint32_t ph = 1;
    bool ok = true;
    for (int un = pair; un < a.units && ok; un += npairs) {
      int sp, r, c;
      unit_at(a, un, sp, r, c);
      const int k0 = sp * a.kper, k1 = min(k0 + a.kper, a.kb);
      const int prow = r * MM_BM + (int)rank * 128, qrow = c * a.bn + (int)rank * half;
      for (int k = k0; k < k1; ++k) {
        if (!(ok = wait_all(&empty[s], ph, 201))) break;
        if (u::elect_one()) {
          unsigned char* sa = st + s * MM_STAGE;
          unsigned char* sb = sa + 16384;
          if (rank == 0) u::mbar_expect_tx(&full[s], bytes);
          const uint32_t bar = u::map_rank(&full[s], 0);
          if (PMN) {
            u::tma_load_2d_pair(sa, &tp, prow, k * 64, bar);
            u::tma_load_2d_pair(sa + 8192, &tp, prow + 64, k * 64, bar);
          } else {
            u::tma_load_2d_pair(sa, &tp, k * 64, prow, bar);
          }
          if (QMN) {
            for (int j = 0; j < qbox; ++j) u::tma_load_2d_pair(sb + j * 8192, &tq, qrow + j * 64, k * 64, bar);
          } else {
            u::tma_load_2d_pair(sb, &tq, k * 64, qrow, bar);
          }
        }
        __syncwarp();
        if (++s == MM_STAGES) { s = 0; ph ^= 1; }
      }
    }
    if (!ok) {   // let copies in flight land before the shared memory goes back
      const long long t0 = clock64();
      while (clock64() - t0 < 4000000) {}
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = u::make_idesc(256, a.bn, PMN, QMN);
      int s = 0, buf = 0;
      uint32_t ph = 0, tph = 1;
      bool ok = true;
      for (int un = pair; un < a.units && ok; un += npairs) {
        const int sp = un / (a.ct * a.rt);
        const int k0 = sp * a.kper, k1 = min(k0 + a.kper, a.kb);
        if (!(ok = wait_all(&tempty[buf], tph, 202))) break;
        u::tc_fence_after();
        for (int k = k0; k < k1; ++k) {
          if (!(ok = wait_all(&full[s], ph, 203))) break;
          u::tc_fence_after();
          if (u::elect_one()) {
            const uint32_t sa = u::smem_u32(st + s * MM_STAGE), sb = sa + 16384;
            const uint64_t ad = PMN ? u::desc_sw128_mn(sa, 0, 0, 8192) : u::desc_sw128_k(sa, 0);
            const uint64_t bd = QMN ? u::desc_sw128_mn(sb, 0, 0, 8192) : u::desc_sw128_k(sb, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              u::mma_bf16_pair(tmem + buf * 256, u::desc_adv(ad, i * (PMN ? 2048 : 32)), u::desc_adv(bd, i * (QMN ? 2048 : 32)), idesc, k > k0 || i > 0);
            u::mma_commit_pair(&empty[s]);
          }
          __syncwarp();
          if (++s == MM_STAGES) { s = 0; ph ^= 1; }
        }
        if (!ok) break;
        if (u::elect_one()) u::mma_commit_pair(&tfull[buf]);
        __syncwarp();
        buf ^= 1;
        if (!buf) tph ^= 1;
      }
    }
  } else if (warp >= 4) {
    const int e = warp - 4, quad = warp & 3, grp = e >> 2;
    const uint32_t release = u::map_rank(&tempty[0], 0);    // (the second is 8 bytes on)
    unsigned char* const slot_p = st + MM_STAGES * MM_STAGE + e * MM_SLOT;
    const uint32_t slot_a = u::smem_u32(slot_p);
    int buf = 0, box = 0;
    uint32_t tph = 0;
    bool ok = true;
    for (int un = pair; un < a.units; un += npairs) {
      int sp, r, c;
      unit_at(a, un, sp, r, c);
      const int row0 = r * MM_BM + (int)rank * 128 + quad * 32;
      const long long row = row0 + lane, n0 = (long long)c * a.bn;
      const int ncol = (int)min((long long)a.bn, a.N - n0);
      const bool live = row < a.M, direct = !a.trans && a.splits == 1;
      uint4 q[4];
      auto ask = [&](int j) {                        // residual of the columns j .. j+31, asked for a chunk ahead
        const __nv_bfloat16* p = a.residual + row * a.rs + n0 + j;
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = live && j + 8 * i < ncol ? __ldg(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0, 0, 0, 0);
      };
      const bool res = direct && a.vec && a.residual;
      if (res) ask(grp * 32);
      if (direct) {
        for (int i = tid - 128; i < 256; i += 32 * MM_EPI) s_bias[buf][i] = a.bias && i < ncol ? a.bias[n0 + i] : __nv_bfloat16(0.f);
        asm volatile("bar.sync 1, %0;" ::"n"(32 * MM_EPI) : "memory");
      }
      ok = ok && wait(&tfull[buf], tph, 204);
      u::tc_fence_after();
      for (int j = grp * 32; j < ncol; j += 64) {
        float v[32];
        u::tmem_ld32(u::tmem_addr(tmem + buf * 256, quad * 32, j), v);
        const int nv = min(32, ncol - j);
        if (!ok)
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __int_as_float(0x7fc00000);
        if (a.splits > 1) {
          if (a.vec) {
            if (lane == 0) u::bulk_wait_read0();
            __syncwarp();
            stage_f32(slot_a, lane, v);
            u::fence_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < a.M) { u::tma_store_3d(&tout, slot_p, (int)n0 + j, row0, sp); u::bulk_commit(); }
          } else if (live && a.trans) {
            float* p = a.part + ((long long)sp * a.N + n0 + j) * a.M + row;
#pragma unroll
            for (int i = 0; i < 32; ++i) if (i < nv) p[i * a.M] = v[i];
          } else if (live) {
            float* p = a.part + ((long long)sp * a.M + row) * a.N + n0 + j;
#pragma unroll
            for (int i = 0; i < 32; ++i) if (i < nv) p[i] = v[i];
          }
          continue;
        }
        if (a.trans || !a.vec) {
          if (live)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < nv) { if (a.trans) finish_one(a, a.M, n0 + j + i, row, v[i]); else finish_one(a, a.N, row, n0 + j + i, v[i]); }
          continue;
        }
        const uint4 h[4] = {q[0], q[1], q[2], q[3]};
        if (res && j + 64 < ncol) ask(j + 64);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint2 w = *reinterpret_cast<const uint2*>(&s_bias[buf][j + 4 * i]);
          const float2 b = u::unpack_bf16(w.x), e2 = u::unpack_bf16(w.y);
          v[4 * i] += b.x; v[4 * i + 1] += b.y; v[4 * i + 2] += e2.x; v[4 * i + 3] += e2.y;
        }
        auto put = [&](const CUtensorMap* map, int at, bool f32) {   // out alone: two boxes in turn, the older store has read its box
          if (lane == 0) { if (a.pre) u::bulk_wait_read0(); else asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }
          __syncwarp();
          if (f32) stage_f32(slot_a + at, lane, v); else stage_bf16(slot_a + at, lane, v);
          u::fence_async_smem();
          __syncwarp();
          if (lane == 0 && row0 < a.M) { u::tma_store_3d(map, slot_p + at, (int)n0 + j, row0, 0); u::bulk_commit(); }
        };
        if (a.pre) put(&tpre, 0, true);
        if (a.act == SSD_ACT_SILU) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = act_of(v[i], SSD_ACT_SILU);
        } else if (a.act == SSD_ACT_SOFTPLUS) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = act_of(v[i], SSD_ACT_SOFTPLUS);
        } else if (a.act == SSD_ACT_RELU2) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = act_of(v[i], SSD_ACT_RELU2);
        }
        if (res) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t w[4] = {h[i].x, h[i].y, h[i].z, h[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 f = u::unpack_bf16(w[k]);
              v[8 * i + 2 * k] += f.x; v[8 * i + 2 * k + 1] += f.y;
            }
          }
        }
        put(&tout, a.pre ? 0 : box * 2048, false);
        box ^= 1;
      }
      u::tc_fence_before();
      __syncwarp();
      if (lane == 0) u::mbar_arrive_remote(release + buf * 8);
      buf ^= 1;
      if (!buf) tph ^= 1;
    }
    if (lane == 0) u::bulk_wait0();
  }
  __syncwarp();
  __syncthreads();
  u::cluster_sync();
  u::tc_fence_after();
  if (warp == 2) u::tmem_dealloc_pair(tmem, 512);
}

// The splits' sums in order, then the epilogue.  Thread = V values of a row (four where rows of sums and of out start on 16 and 8 bytes).
template <int V>
__global__ void __launch_bounds__(256) k_mm2_join(Mm2 a, long long rows, int cols) {
  pdl_wait();
  const long long n = rows * cols;
  const int pieces = cols / V;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * pieces; i += (long long)gridDim.x * 256) {
    const long long m = i / pieces;
    const int c = (int)(i - m * pieces) * V;
    float v[V] = {};
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) {
      float f[V];
      load_floats(a.part + s * n + m * cols + c, f);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] += f[k];
    }
    if (V == 4 && !a.pre && !a.residual) {
      if (a.bias)
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] += __bfloat162float(a.bias[c + k]);
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = act_of(v[k], a.act);
      *reinterpret_cast<uint2*>(a.out + m * a.os + c) = make_uint2(u::pack_bf16(v[0], v[V > 1 ? 1 : 0]), u::pack_bf16(v[V > 2 ? 2 : 0], v[V > 3 ? 3 : 0]));
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) finish_one(a, cols, m, c + k, v[k]);
    }
  }
}

// dpre = dout act'(pre), rounded to the storage type, and the column sums of the unrounded dpre over a
// part of the rows (`parts` of them on the y axis).  Thread = V neighbouring columns, block = 32 V columns x 8 rows at a time, four
// rows of a thread requested together.  V = 16 bytes where all rows start on 16 bytes, else one value.
// The rounding is what bf16 operands of the two products mean: dx and dweight carry it beside the rounding of the result, each 0.0017 rms of
// the gradient, 0.0023 to 0.0024 together (16384 x 1536 x 768).  Without it dpre would be two bf16 parts and both products twice as long
// (43 us each there).  fp32 storage rounds nothing here.
template <typename T, int V>
__global__ void __launch_bounds__(256) k_dpre(long long M, int N, int act, const T* __restrict__ dout, long long dos, const float* __restrict__ pre,
                                              T* __restrict__ dpre, float* __restrict__ partial, int* status) {
  __shared__ float s[8][32 * V];
  pdl_wait();
  clear_status(status);
  typedef typename std::conditional<V == 1, T, uint4>::type Raw;   // V values as they lie in memory
  constexpr int R = 4;
  const int n = (blockIdx.x * 32 + threadIdx.x) * V;
  const long long per = (M + gridDim.y - 1) / gridDim.y, lo = per * blockIdx.y, hi = min(lo + per, M);
  float a[V] = {};
  if (n < N) {
    for (long long m = lo + threadIdx.y; m < hi; m += 8 * R) {
      Raw g[R];
      float q[R][V], t[V] = {};
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (m + 8 * r < hi) {
          g[r] = *reinterpret_cast<const Raw*>(dout + (m + 8 * r) * dos + n);
          if (act) load_floats(pre + (m + 8 * r) * N + n, q[r]);
        }
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (m + 8 * r < hi) {
          float x[V];
          values_of(g[r], x);
          if (act)
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] *= dact_of(q[r][j], act);
#pragma unroll
          for (int j = 0; j < V; ++j) t[j] += x[j];
          if (dpre) put_values(dpre + (m + 8 * r) * N + n, x);
        }
#pragma unroll
      for (int j = 0; j < V; ++j) a[j] += t[j];
    }
  }
  if (!partial) return;
#pragma unroll
  for (int j = 0; j < V; ++j) s[threadIdx.y][threadIdx.x * V + j] = a[j];
  __syncthreads();
  for (int i = threadIdx.y * 32 + threadIdx.x; i < 32 * V; i += 256) {
    const int col = blockIdx.x * 32 * V + i;
    if (col >= N) break;
    float b = s[0][i];
#pragma unroll
    for (int k = 1; k < 8; ++k) b += s[k][i];
    partial[(long long)blockIdx.y * N + col] = b;
  }
}
template <typename T>
__global__ void __launch_bounds__(1024) k_dbias(int N, int parts, const float* __restrict__ partial, T* __restrict__ dbias) {
  __shared__ float s[32][33];
  pdl_wait();
  const int n = blockIdx.x * 32 + threadIdx.x;
  float a = 0.f;
  if (n < N)
    for (int p = threadIdx.y; p < parts; p += 32) a += partial[(long long)p * N + n];
  s[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.y || n >= N) return;
#pragma unroll
  for (int k = 1; k < 32; ++k) a += s[k][threadIdx.x];
  stf(dbias + n, a);
}

// ---- tensor-core products: shape of the tiles and the launch ------------------------------------------------------------
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn get_encode() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
               ? (EncodeFn)p : nullptr;
  }();
  return fn;
}
// [rows, cols] bf16, rows `stride` elements apart; box = 64 columns x `box` rows, 128-byte swizzle
int make_map2(CUtensorMap* m, const void* p, long long rows, long long cols, long long stride, int box, const char* what) {
  EncodeFn enc = get_encode();
  if (!enc) { set_error("cuTensorMapEncodeTiled is not available from the driver"); return SSD_ERR_CUDA; }
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride * 2};
  const cuuint32_t b[2] = {64, (cuuint32_t)box}, es[2] = {1, 1};
  const CUresult r = u::in_context([&] {
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), dims, strides, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
  if (r != CUDA_SUCCESS) { set_error("cuTensorMapEncodeTiled(%s) failed with CUresult %d", what, (int)r); return SSD_ERR_CUDA; }
  return SSD_OK;
}
// output boxes of 32 x 32: [rows, cols] bf16, or the splits' sums [splits, rows, cols] fp32
int make_out_map(CUtensorMap* m, const void* p, bool f32, long long splits, long long rows, long long cols, long long stride, const char* what) {
  EncodeFn enc = get_encode();
  if (!enc) { set_error("cuTensorMapEncodeTiled is not available from the driver"); return SSD_ERR_CUDA; }
  const int es = f32 ? 4 : 2;
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)splits};
  const cuuint64_t strides[2] = {(cuuint64_t)stride * es, (cuuint64_t)stride * rows * es};
  const cuuint32_t b[3] = {32, 32, 1}, one[3] = {1, 1, 1};
  const CUresult r = u::in_context([&] {
    return enc(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, b, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
  if (r != CUDA_SUCCESS) { set_error("cuTensorMapEncodeTiled(%s, output) failed with CUresult %d", what, (int)r); return SSD_ERR_CUDA; }
  return SSD_OK;
}
bool map_fits(const void* p, long long rows, long long stride) {
  return ((uintptr_t)p & 15) == 0 && stride % 8 == 0 && rows <= 0x7fffffffLL && stride < (1LL << 38);
}

// Shape of the tiles for an M x N product over K, estimated in SM clocks: a pair's block of 64 k takes 420 + 1.1 bn (measured at
// bn 64 to 256); 2500 to fill the pipeline and empty the last accumulator; split sums are written and read, mostly in the L2, and cost a
// launch.  With `may_trans` the weights may be the tiles' rows (few tokens).
struct TileShape { int trans, bn, splits, kper; long long rt, ct; double cost; };
TileShape find_tiles(long long M, long long N, long long K, bool may_trans) {
  const int pairs = 74, kb = (int)((K + 63) / 64);
  TileShape best{0, 0, 0, 0, 0, 0, 1e30};
  for (int trans = 0; trans <= (may_trans && M <= 128 ? 1 : 0); ++trans) {   // (beyond that its stores, a value at a time, show)
    const long long R = trans ? N : M, C = trans ? M : N;
    const long long rt = (R + MM_BM - 1) / MM_BM;
    for (int bn = 32; bn <= 256; bn += 32) {     // what an MMA of a pair takes
      if (bn > 32 && bn - 32 >= C) break;
      const long long ct = (C + bn - 1) / bn;
      const double tk = 420.0 + 1.1 * bn;
      for (int s = 1; s <= 32 && s <= kb; ++s) {
        const int kper = (kb + s - 1) / s;
        if ((kb + kper - 1) / kper != s) continue;
        const double units = (double)rt * ct * s, waves = (double)(long long)((units + pairs - 1) / pairs);
        const double cost = waves * (kper * tk + 200.0) + 2500.0 + (s > 1 ? 4000.0 + 8.0 * s * M * N / 6000.0 : 0.0);
        if (cost < best.cost) best = TileShape{trans, bn, s, kper, rt, ct, cost};
      }
    }
  }
  return best;
}
// The same for a size that this thread met before (the search takes some microseconds on the host).
TileShape choose_tiles(long long M, long long N, long long K, bool may_trans) {
  struct Entry { long long M, N, K; bool may_trans; TileShape t; };
  static thread_local Entry memo[64] = {};
  Entry& e = memo[(size_t)(M * 31 + N * 7 + K * 3 + may_trans) % 64];
  if (e.M != M || e.N != N || e.K != K || e.may_trans != may_trans) e = Entry{M, N, K, may_trans, find_tiles(M, N, K, may_trans)};
  return e.t;
}
size_t part_bytes(const TileShape& t, long long M, long long N) { return t.splits > 1 ? (size_t)t.splits * M * N * sizeof(float) : 0; }

// out [M,N] of P (rows M) and Q (rows N): pointer, whether its k runs along memory, and the stride of its memory rows.
struct Operand { const void* p; bool kmajor; long long stride; };
struct Result { __nv_bfloat16* out; float* pre; const __nv_bfloat16 *bias, *residual; long long os, rs; int act; };
int run_mm2(const char* what, const TileShape& t, Operand P, Operand Q, long long M, long long N, long long K, const Result& o, float* part,
            int* status, bool first, cudaStream_t s) {
  Mm2 a;
  if (t.trans) { const Operand x = P; P = Q; Q = x; }
  a.M = t.trans ? N : M; a.N = t.trans ? M : N;
  a.kb = (int)((K + 63) / 64); a.kper = t.kper; a.splits = t.splits; a.bn = t.bn; a.rt = (int)t.rt; a.ct = (int)t.ct;
  a.units = (int)(t.rt * t.ct * t.splits); a.trans = t.trans; a.act = o.act;
  a.os = o.os; a.rs = o.rs; a.bias = o.bias; a.residual = o.residual; a.out = o.out; a.pre = o.pre; a.part = part; a.status = status; a.first = first;
  if (t.splits > 1) a.vec = !t.trans && N % 4 == 0 && N < (1LL << 36) / M;
  else a.vec = !t.trans && N % 8 == 0 && (((uintptr_t)o.out | (uintptr_t)o.pre | (uintptr_t)o.residual) & 15) == 0 && o.os % 8 == 0 &&
               (!o.residual || o.rs % 8 == 0) && o.os < (1LL << 36) / M;
  CUtensorMap tp, tq, tout, tpre;
  int rc = P.kmajor ? make_map2(&tp, P.p, a.M, K, P.stride, 128, what) : make_map2(&tp, P.p, K, a.M, P.stride, 64, what);
  if (rc) return rc;
  rc = Q.kmajor ? make_map2(&tq, Q.p, a.N, K, Q.stride, t.bn / 2, what) : make_map2(&tq, Q.p, K, a.N, Q.stride, 64, what);
  if (rc) return rc;
  tout = tpre = tp;
  if (a.vec) {
    rc = t.splits > 1 ? make_out_map(&tout, part, true, t.splits, M, N, N, what) : make_out_map(&tout, o.out, false, 1, M, N, o.os, what);
    if (!rc && t.splits == 1 && o.pre) rc = make_out_map(&tpre, o.pre, true, 1, M, N, N, what);
    if (rc) return rc;
  }
  const int pairs = a.units < 74 ? a.units : 74;
#define MM2_RUN(A, B) launch<k_mm2<A, B>>(2 * pairs, MM_THREADS, MM_SMEM, s, tp, tq, tout, tpre, a)
  if (P.kmajor) { if (Q.kmajor) MM2_RUN(false, false); else MM2_RUN(false, true); }
  else { if (Q.kmajor) MM2_RUN(true, false); else MM2_RUN(true, true); }
#undef MM2_RUN
  SSD_CUDA_CHECK_LAUNCH(what);
  if (t.splits > 1) {
    const bool four = N % 4 == 0 && o.os % 4 == 0 && ((uintptr_t)o.out & 7) == 0;
    const long long n = (M * N / (four ? 4 : 1) + 255) / 256, most = (long long)sm_count() * 8;
    if (four) launch<k_mm2_join<4>>((unsigned)(n < most ? n : most), 256, 0, s, a, M, (int)N);
    else launch<k_mm2_join<1>>((unsigned)(n < most ? n : most), 256, 0, s, a, M, (int)N);
    SSD_CUDA_CHECK_LAUNCH("linear_join");
  }
  return SSD_OK;
}

// ---- CUDA-core products: tiles of 128 where they fill the SMs, else of 64, and splits of K where those do not either and the steps
// saved are worth the launch that joins the sums (about 0.4 us per 32 k against 4)
struct CoreShape { bool big; long long tiles, kper; int splits; };
CoreShape core_shape(long long M, long long N, long long K) {
  CoreShape c;
  const long long big = ((M + 127) / 128) * ((N + 127) / 128);
  c.big = big >= 148;
  c.tiles = c.big ? big : ((M + 63) / 64) * ((N + 63) / 64);
  const long long fit = c.tiles < 148 ? 2 * 148 / c.tiles : 1, steps = (K + 31) / 32;
  long long s = 1;
  double least = 0.4 * steps;
  for (long long t = 2; t <= fit && t <= steps; ++t) {
    const double cost = 0.4 * ((steps + t - 1) / t) + 4.0 + 0.02 * t;
    if (cost < least) { least = cost; s = t; }
  }
  c.kper = (steps + s - 1) / s * 32;
  c.splits = (int)((K + c.kper - 1) / c.kper);
  return c;
}
size_t core_bytes(long long M, long long N, long long K) {
  const CoreShape c = core_shape(M, N, K);
  return c.splits > 1 ? (size_t)c.splits * M * N * sizeof(float) : 0;
}

// ---- host --------------------------------------------------------------------------------------------------------------
size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
struct LinPlan {
  long long M, xs, os, rs;
  int K, N, act, es, parts;
  bool tc;                                          // bf16: products on the tensor cores where the operands' rows allow it
  TileShape fwd, tdx, tdw;
  size_t part_fwd, dpre, partial, part_bwd, fwd_bytes, bwd_bytes;   // a status word comes first in both workspaces
};
int make_lin_plan(const SsdLinearDims* d, int pass, LinPlan* o) {
  if (!d) { set_error("linear: dims is NULL"); return SSD_ERR_NULL_POINTER; }
  if (d->rows <= 0 || d->in_features <= 0 || d->out_features <= 0) {
    set_error("linear: rows, in_features and out_features must be positive (got %lld %d %d)", (long long)d->rows, d->in_features, d->out_features);
    return SSD_ERR_BAD_SHAPE;
  }
  if (d->dtype != SSD_F32 && d->dtype != SSD_BF16) { set_error("linear: unknown dtype %d", d->dtype); return SSD_ERR_UNSUPPORTED; }
  if (d->activation < SSD_ACT_NONE || d->activation > SSD_ACT_RELU2) { set_error("linear: unknown activation %d", d->activation); return SSD_ERR_UNSUPPORTED; }
  o->M = d->rows; o->K = d->in_features; o->N = d->out_features; o->act = d->activation; o->es = d->dtype == SSD_BF16 ? 2 : 4;
  o->xs = d->x_stride_row ? d->x_stride_row : o->K;
  o->os = d->out_stride_row ? d->out_stride_row : o->N;
  o->rs = d->residual_stride_row ? d->residual_stride_row : o->N;
  if (o->xs < o->K || o->os < o->N || o->rs < o->N) { set_error("linear: row strides must be at least the row size"); return SSD_ERR_BAD_SHAPE; }
  if (((o->M + 63) / 64) * (((o->N > o->K ? o->N : o->K) + 63LL) / 64) > 0x7fffffffLL) { set_error("linear: too many output tiles for one grid"); return SSD_ERR_UNSUPPORTED; }
  const long long cols = (o->N + 255) / 256, want = (8 * 148 + cols - 1) / cols, most = (o->M + 63) / 64;
  o->parts = (int)(want < most ? want : most);
  size_t at = 0;
  auto take = [&](size_t n) { const size_t r = at; at += up256(n); return r; };
  take(256);
  // split sums: the largest that any kernel of the pass may leave (operands decide on the kernel, the workspace is sized before)
  o->tc = d->dtype == SSD_BF16 && o->M <= 0x7fffff00LL;
  size_t join = 0;
  auto keep = [&](size_t v) { if (v > join) join = v; };
  if (pass == SSD_PASS_FWD) {
    keep(core_bytes(o->M, o->N, o->K));
    if (o->tc) { o->fwd = choose_tiles(o->M, o->N, o->K, true); keep(part_bytes(o->fwd, o->M, o->N)); }
  } else {
    keep(core_bytes(o->M, o->K, o->N));
    keep(core_bytes(o->N, o->K, o->M));
    if (o->tc) {
      o->tdx = choose_tiles(o->M, o->K, o->N, true);
      o->tdw = choose_tiles(o->N, o->K, o->M, false);
      keep(part_bytes(o->tdx, o->M, o->K));
      keep(part_bytes(o->tdw, o->N, o->K));
    }
  }
  o->part_fwd = at;
  o->fwd_bytes = at + up256(join) + 256;
  o->dpre = take(o->act ? (size_t)o->M * o->N * o->es : 0);
  o->partial = take((size_t)o->parts * o->N * sizeof(float));
  o->part_bwd = take(join);
  o->bwd_bytes = at + 256;
  return SSD_OK;
}
int check_device(const SsdLinearDims* d) {
  if (d->device < 0) return SSD_OK;
  int cur = -1;
  if (cudaGetDevice(&cur) != cudaSuccess || cur != d->device) {
    set_error("linear: current CUDA device is %d but dims.device is %d (the library never switches devices)", cur, d->device);
    return SSD_ERR_CUDA;
  }
  return SSD_OK;
}
char* aligned_base(void* ws) { return (char*)(((uintptr_t)ws + 255) & ~(uintptr_t)255); }

template <typename T> int run_mm(const char* what, const MmArgs& a, cudaStream_t s) {
  const CoreShape c = core_shape(a.M, a.N, a.K);
  MmArgs b = a;
  b.splits = c.splits; b.kper = c.kper;
  if (c.big) launch<k_mm<T, 8>>((unsigned)(c.tiles * c.splits), 256, 0, s, b);
  else launch<k_mm<T, 4>>((unsigned)(c.tiles * c.splits), 256, 0, s, b);
  SSD_CUDA_CHECK_LAUNCH(what);
  if (c.splits > 1) {
    const long long n = (a.M * a.N + 255) / 256, most = (long long)sm_count() * 8;
    launch<k_join<T>>((unsigned)(n < most ? n : most), 256, 0, s, b);
    SSD_CUDA_CHECK_LAUNCH("linear_join");
  }
  return SSD_OK;
}
constexpr int FEW = 8;
template <typename T> int run_few(const MmArgs& a, cudaStream_t s) {
  const int rm = a.M <= 1 ? 1 : a.M <= 2 ? 2 : a.M <= 4 ? 4 : 8;
  const bool two = a.N >= 8192;   // enough warps for the SMs with two features each
  const unsigned grid = (unsigned)((a.N + (two ? 16 : 8) - 1) / (two ? 16 : 8));
#define FEW_RUN(RM) do { if (two) launch<k_mm_few<T, RM, 2>>(grid, 256, 0, s, a); else launch<k_mm_few<T, RM, 1>>(grid, 256, 0, s, a); } while (0)
  if (rm == 1) FEW_RUN(1); else if (rm == 2) FEW_RUN(2); else if (rm == 4) FEW_RUN(4); else FEW_RUN(8);
#undef FEW_RUN
  SSD_CUDA_CHECK_LAUNCH("linear_few");
  return SSD_OK;
}

template <typename T>
int linear_backward(const LinPlan& p, const void* x, const void* w, const void* pre, const void* dout, long long dos, void* dx, void* dw,
                    void* db, char* ws, int* status, cudaStream_t s) {
  const bool need_dpre = p.act && (dx || dw);
  bool first = true;                                  // no kernel of this call has cleared the status word yet
  if (!dx && !dw && !db) {
    const cudaError_t e = cudaMemsetAsync(status, 0, sizeof(int), s);
    if (e != cudaSuccess) { set_error("linear backward: %s", cudaGetErrorString(e)); return SSD_ERR_CUDA; }
    return SSD_OK;
  }
  const void* g = dout;
  long long gs = dos;
  if (need_dpre || db) {
    T* dpre = need_dpre ? (T*)(ws + p.dpre) : nullptr;
    float* partial = db ? (float*)(ws + p.partial) : nullptr;
    constexpr int V = 16 / (int)sizeof(T);
    if (p.N % V == 0 && dos % V == 0 && (((uintptr_t)dout | (p.act ? (uintptr_t)pre : 0)) & 15) == 0)
      launch<k_dpre<T, V>>(dim3((p.N + 32 * V - 1) / (32 * V), p.parts), dim3(32, 8), 0, s, p.M, p.N, p.act, (const T*)dout, dos, (const float*)pre, dpre, partial, status);
    else
      launch<k_dpre<T, 1>>(dim3((p.N + 31) / 32, p.parts), dim3(32, 8), 0, s, p.M, p.N, p.act, (const T*)dout, dos, (const float*)pre, dpre, partial, status);
    SSD_CUDA_CHECK_LAUNCH("linear_dpre");
    first = false;
    if (db) {
      launch<k_dbias<T>>((p.N + 31) / 32, dim3(32, 32), 0, s, p.N, p.parts, (const float*)partial, (T*)db);
      SSD_CUDA_CHECK_LAUNCH("linear_dbias");
    }
    if (need_dpre) { g = dpre; gs = p.N; }
  }
  int rc = SSD_OK;
  float* part = (float*)(ws + p.part_bwd);
  if (std::is_same<T, __nv_bfloat16>::value && p.tc && map_fits(g, p.M, gs) && map_fits(w, p.N, p.K)) {
    typedef __nv_bfloat16 bf;
    if (dx && (rc = run_mm2("linear_dx", p.tdx, {g, true, gs}, {w, false, p.K}, p.M, p.K, p.N, {(bf*)dx, nullptr, nullptr, nullptr, p.K, 0, 0}, part, status, first,
                           s)))
      return rc;
    if (!dw) return rc;
    first = first && !dx;
    if (map_fits(x, p.M, p.xs))
      return run_mm2("linear_dw", p.tdw, {g, false, gs}, {x, false, p.xs}, p.N, p.K, p.M, {(bf*)dw, nullptr, nullptr, nullptr, p.K, 0, 0}, part, status, first, s);
    dx = nullptr;
  }
  if (dx && (rc = run_mm<T>("linear_dx", MmArgs{g, w, nullptr, nullptr, dx, nullptr, p.M, p.K, p.N, gs, 1, 1, p.K, p.K, 0, 0, 1, 0, part, first ? status : nullptr}, s)))
    return rc;
  first = first && !dx;
  if (dw && (rc = run_mm<T>("linear_dw", MmArgs{g, x, nullptr, nullptr, dw, nullptr, p.N, p.K, p.M, 1, gs, 1, p.xs, p.K, 0, 0, 1, 0, part, first ? status : nullptr}, s)))
    return rc;
  return rc;
}

}  // namespace
}  // namespace ssd

using namespace ssd;

extern "C" {

size_t ssd_linear_workspace_bytes(const SsdLinearDims* dims, int32_t pass) {
  clear_error();
  LinPlan p;
  if (make_lin_plan(dims, pass, &p)) return 0;
  return pass == SSD_PASS_BWD ? p.bwd_bytes : p.fwd_bytes;
}

int32_t ssd_linear_forward(const SsdLinearDims* dims, const void* x, const void* weight, const void* bias, const void* residual, void* out,
                           void* pre, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  clear_error();
  LinPlan p;
  int rc = make_lin_plan(dims, SSD_PASS_FWD, &p);
  if (rc || (rc = check_device(dims))) return rc;
  if (!x || !weight || !out || !workspace) { set_error("linear: x, weight, out and workspace must be non-NULL"); return SSD_ERR_NULL_POINTER; }
  if ((uintptr_t)workspace & 3) { set_error("linear: workspace must be 4-byte aligned (its first word is the status)"); return SSD_ERR_BAD_ALIGNMENT; }
  if (workspace_bytes < p.fwd_bytes) { set_error("linear: workspace too small: %zu < %zu", workspace_bytes, p.fwd_bytes); return SSD_ERR_WORKSPACE_TOO_SMALL; }
  cudaStream_t s = (cudaStream_t)cuda_stream;
  char* ws = aligned_base(workspace);
  const MmArgs a{x, weight, bias, residual, out, (float*)pre, p.M, p.N, p.K, p.xs, 1, p.K, 1, p.os, p.rs, p.act, 1, 0, (float*)(ws + p.part_fwd), (int*)workspace};
  const bool bf16 = dims->dtype == SSD_BF16, vectors = (((uintptr_t)x | (uintptr_t)weight) & 15) == 0 && p.K % (16 / p.es) == 0 && (p.M == 1 || p.xs % (16 / p.es) == 0);
  if (p.M <= FEW && vectors) return bf16 ? run_few<__nv_bfloat16>(a, s) : run_few<float>(a, s);
  if (p.tc && map_fits(x, p.M, p.xs) && map_fits(weight, p.N, p.K)) {
    typedef __nv_bfloat16 bf;
    return run_mm2("linear_fwd", p.fwd, {x, true, p.xs}, {weight, true, p.K}, p.M, p.N, p.K,
                   {(bf*)out, (float*)pre, (const bf*)bias, (const bf*)residual, p.os, p.rs, p.act}, (float*)(ws + p.part_fwd), (int*)workspace, true, s);
  }
  return bf16 ? run_mm<__nv_bfloat16>("linear_fwd", a, s) : run_mm<float>("linear_fwd", a, s);
}

int32_t ssd_linear_backward(const SsdLinearDims* dims, const void* x, const void* weight, const void* pre, const void* dout,
                            int64_t dout_stride_row, void* dx, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                            void* cuda_stream) {
  clear_error();
  LinPlan p;
  int rc = make_lin_plan(dims, SSD_PASS_BWD, &p);
  if (rc || (rc = check_device(dims))) return rc;
  if (!x || !weight || !dout || !workspace) { set_error("linear backward: x, weight, dout and workspace must be non-NULL"); return SSD_ERR_NULL_POINTER; }
  if (p.act && !pre) { set_error("linear backward: an activation needs the forward's pre"); return SSD_ERR_NULL_POINTER; }
  const long long dos = dout_stride_row ? dout_stride_row : p.N;
  if (dos < p.N) { set_error("linear backward: dout's row stride must be at least the row size"); return SSD_ERR_BAD_SHAPE; }
  if ((uintptr_t)workspace & 3) { set_error("linear: workspace must be 4-byte aligned (its first word is the status)"); return SSD_ERR_BAD_ALIGNMENT; }
  if (workspace_bytes < p.bwd_bytes) { set_error("linear backward: workspace too small: %zu < %zu", workspace_bytes, p.bwd_bytes); return SSD_ERR_WORKSPACE_TOO_SMALL; }
  char* ws = aligned_base(workspace);
  cudaStream_t s = (cudaStream_t)cuda_stream;
  return dims->dtype == SSD_BF16 ? linear_backward<__nv_bfloat16>(p, x, weight, pre, dout, dos, dx, dweight, dbias, ws, (int*)workspace, s)
                                 : linear_backward<float>(p, x, weight, pre, dout, dos, dx, dweight, dbias, ws, (int*)workspace, s);
}

}  // extern "C"
