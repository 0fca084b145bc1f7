// A layer's projection with its epilogue:  out = act(x W^T + bias) + residual, and its gradients.
//
// k_mm is the general form: any sizes, strides and both storage types, fp32 products and sums on the CUDA cores.
#include "common.cuh"
#include "ssd_internal.h"

namespace ssd {
namespace {

__device__ __forceinline__ float act_of(float v, int act) {
  if (act == SSD_ACT_SILU) return v * __fdividef(1.f, 1.f + __expf(-v));
  if (act == SSD_ACT_SOFTPLUS) return fmaxf(v, 0.f) + log1pf(__expf(-fabsf(v)));
  if (act == SSD_ACT_RELU2) { const float r = fmaxf(v, 0.f); return r * r; }
  return v;
}
__device__ __forceinline__ float dact_of(float v, int act) {
  if (act == SSD_ACT_SILU) { const float s = __fdividef(1.f, 1.f + __expf(-v)); return s * fmaf(v, 1.f - s, 1.f); }
  if (act == SSD_ACT_SOFTPLUS) return __fdividef(1.f, 1.f + __expf(-v));
  if (act == SSD_ACT_RELU2) return 2.f * fmaxf(v, 0.f);
  return 1.f;
}

// out[m][n] = epilogue(sum_k P(m,k) Q(n,k)); element strides of P and Q along both dims.
struct MmArgs {
  const void *P, *Q, *bias, *residual;
  void *out, *pre;
  long long M, N, K, psm, psk, qsn, qsk, os, rs;
  int act;
};

template <typename T>
__global__ void __launch_bounds__(256) k_mm(MmArgs a) {
  constexpr int BM = 64, BN = 64, BK = 16;
  __shared__ float sp[BK][BM + 1], sq[BK][BN + 1];
  pdl_wait();
  const int tid = threadIdx.x;
  const long long nn = (a.N + BN - 1) / BN, m0 = (long long)(blockIdx.x / nn) * BM, n0 = (long long)(blockIdx.x % nn) * BN;
  const int tm = tid / 16, tn = tid % 16;
  const T *P = (const T*)a.P, *Q = (const T*)a.Q;
  float acc[4][4] = {};
  const bool pk = a.psk == 1, qk = a.qsk == 1;      // which index runs along memory: neighbouring threads follow it
  for (long long k0 = 0; k0 < a.K; k0 += BK) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BM * BK / 256; ++i) {
      const int e = tid + i * 256;
      const int k = pk ? e % BK : e / BM, m = pk ? e / BK : e % BM;
      sp[k][m] = m0 + m < a.M && k0 + k < a.K ? ldf(P + (m0 + m) * a.psm + (k0 + k) * a.psk) : 0.f;
      const int kq = qk ? e % BK : e / BN, n = qk ? e / BK : e % BN;
      sq[kq][n] = n0 + n < a.N && k0 + kq < a.K ? ldf(Q + (n0 + n) * a.qsn + (k0 + kq) * a.qsk) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < BK; ++k) {
      float x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { x[i] = sp[k][tm + 16 * i]; y[i] = sq[k][tn + 16 * i]; }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long m = m0 + tm + 16 * i;
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long n = n0 + tn + 16 * j;
      if (n >= a.N) continue;
      float v = acc[i][j];
      if (a.bias) v += ldf((const T*)a.bias + n);
      if (a.pre) stf((T*)a.pre + m * a.N + n, v);
      v = act_of(v, a.act);
      if (a.residual) v += ldf((const T*)a.residual + m * a.rs + n);
      stf((T*)a.out + m * a.os + n, v);
    }
  }
}

// dpre = dout act'(pre), rounded to the storage type (what the two products read), and the column sums of the unrounded dpre over a
// part of the rows.  Block = 32 columns x 8 rows at a time; `parts` parts of the rows on the y axis.
template <typename T>
__global__ void __launch_bounds__(256) k_dpre(long long M, int N, int act, const T* __restrict__ dout, long long dos, const T* __restrict__ pre,
                                              T* __restrict__ dpre, float* __restrict__ partial) {
  __shared__ float s[8][32];
  pdl_wait();
  const int n = blockIdx.x * 32 + threadIdx.x;
  const long long per = (M + gridDim.y - 1) / gridDim.y, lo = per * blockIdx.y, hi = min(lo + per, M);
  float a = 0.f;
  if (n < N) {
    float t = 0.f;
    int c = 0;
    for (long long m = lo + threadIdx.y; m < hi; m += 8) {
      float g = ldf(dout + m * dos + n);
      if (act) g *= dact_of(ldf(pre + m * N + n), act);
      if (dpre) stf(dpre + m * N + n, g);
      t += g;
      if (++c == 16) { a += t; t = 0.f; c = 0; }
    }
    a += t;
  }
  if (!partial) return;
  s[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.y || n >= N) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) a += s[k][threadIdx.x];
  partial[(long long)blockIdx.y * N + n] = a;
}
template <typename T>
__global__ void __launch_bounds__(256) k_dbias(int N, int parts, const float* __restrict__ partial, T* __restrict__ dbias) {
  pdl_wait();
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  float a = 0.f;
  for (int p = 0; p < parts; ++p) a += partial[(long long)p * N + n];
  stf(dbias + n, a);
}

// ---- host --------------------------------------------------------------------------------------------------------------
size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
struct LinPlan {
  long long M, xs, os, rs;
  int K, N, act, es, parts;
  size_t dpre, partial, fwd_bytes, bwd_bytes;
};
int make_lin_plan(const SsdLinearDims* d, LinPlan* o) {
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
  if (((o->M + 63) / 64) * ((o->N + 63) / 64) > 0x7fffffffLL) { set_error("linear: too many output tiles for one grid"); return SSD_ERR_UNSUPPORTED; }
  const long long cols = (o->N + 31) / 32, want = (4 * 148 + cols - 1) / cols, most = (o->M + 63) / 64;
  o->parts = (int)(want < most ? want : most);
  size_t at = 0;
  auto take = [&](size_t n) { const size_t r = at; at += up256(n); return r; };
  o->fwd_bytes = 256;
  o->dpre = take(o->act ? (size_t)o->M * o->N * o->es : 0);
  o->partial = take((size_t)o->parts * o->N * sizeof(float));
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
  const long long blocks = ((a.M + 63) / 64) * ((a.N + 63) / 64);
  launch<k_mm<T>>((unsigned)blocks, 256, 0, s, a);
  SSD_CUDA_CHECK_LAUNCH(what);
  return SSD_OK;
}

template <typename T>
int linear_backward(const LinPlan& p, const void* x, const void* w, const void* pre, const void* dout, long long dos, void* dx, void* dw,
                    void* db, char* ws, cudaStream_t s) {
  const bool need_dpre = p.act && (dx || dw);
  const void* g = dout;
  long long gs = dos;
  if (need_dpre || db) {
    T* dpre = need_dpre ? (T*)(ws + p.dpre) : nullptr;
    float* partial = db ? (float*)(ws + p.partial) : nullptr;
    launch<k_dpre<T>>(dim3((p.N + 31) / 32, p.parts), dim3(32, 8), 0, s, p.M, p.N, p.act, (const T*)dout, dos, (const T*)pre, dpre, partial);
    SSD_CUDA_CHECK_LAUNCH("linear_dpre");
    if (db) {
      launch<k_dbias<T>>((p.N + 255) / 256, 256, 0, s, p.N, p.parts, (const float*)partial, (T*)db);
      SSD_CUDA_CHECK_LAUNCH("linear_dbias");
    }
    if (need_dpre) { g = dpre; gs = p.N; }
  }
  int rc = SSD_OK;
  if (dx && (rc = run_mm<T>("linear_dx", MmArgs{g, w, nullptr, nullptr, dx, nullptr, p.M, p.K, p.N, gs, 1, 1, p.K, p.K, 0, 0}, s))) return rc;
  if (dw && (rc = run_mm<T>("linear_dw", MmArgs{g, x, nullptr, nullptr, dw, nullptr, p.N, p.K, p.M, 1, gs, 1, p.xs, p.K, 0, 0}, s))) return rc;
  return rc;
}

}  // namespace
}  // namespace ssd

using namespace ssd;

extern "C" {

size_t ssd_linear_workspace_bytes(const SsdLinearDims* dims, int32_t pass) {
  clear_error();
  LinPlan p;
  if (make_lin_plan(dims, &p)) return 0;
  return pass == SSD_PASS_BWD ? p.bwd_bytes : p.fwd_bytes;
}

int32_t ssd_linear_forward(const SsdLinearDims* dims, const void* x, const void* weight, const void* bias, const void* residual, void* out,
                           void* pre, void* workspace, size_t workspace_bytes, void* cuda_stream) {
  clear_error();
  LinPlan p;
  int rc = make_lin_plan(dims, &p);
  if (rc || (rc = check_device(dims))) return rc;
  if (!x || !weight || !out || !workspace) { set_error("linear: x, weight, out and workspace must be non-NULL"); return SSD_ERR_NULL_POINTER; }
  if (workspace_bytes < p.fwd_bytes) { set_error("linear: workspace too small: %zu < %zu", workspace_bytes, p.fwd_bytes); return SSD_ERR_WORKSPACE_TOO_SMALL; }
  cudaStream_t s = (cudaStream_t)cuda_stream;
  const MmArgs a{x, weight, bias, residual, out, pre, p.M, p.N, p.K, p.xs, 1, p.K, 1, p.os, p.rs, p.act};
  return dims->dtype == SSD_BF16 ? run_mm<__nv_bfloat16>("linear_fwd", a, s) : run_mm<float>("linear_fwd", a, s);
}

int32_t ssd_linear_backward(const SsdLinearDims* dims, const void* x, const void* weight, const void* pre, const void* dout,
                            int64_t dout_stride_row, void* dx, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                            void* cuda_stream) {
  clear_error();
  LinPlan p;
  int rc = make_lin_plan(dims, &p);
  if (rc || (rc = check_device(dims))) return rc;
  if (!x || !weight || !dout || !workspace) { set_error("linear backward: x, weight, dout and workspace must be non-NULL"); return SSD_ERR_NULL_POINTER; }
  if (p.act && !pre) { set_error("linear backward: an activation needs the forward's pre"); return SSD_ERR_NULL_POINTER; }
  const long long dos = dout_stride_row ? dout_stride_row : p.N;
  if (dos < p.N) { set_error("linear backward: dout's row stride must be at least the row size"); return SSD_ERR_BAD_SHAPE; }
  if (workspace_bytes < p.bwd_bytes) { set_error("linear backward: workspace too small: %zu < %zu", workspace_bytes, p.bwd_bytes); return SSD_ERR_WORKSPACE_TOO_SMALL; }
  char* ws = aligned_base(workspace);
  cudaStream_t s = (cudaStream_t)cuda_stream;
  return dims->dtype == SSD_BF16 ? linear_backward<__nv_bfloat16>(p, x, weight, pre, dout, dos, dx, dweight, dbias, ws, s)
                                 : linear_backward<float>(p, x, weight, pre, dout, dos, dx, dweight, dbias, ws, s);
}

}  // extern "C"
