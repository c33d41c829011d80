// Root-mean-square norm with the residual's addition, forward and backward,
// and its output in 8 bits (e4m3) with scales.
//
//   h = round(x + r)              (r absent: h = x)
//   rstd = (mean(h^2) + eps)^(-1/2),  n = h rstd,  y = n w
// The norm reads h as it is stored: the next layer adds to the stored stream,
// and the backward, which has only the stored h, differentiates this function.
//   8 bits: t = h w, a = max(|t|, 2^-100) over a row or 128 columns,
//           q = e4m3(448 t / a), scale = a rstd / 448       (q scale = y)
// rstd cancels in t / a, so the codes do not depend on how the mean was summed.
// The quotient is rounded once (__fdiv_rn): with bf16 factors t and 448 t are
// exact, and values that lie midway between two codes go to the even one.
//   backward, g = dy w:  d = dh + rstd (g - n mean(g n));  dx = dr = d
//                        dw = sum over rows of dy n
// Sums and statistics are fp32; each output is rounded once to its type.
//
// Bound: HBM.  Each row is read once into registers (8 consecutive elements per
// thread and chunk, 16-byte accesses) and written once.  Rows of up to 1024
// columns take one warp each, longer ones one CTA each.
#include <cuda_fp8.h>

#include <type_traits>

#include "lh_common.cuh"

namespace lh {
namespace norm {

constexpr int kChunks = 4;                   // chunks of 8 elements per thread
constexpr int kWarpRow = 32 * 8 * kChunks;   // longest row that one warp holds
constexpr int kCtaThreads = 512;             // most threads of a CTA row: D <= 16384
constexpr float kE4m3Max = 448.f;
constexpr float kAmaxMin = 7.888609052210118e-31f;   // 2^-100

struct None {};

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&f)[8]) { load16(p, f); }
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) { load16(p, f); load16(p + 4, f + 4); }
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) { store16(p, f); }
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) { store16(p, f); store16(p + 4, f + 4); }
__device__ __forceinline__ void load8w(const void* w, bool f32, int col, float (&f)[8]) {
  if (f32) load8(reinterpret_cast<const float*>(w) + col, f);
  else load8(reinterpret_cast<const __nv_bfloat16*>(w) + col, f);
}
__device__ __forceinline__ void store8(__nv_fp8_storage_t* p, const float (&f)[8]) {
  uint2 u;
  __nv_fp8x2_storage_t* h = reinterpret_cast<__nv_fp8x2_storage_t*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i], f[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  *reinterpret_cast<uint2*>(p) = u;
}

// Sum and maximum over the threads that hold one row: a warp, or (CTA) the
// block, whose warps exchange partials through shared memory.
template <bool CTA>
__device__ __forceinline__ void row_reduce(float& sum, float& mx, float2* part) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    sum += __shfl_xor_sync(~0u, sum, o);
    mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
  }
  if (CTA) {
    const int nw = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_float2(sum, mx);
    __syncthreads();
    const int l = threadIdx.x & 31;
    float2 v = l < nw ? part[l] : make_float2(0.f, 0.f);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      v.x += __shfl_xor_sync(~0u, v.x, o);
      v.y = fmaxf(v.y, __shfl_xor_sync(~0u, v.y, o));
    }
    sum = v.x;
    mx = v.y;
  }
}

struct FwdArgs {
  const void *x, *r, *w;
  void *y, *h;
  float *scale, *rstd;
  long long N;
  int D, group;
  bool w_f32;
  float eps, inv_d;
};

template <class TX, class TR, class TY, bool CTA>
__global__ void __launch_bounds__(CTA ? kCtaThreads : 256)
rms_norm_fwd_kernel(const FwdArgs a) {
  constexpr bool kRes = !std::is_same<TR, None>::value;
  constexpr bool kFp8 = std::is_same<TY, __nv_fp8_storage_t>::value;
  __shared__ float2 part[32];
  const long long row = CTA ? blockIdx.x : ((long long)blockIdx.x * 8 + (threadIdx.x >> 5));
  if (!CTA && row >= a.N) return;
  const int t = CTA ? threadIdx.x : (threadIdx.x & 31);
  const int T = CTA ? blockDim.x : 32;
  const size_t base = (size_t)row * a.D;
  float v[kChunks][8];
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
    const int col = (c * T + t) * 8;
    if (col < a.D) {
      load8(reinterpret_cast<const TX*>(a.x) + base + col, v[c]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
    }
  }
  if constexpr (kRes) {
    float r[kChunks][8];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = (c * T + t) * 8;
      if (col < a.D) load8(reinterpret_cast<const TR*>(a.r) + base + col, r[c]);
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = (c * T + t) * 8;
      if (col < a.D) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = round_to(v[c][e] + r[c][e], (const TR*)nullptr);
        store8(reinterpret_cast<TR*>(a.h) + base + col, v[c]);
      }
    }
  }
  float ss = 0.f, mx = 0.f;
#pragma unroll
  for (int c = 0; c < kChunks; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(v[c][e], v[c][e], ss);
  float amax[kChunks];
  if constexpr (kFp8) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = (c * T + t) * 8;
      amax[c] = 0.f;
      if (col < a.D) {
        float w[8];
        load8w(a.w, a.w_f32, col, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[c][e] *= w[e];
          amax[c] = fmaxf(amax[c], fabsf(v[c][e]));
        }
      }
      mx = fmaxf(mx, amax[c]);
    }
  }
  row_reduce<CTA>(ss, mx, part);
  const float rstd = rsqrtf(fmaf(ss, a.inv_d, a.eps));
  if (t == 0 && a.rstd) a.rstd[row] = rstd;
  if constexpr (kFp8) {
    if (a.group == 0) {
      mx = fmaxf(mx, kAmaxMin);
      if (t == 0) a.scale[row] = mx * rstd / kE4m3Max;
    }
    const int n_groups = (a.D + 127) / 128;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = (c * T + t) * 8;
      float m = mx;
      if (a.group) {                          // 16 neighbouring lanes hold one group of 128 columns
        m = amax[c];
#pragma unroll
        for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        m = fmaxf(m, kAmaxMin);
        if ((col & 127) == 0 && col < a.D) a.scale[row * n_groups + (col >> 7)] = m * rstd / kE4m3Max;
      }
      if (col < a.D) {
        float q[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = __fdiv_rn(v[c][e] * kE4m3Max, m);
        store8(reinterpret_cast<TY*>(a.y) + base + col, q);
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = (c * T + t) * 8;
      if (col < a.D) {
        float w[8], y[8];
        load8w(a.w, a.w_f32, col, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = v[c][e] * rstd * w[e];
        store8(reinterpret_cast<TY*>(a.y) + base + col, y);
      }
    }
  }
}

struct BwdArgs {
  const void *dy, *dh, *h, *w;
  const float* rstd;
  void *dx, *dr;                 // dr NULL: no residual, or the same tensor as dx
  float* dw_part;                // (gridDim.x, D)
  long long N;
  int D;
  bool w_f32;
  float inv_d;
};

// Persistent: every warp (or CTA) walks rows and keeps its columns' share of dw
// in registers; the shares meet in dw_part, which dw_reduce_kernel sums in a
// fixed order (no atomics).
template <class TY, class TH, class TX, bool CTA>
__global__ void __launch_bounds__(CTA ? kCtaThreads : 256)
rms_norm_bwd_kernel(const BwdArgs a) {
  __shared__ float2 part[2][32];
  extern __shared__ float dw_sm[];                       // !CTA: 8 x D
  const int t = CTA ? threadIdx.x : (threadIdx.x & 31);
  const int T = CTA ? blockDim.x : 32;
  const long long step = CTA ? gridDim.x : (long long)gridDim.x * 8;
  float dw[kChunks][8];
#pragma unroll
  for (int c = 0; c < kChunks; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[c][e] = 0.f;
  int buf = 0;
  for (long long row = CTA ? blockIdx.x : ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)); row < a.N; row += step) {
    const size_t base = (size_t)row * a.D;
    const float rstd = __ldg(a.rstd + row);
    float n[kChunks][8], g[kChunks][8];
    float s = 0.f, unused = 0.f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = (c * T + t) * 8;
      if (col < a.D) {
        load8(reinterpret_cast<const TH*>(a.h) + base + col, n[c]);
        load8(reinterpret_cast<const TY*>(a.dy) + base + col, g[c]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) n[c][e] = g[c][e] = 0.f;
      }
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = (c * T + t) * 8;
      if (col < a.D) {
        float w[8];
        load8w(a.w, a.w_f32, col, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          n[c][e] *= rstd;
          dw[c][e] = fmaf(g[c][e], n[c][e], dw[c][e]);
          g[c][e] *= w[e];
          s = fmaf(g[c][e], n[c][e], s);
        }
      }
    }
    row_reduce<CTA>(s, unused, part[buf]);
    buf ^= 1;
    const float m = s * a.inv_d;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = (c * T + t) * 8;
      if (col < a.D) {
        float d[8];
        if (a.dh) load8(reinterpret_cast<const TH*>(a.dh) + base + col, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = rstd * fmaf(-n[c][e], m, g[c][e]);
          d[e] = a.dh ? d[e] + v : v;
        }
        store8(reinterpret_cast<TX*>(a.dx) + base + col, d);
        if (a.dr) store8(reinterpret_cast<TH*>(a.dr) + base + col, d);
      }
    }
  }
  if (CTA) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = (c * T + t) * 8;
      if (col < a.D) store8(a.dw_part + (size_t)blockIdx.x * a.D + col, dw[c]);
    }
  } else {
    float* mine = dw_sm + (size_t)(threadIdx.x >> 5) * a.D;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int col = (c * T + t) * 8;
      if (col < a.D) store8(mine + col, dw[c]);
    }
    __syncthreads();
    for (int col = threadIdx.x; col < a.D; col += blockDim.x) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += dw_sm[(size_t)k * a.D + col];
      a.dw_part[(size_t)blockIdx.x * a.D + col] = s;
    }
  }
}

// dw = column sums of dw_part (parts, D): 32 columns per block, 32 strided
// slices of the rows, then a tree over the slices.
__global__ void __launch_bounds__(1024)
dw_reduce_kernel(const float* __restrict__ part, int parts, int D, void* dw, bool w_f32) {
  __shared__ float sm[32][33];
  const int c = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < D)
    for (int i = k; i < parts; i += 32) s += part[(size_t)i * D + col];
  sm[k][c] = s;
  __syncthreads();
  if (k == 0 && col < D) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += sm[i][c];
    if (w_f32) reinterpret_cast<float*>(dw)[col] = v;
    else reinterpret_cast<__nv_bfloat16*>(dw)[col] = __float2bfloat16_rn(v);
  }
}

int cta_threads(int D) { return ((D + 8 * kChunks - 1) / (8 * kChunks) + 31) / 32 * 32; }

template <class TX, class TR, class TY>
int launch_fwd(const FwdArgs& a, cudaStream_t st) {
  if (a.D <= kWarpRow) {
    rms_norm_fwd_kernel<TX, TR, TY, false><<<(unsigned)((a.N + 7) / 8), 256, 0, st>>>(a);
  } else {
    rms_norm_fwd_kernel<TX, TR, TY, true><<<(unsigned)a.N, cta_threads(a.D), 0, st>>>(a);
  }
  return check_launch("rms_norm_fwd_kernel");
}

template <class TX, class TR>
int fwd_y(const FwdArgs& a, int y_dtype, cudaStream_t st) {
  if (y_dtype == LH_DTYPE_BF16) return launch_fwd<TX, TR, __nv_bfloat16>(a, st);
  if (y_dtype == LH_DTYPE_F32) return launch_fwd<TX, TR, float>(a, st);
  return launch_fwd<TX, TR, __nv_fp8_storage_t>(a, st);
}
template <class TX>
int fwd_r(const FwdArgs& a, int r_dtype, int y_dtype, cudaStream_t st) {
  if (!a.r) return fwd_y<TX, None>(a, y_dtype, st);
  return r_dtype == LH_DTYPE_BF16 ? fwd_y<TX, __nv_bfloat16>(a, y_dtype, st) : fwd_y<TX, float>(a, y_dtype, st);
}

// CTAs of the persistent backward: enough warps to fill the 148 SMs.
int bwd_grid(long long N, int D) {
  const long long want = D <= kWarpRow ? (N + 7) / 8 : N;
  const long long cap = D <= kWarpRow ? 148 * 2 : 148 * (cta_threads(D) <= 256 ? 4 : cta_threads(D) <= 512 ? 2 : 1);
  return (int)(want < cap ? want : cap);
}

template <class TY, class TH, class TX>
int launch_bwd(const BwdArgs& a, void* dw, cudaStream_t st) {
  const int grid = bwd_grid(a.N, a.D);
  if (a.D <= kWarpRow)
    rms_norm_bwd_kernel<TY, TH, TX, false><<<grid, 256, 8 * a.D * sizeof(float), st>>>(a);
  else
    rms_norm_bwd_kernel<TY, TH, TX, true><<<grid, cta_threads(a.D), 0, st>>>(a);
  int rc = check_launch("rms_norm_bwd_kernel");
  if (rc) return rc;
  dw_reduce_kernel<<<(a.D + 31) / 32, 1024, 0, st>>>(a.dw_part, grid, a.D, dw, a.w_f32);
  return check_launch("dw_reduce_kernel");
}

template <class TY, class TH>
int bwd_x(const BwdArgs& a, int dx_dtype, void* dw, cudaStream_t st) {
  return dx_dtype == LH_DTYPE_BF16 ? launch_bwd<TY, TH, __nv_bfloat16>(a, dw, st) : launch_bwd<TY, TH, float>(a, dw, st);
}
template <class TY>
int bwd_h(const BwdArgs& a, int h_dtype, int dx_dtype, void* dw, cudaStream_t st) {
  return h_dtype == LH_DTYPE_BF16 ? bwd_x<TY, __nv_bfloat16>(a, dx_dtype, dw, st) : bwd_x<TY, float>(a, dx_dtype, dw, st);
}

}  // namespace norm

int rms_norm_fwd(const void* x, int x_dtype, const void* r, int r_dtype, const void* w, int w_dtype, long long N, int D,
                 float eps, void* y, int y_dtype, float* scale, int group, void* h, float* rstd, cudaStream_t st) {
  norm::FwdArgs a{x, r, w, y, h, scale, rstd, N, D, group, w_dtype == LH_DTYPE_F32, eps, 1.f / D};
  return x_dtype == LH_DTYPE_BF16 ? norm::fwd_r<__nv_bfloat16>(a, r_dtype, y_dtype, st)
                                  : norm::fwd_r<float>(a, r_dtype, y_dtype, st);
}

size_t rms_norm_bwd_workspace_size(long long N, int D) { return (size_t)norm::bwd_grid(N, D) * D * sizeof(float); }

int rms_norm_bwd(const void* dy, int dy_dtype, const void* dh, const void* h, int h_dtype, const void* w, int w_dtype,
                 const float* rstd, long long N, int D, void* dx, int dx_dtype, void* dr, void* dw, void* ws,
                 cudaStream_t st) {
  norm::BwdArgs a{dy, dh, h, w, rstd, dx, dr, (float*)ws, N, D, w_dtype == LH_DTYPE_F32, 1.f / D};
  return dy_dtype == LH_DTYPE_BF16 ? norm::bwd_h<__nv_bfloat16>(a, h_dtype, dx_dtype, dw, st)
                                   : norm::bwd_h<float>(a, h_dtype, dx_dtype, dw, st);
}

}  // namespace lh
