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
// The quotient is n / a from the rounded reciprocal y of a: q0 = n y, then
// q0 + (n - q0 a) y with both sums fused.  With q0 = (n / a)(1 + d) the result is
// (n / a)(1 - d e) before its rounding, e the error of y, d and e about 2^-24: a
// quotient that fp32 holds comes out exact.  With bf16 factors t and n = 448 t are
// exact too, so values that lie midway between two codes go to the even one.
// (One division per element instead takes 300 us where this takes 219, at
// 32768 x 5120.)
//   backward, g = dy w:  d = dh + rstd (g - n mean(g n));  dx = dr = d
//                        dw = sum over rows of dy n
// Sums and statistics are fp32; each output is rounded once to its type.
//
// Bound: HBM.  Each row is read once into registers (chunks of 8 consecutive
// elements per thread, 16-byte accesses) and written once.  Rows of up to 256
// columns take one warp each, longer ones one CTA each.
#include <cuda_fp8.h>

#include <type_traits>

#include "lh_common.cuh"

namespace lh {
namespace norm {

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

template <class TX, class TR, class TY, bool CTA, int CH>
__global__ void __launch_bounds__(CTA ? 1024 : 256)
rms_norm_fwd_kernel(const FwdArgs a) {
  constexpr bool kRes = !std::is_same<TR, None>::value;
  constexpr bool kFp8 = std::is_same<TY, __nv_fp8_storage_t>::value;
  __shared__ float2 part[32];
  const long long row = CTA ? blockIdx.x : ((long long)blockIdx.x * 8 + (threadIdx.x >> 5));
  if (!CTA && row >= a.N) return;
  const int t = CTA ? threadIdx.x : (threadIdx.x & 31);
  const int T = CTA ? blockDim.x : 32;
  const size_t base = (size_t)row * a.D;
  float v[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = (c * T + t) * 8;
    if (col < a.D) {
      load8(reinterpret_cast<const TX*>(a.x) + base + col, v[c]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
    }
  }
  if constexpr (kRes) {
    float r[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * T + t) * 8;
      if (col < a.D) load8(reinterpret_cast<const TR*>(a.r) + base + col, r[c]);
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) {
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
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(v[c][e], v[c][e], ss);
  float amax[CH];
  if constexpr (kFp8) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
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
    for (int c = 0; c < CH; ++c) {
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
        const float inv = __frcp_rn(m);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float n = v[c][e] * kE4m3Max, q0 = n * inv;
          q[e] = fmaf(fmaf(-q0, m, n), inv, q0);
        }
        store8(reinterpret_cast<TY*>(a.y) + base + col, q);
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
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

// Eight elements as they lie in memory, fetched now and opened later.
template <class T> struct Raw8;
template <> struct Raw8<__nv_bfloat16> { uint4 a; };
template <> struct Raw8<float> { uint4 a, b; };
__device__ __forceinline__ void fetch(const __nv_bfloat16* p, Raw8<__nv_bfloat16>& r) {
  r.a = __ldg(reinterpret_cast<const uint4*>(p));
}
__device__ __forceinline__ void fetch(const float* p, Raw8<float>& r) {
  r.a = __ldg(reinterpret_cast<const uint4*>(p));
  r.b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
}
__device__ __forceinline__ void open8(const Raw8<__nv_bfloat16>& r, float (&f)[8]) {
  unpack16(r.a, f, (const __nv_bfloat16*)nullptr);
}
__device__ __forceinline__ void open8(const Raw8<float>& r, float (&f)[8]) {
  unpack16(r.a, f, (const float*)nullptr);
  unpack16(r.b, f + 4, (const float*)nullptr);
}

struct BwdArgs {
  const void *dy, *dh, *h, *w;
  const float* rstd;
  void *dx, *dr;                 // dr NULL: no residual
  float* dw_part;                // (gridDim.x, D)
  long long N;
  int D;
  bool w_f32;
  float inv_d;
};

// Persistent: every warp (or CTA) walks rows and keeps its columns' share of dw
// in registers; the shares meet in dw_part, which dw_reduce_kernel sums in a
// fixed order (no atomics).
template <class TY, class TH, class TX, bool CTA, int CH, int MAXT, int MINB>
__global__ void __launch_bounds__(MAXT, MINB)
rms_norm_bwd_kernel(const BwdArgs a) {
  let_next_start();                                      // dw_reduce_kernel
  __shared__ float2 part[2][32];
  extern __shared__ float dw_sm[];                       // !CTA: 8 x D
  const int t = CTA ? threadIdx.x : (threadIdx.x & 31);
  const int T = CTA ? blockDim.x : 32;
  const long long step = CTA ? gridDim.x : (long long)gridDim.x * 8;
  float dw[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[c][e] = 0.f;
  int buf = 0;
  long long row = CTA ? blockIdx.x : ((long long)blockIdx.x * 8 + (threadIdx.x >> 5));
  Raw8<TH> rh[CH], rd[CH];
  Raw8<TY> ry[CH];
  float rs = 0.f;
  auto get = [&](long long r) {
    const size_t base = (size_t)r * a.D;
    rs = __ldg(a.rstd + r);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * T + t) * 8;
      if (col < a.D) {
        fetch(reinterpret_cast<const TH*>(a.h) + base + col, rh[c]);
        fetch(reinterpret_cast<const TY*>(a.dy) + base + col, ry[c]);
        if (a.dh) fetch(reinterpret_cast<const TH*>(a.dh) + base + col, rd[c]);
      }
    }
  };
  if (row < a.N) get(row);
  for (; row < a.N; row += step) {
    const size_t base = (size_t)row * a.D;
    const float rstd = rs;
    float s = 0.f, unused = 0.f;
    Raw8<TH> ch[CH], cd[CH];
    Raw8<TY> cy[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) { ch[c] = rh[c]; cd[c] = rd[c]; cy[c] = ry[c]; }
    if (row + step < a.N) get(row + step);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * T + t) * 8;
      if (col < a.D) {
        float w[8], n[8], g[8];
        load8w(a.w, a.w_f32, col, w);
        open8(ch[c], n);
        open8(cy[c], g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          n[e] *= rstd;
          const float gn = g[e] * n[e];
          dw[c][e] += gn;
          s = fmaf(gn, w[e], s);
        }
      }
    }
    row_reduce<CTA>(s, unused, part[buf]);
    buf ^= 1;
    const float m = s * a.inv_d;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * T + t) * 8;
      if (col < a.D) {
        float w[8], n[8], g[8], d[8];
        load8w(a.w, a.w_f32, col, w);
        open8(ch[c], n);
        open8(cy[c], g);
        if (a.dh) open8(cd[c], d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = rstd * fmaf(-n[e] * rstd, m, g[e] * w[e]);
          d[e] = a.dh ? d[e] + v : v;
        }
        store8(reinterpret_cast<TX*>(a.dx) + base + col, d);
        if (a.dr) store8(reinterpret_cast<TH*>(a.dr) + base + col, d);
      }
    }
  }
  if (CTA) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * T + t) * 8;
      if (col < a.D) store8(a.dw_part + (size_t)blockIdx.x * a.D + col, dw[c]);
    }
  } else {
    float* mine = dw_sm + (size_t)(threadIdx.x >> 5) * a.D;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
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
dw_reduce_kernel(const float* part, int parts, int D, void* dw, bool w_f32) {
  after_previous();
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

// Threads of a CTA whose threads hold ch chunks of a row each.
int cta_threads(int D, int ch) { return ((D + 8 * ch - 1) / (8 * ch) + 31) / 32 * 32; }

// One chunk per thread wherever a CTA has the threads for it: 8191 x 4096 bf16
// takes 47 us with one chunk, 55 with two or four, and four single rows with
// 8-bit output 8.2 against 10.2 (events around the call).
template <class TX, class TR, class TY>
int launch_fwd(const FwdArgs& a, cudaStream_t st) {
  if (a.D <= 256)
    rms_norm_fwd_kernel<TX, TR, TY, false, 1><<<(unsigned)((a.N + 7) / 8), 256, 0, st>>>(a);
  else if (a.D <= 8192)
    rms_norm_fwd_kernel<TX, TR, TY, true, 1><<<(unsigned)a.N, cta_threads(a.D, 1), 0, st>>>(a);
  else
    rms_norm_fwd_kernel<TX, TR, TY, true, 2><<<(unsigned)a.N, cta_threads(a.D, 2), 0, st>>>(a);
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

// Shapes of the persistent backward: chunks per thread and CTAs per SM.  The next
// row's loads are in flight while a row is worked on, in registers, so a thread
// holds few chunks: 65536 x 1024 (fp32 stream) takes 144 us with one chunk, 161
// with two; 8191 x 4096 (bf16) 62 us with two chunks and 256 threads.
enum BwdShape { kWarp, kOne, kTwo, kTwoWide, kFour };
BwdShape bwd_shape(int D) {
  return D <= 256 ? kWarp : D <= 2048 ? kOne : D <= 4096 ? kTwo : D <= 8192 ? kTwoWide : kFour;
}
int bwd_threads(int D) {
  const BwdShape s = bwd_shape(D);
  return s == kWarp ? 256 : cta_threads(D, s == kOne ? 1 : s == kFour ? 4 : 2);
}
// CTAs: what the register limits of the launch bounds let live on 148 SMs.
int bwd_grid(long long N, int D) {
  const BwdShape s = bwd_shape(D);
  const int warps = s == kWarp || s == kOne ? 24 : 16, t = bwd_threads(D) / 32;
  const long long want = s == kWarp ? (N + 7) / 8 : N, cap = 148ll * (warps / t > 1 ? warps / t : 1);
  return (int)(want < cap ? want : cap);
}

template <class TY, class TH, class TX>
int launch_bwd(const BwdArgs& a, void* dw, cudaStream_t st) {
  const int grid = bwd_grid(a.N, a.D), t = bwd_threads(a.D);
  switch (bwd_shape(a.D)) {
    case kWarp: rms_norm_bwd_kernel<TY, TH, TX, false, 1, 256, 3><<<grid, t, 8 * a.D * sizeof(float), st>>>(a); break;
    case kOne: rms_norm_bwd_kernel<TY, TH, TX, true, 1, 256, 3><<<grid, t, 0, st>>>(a); break;
    case kTwo: rms_norm_bwd_kernel<TY, TH, TX, true, 2, 256, 2><<<grid, t, 0, st>>>(a); break;
    case kTwoWide: rms_norm_bwd_kernel<TY, TH, TX, true, 2, 512, 1><<<grid, t, 0, st>>>(a); break;
    case kFour: rms_norm_bwd_kernel<TY, TH, TX, true, 4, 512, 1><<<grid, t, 0, st>>>(a); break;
  }
  int rc = check_launch("rms_norm_bwd_kernel");
  if (rc) return rc;
  return launch_behind("dw_reduce_kernel", dw_reduce_kernel, (a.D + 31) / 32, 1024, 0, st, a.dw_part, grid, a.D, dw, a.w_f32);
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
