// Losses of an output projection whose logits are never stored: softmax cross
// entropy, and distillation from a teacher's top logits, forward and backward.
//
// With hidden rows h_i (N, D), weights w_v (V, D), s_iv = h_i . w_v, and a few
// targets (v_k, p_k) per row (cross entropy: one, p = 1; distillation: p =
// softmax(t_k / T) over the row's K teacher logits, s divided by T):
//   lse_i  = log sum_v exp(s_iv)
//   loss_i = T^2 (sum_k p_k log p_k - sum_k p_k s_ik + lse_i)
//   G_iv   = c_i (exp(s_iv - lse_i) - sum_{k: v_k = v} p_k),  c_i = T dloss_i
//   dH = G W,   dW = G^T H
// Forward: one GEMM whose epilogue keeps a row's maximum and sum of exponentials
// per 128 columns, V / 128 pairs per row, which finish_kernel joins.
// Backward, in pieces of the vocabulary of C columns: the logits again, their
// epilogue writing G (N, C) in bf16; then dH += G W_piece and dW_piece = G^T H.
// G is rounded to bf16 once, as an operand of bf16 MMAs has to be; its relative
// error of 2^-9 is that of the bf16 gradients it ends in.  All sums are fp32.
//
// One persistent GEMM kernel does all four products: a pair of SMs
// (tcgen05.mma.cta_group::2) per 256 x 256 tile, so that each SM loads 128 rows
// of either operand and both accumulators (2 x 256 TMEM columns) alternate
// between the MMAs of one tile and the epilogue of the one before.  Roles: warp
// 0 TMA producer, warp 1 MMA issuer (leader's), warps 4-11 epilogue (thread = row
// = TMEM lane, two warps per row block, half the columns each).  Operands are K-major or MN-major as they lie in memory: no
// transposed copy exists.  Where a product has few tiles, its K range is split
// and the parts meet in fp32 planes which planes_kernel sums in a fixed order.
// Every mbarrier wait is bounded; on expiry the CTAs leave and a status flag is set.
#include <cudaTypedefs.h>

#include "lh_common.cuh"
#include "sm100.cuh"

namespace lh {

using namespace sm100;

__device__ int g_loss_status;    // set to 1 when a bounded wait gave up

namespace ll {

constexpr int kTM = 256, kTN = 256, kTK = 64;    // tile of a pair of SMs
constexpr int kBox = 64 * 64 * 2;                // one 64 x 64 bf16 TMA box, 128-byte rows
constexpr int kOpBytes = 2 * kBox;               // 128 rows of an operand: one CTA's share of a stage
constexpr int kThreads = 384;
constexpr int kOutBuf = 4096;                    // 32 rows x 128 bytes: one store of an epilogue warp
constexpr int kPairs = 74;
constexpr int kNone = 0x7fffffff;
constexpr float kLn2 = 0.69314718055994531f, kLog2e = 1.4426950408889634f;

enum Mode { kStats, kGrad, kDH, kDW };
enum Out { kOutBf16, kOutPlane, kOutPlaneAdd };

// Stages of the operand ring and staging buffers per epilogue warp: a warp's half
// of a bf16 row block is two stores, each with a buffer of its own, so that it
// waits for a store of the tile before only; kStats stores nothing.
__host__ __device__ constexpr int stages(int mode) { return mode == kStats ? 6 : 5; }
__host__ __device__ constexpr int bufs(int mode) { return mode == kStats ? 1 : 2; }
constexpr int smem_bytes(int mode) { return 1024 + stages(mode) * 2 * kOpBytes + 8 * bufs(mode) * kOutBuf + 512; }

struct Smem {
  uint64_t full[6], empty[6], acc_full[2], acc_empty[2], drain;
  uint32_t tmem_base;
  int abort;
};
static_assert(sizeof(Smem) <= 512 && smem_bytes(kStats) <= 232448 && smem_bytes(kGrad) <= 232448, "barriers do not fit their space");

struct Args {
  int M, N;                       // rows and columns of the result
  int tiles_m, tiles_n, splits, kb, gm;
  FastDiv per_split, per_group, per_col, per_col_last;   // tiles of a split, a group, and of its columns
  int b_off;                      // first row of B's operand (vocabulary piece)
  int out;                        // kDH, kDW: Out
  // targets: int64 (K = 1, SPARSE false) or sorted int32 (K, M), a row's entries M apart
  const long long* target;
  const int* idx;
  int K;
  float a2;                       // log2(e) / T
  float2* stats;                  // kStats: (2 tiles_n, M) maximum and sum of a row's 128 columns
  float* slog;                    // kStats: logits of the targets (K, M) out
  unsigned* ticket;               // kStats: set to 0 for finish_kernel
  const float* gval;              // kGrad: exp(s - lse) - p at the targets (K, M)
  const float* lse2;              // kGrad: log2-sum-exp2 of s a2
  const float *gout, *row_scale, *inv_count;
  int gstride;
  float cscale;
};

// Position of the first of a row's K sorted targets, M apart, that is >= v.
__device__ __forceinline__ int lower_bound(const int* __restrict__ idx, int K, size_t M, int v) {
  int lo = 0, hi = K;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(idx + mid * M) < v) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

template <int MODE, bool SPARSE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
loss_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const __grid_constant__ CUtensorMap tmO, const Args a) {
  constexpr bool kAMn = MODE == kDW, kBMn = MODE == kDH || MODE == kDW;
  constexpr int kStages = stages(MODE), kBufs = bufs(MODE);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = base;
  uint8_t* sB = base + kStages * kOpBytes;
  uint8_t* sO = base + 2 * kStages * kOpBytes;
  Smem* sm = reinterpret_cast<Smem*>(sO + 8 * kBufs * kOutBuf);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const int total = a.tiles_m * a.tiles_n * a.splits;

  if (threadIdx.x == 0) {
    if (MODE == kStats && blockIdx.x == 0) *a.ticket = 0;
    for (int s = 0; s < kStages; ++s) { mbar_init(&sm->full[s], 1); mbar_init(&sm->empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&sm->acc_full[b], 1); mbar_init(&sm->acc_empty[b], 16); }
    mbar_init(&sm->drain, 1);
    // an earlier launch gave up a wait: do nothing until the host resets
    sm->abort = *reinterpret_cast<volatile int*>(&g_loss_status) ? 2 : 0;
    fence_mbar_init();
  }
  if (warp == 2) tmem_alloc_pair(&sm->tmem_base, 512);
  tc_fence_before();
  __syncwarp();
  cluster_sync();
  tc_fence_after();
  const uint32_t tbase = sm->tmem_base;
  volatile int* abort = &sm->abort;

  // tile t -> split, row block, column block: gm row blocks at a time, rows first
  auto decode = [&](int t, int& m, int& n, int& k0, int& k1, int& split) {
    uint32_t sp, r, g, x, y;
    a.per_split.divmod(t, sp, r);
    a.per_group.divmod(r, g, r);
    if ((int)((g + 1) * a.gm) <= a.tiles_m) a.per_col.divmod(r, x, y);
    else a.per_col_last.divmod(r, x, y);
    m = g * a.gm + y;
    n = x;
    split = sp;
    const int q = a.kb / a.splits, rem = a.kb - q * a.splits;
    k0 = split * q + min(split, rem);
    k1 = k0 + q + (split < rem ? 1 : 0);
  };

  if (*abort == 0) {
    if (warp == 0) {
      // ---------------------------------------------------------- TMA producer
      if (lane == 0) {
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
        uint32_t it = 0;
        bool ok = true;
        for (int t = pair; t < total && ok; t += n_pairs) {
          int m, n, k0, k1, split;
          decode(t, m, n, k0, k1, split);
          const int ra = m * kTM + rank * 128, rb = n * kTN + rank * 128;
          for (int k = k0; k < k1; ++k, ++it) {
            const int s = it % kStages;
            const uint32_t round = it / kStages;
            if (round > 0 && !mbar_wait(&sm->empty[s], (round - 1) & 1, abort)) { ok = false; break; }
            if (rank == 0) mbar_expect_tx(&sm->full[s], 4 * kOpBytes);
            const uint32_t bar = leader_addr(&sm->full[s]);
            uint8_t* pa = sA + s * kOpBytes;
            uint8_t* pb = sB + s * kOpBytes;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if (kAMn) tma_load_2d_pair(pa + j * kBox, &tmA, bar, ra + 64 * j, k * kTK);
              else tma_load_2d_pair(pa + j * kBox, &tmA, bar, k * kTK, ra + 64 * j);
              if (kBMn) tma_load_2d_pair(pb + j * kBox, &tmB, bar, rb + 64 * j, a.b_off + k * kTK);
              else tma_load_2d_pair(pb + j * kBox, &tmB, bar, k * kTK, a.b_off + rb + 64 * j);
            }
          }
        }
        // the copies of the last stages have landed before the CTA may leave (on a
        // normal end the MMAs have already waited for them)
        if (!ok && rank == 0)
          for (uint32_t i = it > kStages ? it - kStages : 0; i < it; ++i)
            for (uint32_t p = 0; p < kSpinLimit && !mbar_try_wait(&sm->full[i % kStages], (i / kStages) & 1); ++p) {}
      }
    } else if (warp == 1 && rank == 0) {
      // ---------------------------------------------------------- MMA issuer
      if (lane == 0) {
        constexpr uint32_t idesc = idesc_bf16_f32(kTM, kTN, kAMn, kBMn);
        uint32_t it = 0;
        int li = 0;
        bool ok = true;
        // (Looking at the next stage's barrier, or waiting for the next accumulator, before a step's
        // MMAs are issued makes the kernel 3 to 8 % slower, not faster.)
        const int q = a.kb / a.splits, rem = a.kb - q * a.splits;
        for (int t = pair; t < total && ok; t += n_pairs, ++li) {
          const int steps = q + ((int)a.per_split.div(t) < rem ? 1 : 0);
          const int b = li & 1;
          const uint32_t acc = tbase + b * kTN;
          if (li >= 2 && !mbar_wait(&sm->acc_empty[b], ((li >> 1) - 1) & 1, abort)) break;
          tc_fence_after();
          for (int k = 0; k < steps; ++k, ++it) {
            const int s = it % kStages;
            if (!mbar_wait(&sm->full[s], (it / kStages) & 1, abort)) { ok = false; break; }
            tc_fence_after();
            const uint32_t pa = smem_u32(sA + s * kOpBytes), pb = smem_u32(sB + s * kOpBytes);
#pragma unroll
            for (int kk = 0; kk < kTK / 16; ++kk)
              mma_ss_pair(acc,
                          kAMn ? smem_desc_sw128(pa + kk * 2048, kBox, 1024) : smem_desc_sw128(pa + kk * 32, 16, 1024),
                          kBMn ? smem_desc_sw128(pb + kk * 2048, kBox, 1024) : smem_desc_sw128(pb + kk * 32, 16, 1024),
                          idesc, (k > 0 || kk > 0) ? 1u : 0u);
            mma_commit_pair(&sm->empty[s]);
          }
          if (ok) mma_commit_pair(&sm->acc_full[b]);
        }
        if (*abort) {                            // the MMAs issued so far end before TMEM is freed
          mma_commit_pair(&sm->drain);
          for (uint32_t p = 0; p < kSpinLimit && !mbar_try_wait(&sm->drain, 0); ++p) {}
        }
      }
    } else if (warp >= 4) {
      // ---------------------------------------------------------- epilogue
      // warps 4-7 take columns 0-127 of the tile, warps 8-11 the rest
      const int quad = warp & 3, half = warp >= 8 ? 1 : 0;
      constexpr int kCols = kTN / 2;
      const uint32_t lane_base = tbase + ((uint32_t)(quad * 32) << 16) + half * kCols;
      uint8_t* stage = sO + (quad + 4 * half) * kBufs * kOutBuf;
      const uint32_t acc_empty0 = leader_addr(&sm->acc_empty[0]), acc_empty1 = leader_addr(&sm->acc_empty[1]);
      int li = 0, buf = 0;
      // 16 bytes to chunk c of this thread's row of a staging tile (128-byte swizzle)
      auto put = [&](uint8_t* p, int c, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
        *reinterpret_cast<uint4*>(p + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(x, y, z, w);
      };
      for (int t = pair; t < total; t += n_pairs, ++li) {
        int m, n, k0, k1, split;
        decode(t, m, n, k0, k1, split);
        const int b = li & 1;
        const uint32_t acc = lane_base + b * kTN;
        const int row0 = m * kTM + rank * 128 + quad * 32, row = row0 + lane, n0 = n * kTN + half * kCols;
        const int cols = min(kCols, a.N - n0);           // of this warp's half, may be negative
        const bool live = row < a.M;
        // next target of this row at or behind the half's first column, as a column of the half,
        // and the one behind it, fetched ahead
        int cur = 0, next = kNone, after = kNone;
        const int g0 = MODE == kGrad ? a.b_off + n0 : n0;
        const int* idx = nullptr;
        auto advance = [&]() {
          ++cur;
          next = after == kNone ? kNone : after - g0;
          after = cur + 1 < a.K ? __ldg(idx + (size_t)(cur + 1) * a.M) : kNone;
        };
        float c = 0.f, lse2 = 0.f;
        if constexpr (MODE == kStats || MODE == kGrad) {
          if (live && cols > 0) {
            if constexpr (SPARSE) {
              idx = a.idx + row;
              cur = lower_bound(idx, a.K, a.M, g0) - 1;
              after = cur + 1 < a.K ? __ldg(idx + (size_t)(cur + 1) * a.M) : kNone;
              advance();
            } else {
              const long long tv = __ldg(a.target + row) - g0;
              if (tv >= 0 && tv < kCols) next = (int)tv;
            }
            if constexpr (MODE == kGrad) {
              const float up = __ldg(a.gout + (size_t)row * a.gstride);
              if (up != 0.f) c = a.cscale * up * __ldg(a.row_scale + row) * (a.inv_count ? __ldg(a.inv_count) : 1.f);
              lse2 = __ldg(a.lse2 + row);
            }
          }
        }
        const bool ok = mbar_wait(&sm->acc_full[b], (li >> 1) & 1, abort);
        if (__any_sync(~0u, !ok)) break;
        tc_fence_after();
        auto release = [&]() {                           // the tile's TMEM has been read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_leader(b ? acc_empty1 : acc_empty0);
        };
        if constexpr (MODE == kStats) {
          float mx = -INFINITY, sum = 0.f;
#pragma unroll 1
          for (int c0 = 0; c0 < kCols; c0 += 32) {
            const int left = cols - c0;
            if (left <= 0) break;
            uint32_t x[32];
            tmem_ld32(acc + c0, x);
            tmem_ld_wait();
            // logits of the targets among these columns, by way of this thread's row in shared memory
            if (__any_sync(~0u, next < c0 + 32)) {
#pragma unroll
              for (int ch = 0; ch < 8; ++ch) put(stage, ch, x[4 * ch], x[4 * ch + 1], x[4 * ch + 2], x[4 * ch + 3]);
              while (next < c0 + 32) {
                const int at = next - c0;
                a.slog[(size_t)cur * a.M + row] = *reinterpret_cast<const float*>(
                    stage + lane * 128 + (((at >> 2) ^ (lane & 7)) << 4) + (at & 3) * 4);
                if constexpr (SPARSE) advance();
                else next = kNone;
              }
            }
            if (left < 32) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (e >= left) x[e] = __float_as_uint(-INFINITY);
            }
            float mp[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 32; e += 2)
              mp[(e >> 1) & 3] = fmax3(mp[(e >> 1) & 3], __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
            const float mn = fmaxf(fmaxf(mx, fmaxf(mp[0], mp[1])), fmaxf(mp[2], mp[3]));
            const float mb = mn == -INFINITY ? 0.f : mn * a.a2;
            sum *= mx == -INFINITY ? 0.f : ex2(fmaf(mx, a.a2, -mb));
            mx = mn;
            float2 sp[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) sp[u] = make_float2(0.f, 0.f);
            const float2 a22 = make_float2(a.a2, a.a2), nb = make_float2(-mb, -mb);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 arg = ffma2(make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), a22, nb);
              sp[(e >> 1) & 3] = fadd2(sp[(e >> 1) & 3], make_float2(ex2(arg.x), ex2(arg.y)));
            }
            const float2 r = fadd2(fadd2(sp[0], sp[1]), fadd2(sp[2], sp[3]));
            sum += r.x + r.y;
          }
          release();
          if (live) a.stats[(size_t)(2 * n + half) * a.M + row] = make_float2(mx, sum);
        } else {
          const int width = MODE == kGrad || a.out == kOutBf16 ? 64 : 32;      // columns of one store
#pragma unroll 1
          for (int c0 = 0; c0 < kCols; c0 += width) {
            uint32_t x[32], y[32];
            tmem_ld32(acc + c0, x);
            if (width == 64) tmem_ld32(acc + c0 + 32, y);
            tmem_ld_wait();
            if (c0 + width == kCols) release();
            if (c0 >= cols || row0 >= a.M) continue;
            uint8_t* p = stage + buf * kOutBuf;
            if (lane == 0) bulk_wait_read_1();
            __syncwarp();
            if constexpr (MODE == kGrad) {
              if (c == 0.f) {                    // a row without a gradient, whatever its logits are
#pragma unroll
                for (int ch = 0; ch < 8; ++ch) put(p, ch, 0, 0, 0, 0);
              } else {
                auto grad = [&](uint32_t u) { return c * ex2(fmaf(__uint_as_float(u), a.a2, -lse2)); };
#pragma unroll
                for (int ch = 0; ch < 4; ++ch)
                  put(p, ch, pack_bf16(grad(x[8 * ch]), grad(x[8 * ch + 1])),
                      pack_bf16(grad(x[8 * ch + 2]), grad(x[8 * ch + 3])),
                      pack_bf16(grad(x[8 * ch + 4]), grad(x[8 * ch + 5])),
                      pack_bf16(grad(x[8 * ch + 6]), grad(x[8 * ch + 7])));
#pragma unroll
                for (int ch = 0; ch < 4; ++ch)
                  put(p, 4 + ch, pack_bf16(grad(y[8 * ch]), grad(y[8 * ch + 1])),
                      pack_bf16(grad(y[8 * ch + 2]), grad(y[8 * ch + 3])),
                      pack_bf16(grad(y[8 * ch + 4]), grad(y[8 * ch + 5])),
                      pack_bf16(grad(y[8 * ch + 6]), grad(y[8 * ch + 7])));
                while (next < c0 + 64) {         // the row's targets among these columns (the same one twice: twice alike)
                  const int at = next - c0;
                  *reinterpret_cast<__nv_bfloat16*>(p + lane * 128 + (((at >> 3) ^ (lane & 7)) << 4) + (at & 7) * 2) =
                      __float2bfloat16_rn(c * __ldg(a.gval + (size_t)cur * a.M + row));
                  if constexpr (SPARSE) advance();
                  else next = kNone;
                }
              }
            } else if (a.out == kOutBf16) {
#pragma unroll
              for (int ch = 0; ch < 4; ++ch) {
                auto pk = [&](const uint32_t* u) { return pack_bf16(__uint_as_float(u[0]), __uint_as_float(u[1])); };
                put(p, ch, pk(x + 8 * ch), pk(x + 8 * ch + 2), pk(x + 8 * ch + 4), pk(x + 8 * ch + 6));
                put(p, 4 + ch, pk(y + 8 * ch), pk(y + 8 * ch + 2), pk(y + 8 * ch + 4), pk(y + 8 * ch + 6));
              }
            } else {
#pragma unroll
              for (int ch = 0; ch < 8; ++ch) put(p, ch, x[4 * ch], x[4 * ch + 1], x[4 * ch + 2], x[4 * ch + 3]);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              if (MODE != kGrad && a.out == kOutPlaneAdd) tma_reduce_add_3d(&tmO, p, n0 + c0, row0, split);
              else tma_store_3d(&tmO, p, n0 + c0, row0, split);
              bulk_commit();
            }
            buf ^= 1;
          }
        }
      }
      if (lane == 0) bulk_wait_all();
    }
  }

  tc_fence_before();
  __syncwarp();
  cluster_sync();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc_pair(tbase, 512);
  }
  if (threadIdx.x == 0 && sm->abort) atomicExch(&g_loss_status, 1);
}

// ---------------------------------------------------------------- small kernels
// One warp per row: the K teacher entries sorted by vocabulary index (absent
// ones behind; stored (K, N)), their probabilities softmax(t / T) and sum p log p.  The rank of
// an entry is the number of entries before it, ties in their given order.
//   row_scale: 1, 0 for a row without entries, NaN for one with an index >= V or
//   a teacher logit that is NaN or +infinity
template <class T>
__global__ void __launch_bounds__(128)
teacher_kernel(const T* __restrict__ tv, const long long* __restrict__ ti, int N, int V, int K, float inv_t,
               int* __restrict__ idx, float* __restrict__ prob, float* __restrict__ ent, float* __restrict__ row_scale) {
  extern __shared__ int sh[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* key = sh + warp * K;
  const int row = blockIdx.x * 4 + warp;
  if (row >= N) return;
  const T* tr = tv + (size_t)row * K;
  const long long* ir = ti + (size_t)row * K;
  bool bad = false;
  float mx = -INFINITY;
  for (int k = lane; k < K; k += 32) {
    const long long i = ir[k];
    const bool here = i >= 0 && i < V;
    const float x = (float)tr[k] * inv_t;
    bad |= i >= V || (here && x != x);
    key[k] = here ? (int)i : kNone;
    if (here) mx = fmaxf(mx, x);
  }
  __syncwarp();
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
  bad = __any_sync(~0u, bad);
  float z = 0.f;
  for (int k = lane; k < K; k += 32)
    if (key[k] != kNone && mx != -INFINITY) z += expf((float)tr[k] * inv_t - mx);
#pragma unroll
  for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(~0u, z, o);
  const bool some = mx != -INFINITY;
  const float logz = logf(z);
  float e = 0.f;
  bool any_nan = false;
  for (int k = lane; k < K; k += 32) {
    const int me = key[k];
    int r = 0;
    for (int j = 0; j < K; ++j) r += key[j] < me || (key[j] == me && j < k);
    float p = 0.f;
    if (me != kNone && some) {
      const float x = (float)tr[k] * inv_t - mx - logz;
      p = expf(x);
      any_nan |= p != p;
      if (p > 0.f) e = fmaf(p, x, e);
    }
    idx[(size_t)r * N + row] = some ? me : kNone;
    prob[(size_t)r * N + row] = p;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) e += __shfl_xor_sync(~0u, e, o);
  any_nan = __any_sync(~0u, any_nan);
  if (lane == 0) {
    ent[row] = e;
    row_scale[row] = bad || any_nan ? __int_as_float(0x7fc00000) : some ? 1.f : 0.f;
  }
}

// Joins the (maximum, sum) parts of RB rows per block (thread = row of the block x
// slot of its parts, slots a power of two), forms the rows' losses and turns the
// targets' logits into exp(s - lse) - p, what the backward takes off the softmax.
// The last block to end adds up the blocks' (loss, count) in their order: the
// reduced loss (sum, or mean over the rows that count; 0 where none does) and
// 1 / count.
struct FinishArgs {
  const float2* stats;
  int parts, N, V, K, slots, reduction;
  const long long* target;
  long long ignore;
  const int* idx;
  const float *prob, *ent;
  float* slog;
  float a2, t2;
  float *row_scale, *lse2, *loss, *inv_count;
  double2* part;
  unsigned* ticket;
};

template <bool SPARSE, int RB>
__global__ void __launch_bounds__(1024)
finish_kernel(const FinishArgs a) {
  __shared__ float2 sh[1024];
  __shared__ double2 tot[32];
  __shared__ bool last;
  const int tid = threadIdx.x, r = tid % RB, slot = tid / RB, N = a.N, K = a.K;
  const int row = blockIdx.x * RB + r;
  auto join = [&](float2 u, float2 v) {
    const float mn = fmaxf(u.x, v.x);
    const float mb = mn == -INFINITY ? 0.f : mn * a.a2;
    return make_float2(mn, (u.x == -INFINITY ? u.y : u.y * ex2(fmaf(u.x, a.a2, -mb))) +
                               (v.x == -INFINITY ? v.y : v.y * ex2(fmaf(v.x, a.a2, -mb))));
  };
  float2 st = make_float2(-INFINITY, 0.f);
  if (row < N) {
#pragma unroll 4
    for (int t = slot; t < a.parts; t += a.slots) st = join(st, a.stats[(size_t)t * N + row]);
  }
  sh[tid] = st;
  __syncthreads();
  for (int o = a.slots >> 1; o; o >>= 1) {
    if (slot < o) sh[tid] = join(sh[tid], sh[tid + o * RB]);
    __syncthreads();
  }
  const float2 all = sh[r];
  const float l2 = fmaf(all.x, a.a2, log2f(all.y));
  float loss = 0.f, scale = 0.f;
  if constexpr (SPARSE) {
    float x = 0.f;
    if (row < N) {
      for (int k = slot; k < K; k += a.slots) {
        const size_t at = (size_t)k * N + row;
        const int me = a.idx[at];
        if (me == kNone) break;
        const float s = a.slog[at], p = a.prob[at];
        if (p > 0.f) x = fmaf(p, (l2 - s * a.a2) * kLn2, x);
        float same = p;                            // entries with the same index add up
        for (int j = k - 1; j >= 0 && a.idx[(size_t)j * N + row] == me; --j) same += a.prob[(size_t)j * N + row];
        for (int j = k + 1; j < K && a.idx[(size_t)j * N + row] == me; ++j) same += a.prob[(size_t)j * N + row];
        a.slog[at] = ex2(fmaf(s, a.a2, -l2)) - same;
      }
    }
    __syncthreads();                               // sh has been read
    sh[tid].x = x;
    __syncthreads();
    for (int o = a.slots >> 1; o; o >>= 1) {
      if (slot < o) sh[tid].x += sh[tid + o * RB].x;
      __syncthreads();
    }
    if (row < N && slot == 0) {
      scale = a.row_scale[row];
      if (scale != 0.f) loss = scale * a.t2 * (a.ent[row] + sh[r].x);
    }
  } else if (row < N && slot == 0) {
    const long long t = a.target[row];
    if (t != a.ignore) {
      const bool in = t >= 0 && t < a.V;
      scale = in ? 1.f : __int_as_float(0x7fc00000);
      loss = in ? l2 * kLn2 - a.slog[row] : scale;
      if (in) a.slog[row] = ex2(fmaf(a.slog[row], a.a2, -l2)) - 1.f;
    }
    a.row_scale[row] = scale;
  }
  if (row < N && slot == 0) {
    a.lse2[row] = l2;
    if (a.reduction == LH_REDUCE_NONE) a.loss[row] = loss;
  }
  if (a.reduction == LH_REDUCE_NONE) return;
  auto block_sum = [&](double& s, double& c) {     // to thread 0
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      s += __shfl_xor_sync(~0u, s, o);
      c += __shfl_xor_sync(~0u, c, o);
    }
    if ((tid & 31) == 0) tot[tid >> 5] = make_double2(s, c);
    __syncthreads();
    if (tid == 0)
      for (int w = 1; w < (int)blockDim.x / 32; ++w) { s += tot[w].x; c += tot[w].y; }
    __syncthreads();
  };
  double s = loss, c = scale != 0.f ? 1.0 : 0.0;   // zeros but in slot 0
  block_sum(s, c);
  if (tid == 0) {
    a.part[blockIdx.x] = make_double2(s, c);
    __threadfence();
    last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  s = c = 0;
#pragma unroll 4
  for (int i = tid; i < (int)gridDim.x; i += blockDim.x) {
    const double2 v = __ldcg(a.part + i);
    s += v.x;
    c += v.y;
  }
  block_sum(s, c);
  if (tid == 0) {
    const double inv = a.reduction == LH_REDUCE_MEAN ? (c > 0 ? 1.0 / c : 0.0) : 1.0;
    *a.loss = (float)(c > 0 ? s * inv : 0.0);
    *a.inv_count = (float)inv;
  }
}

// out (bf16) = sum of the fp32 planes (rows x cols each), in their order.
__global__ void __launch_bounds__(256)
planes_kernel(const float* __restrict__ planes, int n, size_t plane, __nv_bfloat16* __restrict__ out) {
  for (size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 8; i < plane; i += (size_t)gridDim.x * 256 * 8) {
    float v[8], u[8];
    load16(planes + i, v);
    load16(planes + i + 4, v + 4);
    for (int k = 1; k < n; ++k) {
      load16(planes + k * plane + i, u);
      load16(planes + k * plane + i + 4, u + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += u[e];
    }
    store16(out + i, v);
  }
}

// ---------------------------------------------------------------- host side
static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (PFN_cuTensorMapEncodeTiled_v12000)p;
  }();
  return fn;
}

// Encoding a tensor map is a driver call and needs a current context, which a
// thread that has only launched through another thread's calls (autograd's) may
// not have yet: cudaSetDevice makes the device's primary context current.
static int make_context_current() {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaSetDevice(dev);
  if (e != cudaSuccess) { set_error("linear loss: %s", cudaGetErrorString(e)); return LH_ERR_LAUNCH; }
  return LH_OK;
}

// bf16 (rows, cols) with a row pitch in elements; 64 x 64 boxes, 128-byte swizzle.
static int map_load(CUtensorMap* m, const void* p, long long rows, long long cols, long long pitch) {
  auto enc = encode_fn();
  if (!enc) { set_error("cuTensorMapEncodeTiled unavailable"); return LH_ERR_LAUNCH; }
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)pitch * 2};
  cuuint32_t box[2] = {64, 64}, es[2] = {1, 1};
  CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), dims, strides, box, es,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { set_error("linear loss: tensor map of an operand failed (%d)", (int)r); return LH_ERR_LAUNCH; }
  return LH_OK;
}
// Result (planes, rows, cols), bf16 or fp32; boxes of 32 rows x 128 bytes.
static int map_store(CUtensorMap* m, void* p, bool f32, long long planes, long long rows, long long cols, long long pitch) {
  auto enc = encode_fn();
  if (!enc) { set_error("cuTensorMapEncodeTiled unavailable"); return LH_ERR_LAUNCH; }
  const int es_ = f32 ? 4 : 2;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
  cuuint64_t strides[2] = {(cuuint64_t)pitch * es_, (cuuint64_t)(pitch * rows) * es_};
  cuuint32_t box[3] = {(cuuint32_t)(128 / es_), 32, 1}, es[3] = {1, 1, 1};
  CUresult r = enc(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, p, dims, strides, box,
                   es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { set_error("linear loss: tensor map of a result failed (%d)", (int)r); return LH_ERR_LAUNCH; }
  return LH_OK;
}

template <int MODE, bool SPARSE>
static int launch(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mo, Args a, long long K, cudaStream_t st) {
  a.tiles_m = (a.M + kTM - 1) / kTM;
  a.tiles_n = (a.N + kTN - 1) / kTN;
  a.kb = (int)((K + kTK - 1) / kTK);
  // Row blocks walked together: as many as keep their operand rows in about half of L2, at least
  // eight (eight by nine tiles are one wave of the 74 pairs).
  long long gm = (48ll << 20) / (kTM * 2ll * a.kb * kTK);
  if (gm < 8) gm = 8;
  a.gm = (int)(gm < a.tiles_m ? gm : a.tiles_m);
  a.per_split = FastDiv(a.tiles_m * a.tiles_n);
  a.per_group = FastDiv(a.gm * a.tiles_n);
  a.per_col = FastDiv(a.gm);
  a.per_col_last = FastDiv(a.tiles_m % a.gm ? a.tiles_m % a.gm : 1);
  const long long total = (long long)a.tiles_m * a.tiles_n * a.splits;
  const int pairs = (int)(total < kPairs ? total : kPairs);
  cudaError_t e = cudaFuncSetAttribute(loss_gemm_kernel<MODE, SPARSE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(MODE));
  if (e != cudaSuccess) { set_error("linear loss: %s", cudaGetErrorString(e)); return LH_ERR_LAUNCH; }
  loss_gemm_kernel<MODE, SPARSE><<<2 * pairs, kThreads, smem_bytes(MODE), st>>>(ma, mb, mo, a);
  return check_launch("loss_gemm_kernel");
}

// Parts of the K range of an (M, N) product: the number that makes the shortest
// rounds of the 74 pairs, counting an epilogue as six 64-deep steps and
// the planes' traffic.
static int pick_splits(long long M, long long N, long long K) {
  const long long tiles = ((M + kTM - 1) / kTM) * ((N + kTN - 1) / kTN), kb = (K + kTK - 1) / kTK;
  double best = 1e30;
  int pick = 1;
  for (int s = 1; s <= kPairs && s <= kb; ++s) {
    if (s > 1 && tiles * s > 4 * kPairs) break;
    const double rounds = (double)((tiles * s + kPairs - 1) / kPairs);
    const double cost = rounds * ((double)((kb + s - 1) / s) + 6.0) + (s > 1 ? 8.0 + 8.0 * s * M * N / 6.5e6 / 0.28 : 0.0);
    if (cost < best) { best = cost; pick = s; }
  }
  return pick;
}

struct Plan {
  long long C;                 // columns of a vocabulary piece, a multiple of 256
  int pieces, dh_splits, dw_splits;
  bool dh_planes;
  size_t g, dh, dw, total;     // bytes
};
constexpr long long kPieceBytes = 512ll << 20;

static size_t up(size_t n) { return (n + 255) & ~size_t(255); }

static Plan plan(long long N, long long V, long long D) {
  Plan p;
  long long C = kPieceBytes / (2 * N) / kTN * kTN;
  if (C < kTN) C = kTN;
  const long long Vp = (V + kTN - 1) / kTN * kTN;
  p.pieces = (int)((Vp + C - 1) / C);
  p.C = ((Vp + p.pieces - 1) / p.pieces + kTN - 1) / kTN * kTN;      // pieces of about equal size
  p.pieces = (int)((Vp + p.C - 1) / p.C);
  p.dh_splits = pick_splits(N, D, p.C < V ? p.C : V);
  p.dw_splits = pick_splits(p.C < V ? p.C : V, D, N);
  p.dh_planes = p.pieces > 1 || p.dh_splits > 1;
  p.g = up((size_t)N * p.C * 2);
  p.dh = p.dh_planes ? up((size_t)p.dh_splits * N * D * 4) : 0;
  p.dw = p.dw_splits > 1 ? up((size_t)p.dw_splits * p.C * D * 4) : 0;
  p.total = p.g + p.dh + p.dw;
  return p;
}

// stats, the blocks' sums and their ticket; distillation (K > 0): sum p log p and p of the rows
static size_t stats_bytes(long long N, long long V) {
  return up((size_t)((V + kTN - 1) / kTN) * 2 * N * sizeof(float2)) + up((size_t)((N + 7) / 8) * sizeof(double2)) + 256;
}
static size_t fwd_workspace(long long N, long long V, long long K) {
  return stats_bytes(N, V) + (K ? up((size_t)N * sizeof(float)) + up((size_t)N * K * sizeof(float)) : 0);
}

static int sum_planes(const float* planes, int n, size_t plane, void* out, cudaStream_t st) {
  size_t blocks = (plane / 8 + 255) / 256;
  if (blocks > 148 * 16) blocks = 148 * 16;
  planes_kernel<<<(unsigned)blocks, 256, 0, st>>>(planes, n, plane, (__nv_bfloat16*)out);
  return check_launch("planes_kernel");
}

struct Targets {
  const long long* target;   // cross entropy
  long long ignore;
  const int* idx;            // distillation
  int K;
  float T;
};

template <bool SPARSE>
static int forward(const void* hidden, const void* weight, int N, int V, int D, const Targets& tg, const float* prob,
                   const float* ent, int reduction, float* loss, float* lse2, float* slog, float* row_scale, float* inv_count, void* ws,
                   cudaStream_t st) {
  int rc = make_context_current();
  if (rc) return rc;
  CUtensorMap mh, mw;
  if ((rc = map_load(&mh, hidden, N, D, D)) || (rc = map_load(&mw, weight, V, D, D))) return rc;
  const int parts = (V + kTN - 1) / kTN * 2;
  float2* stats = (float2*)ws;
  double2* part = (double2*)((char*)ws + up((size_t)parts * N * sizeof(float2)));
  unsigned* ticket = (unsigned*)((char*)part + up((size_t)((N + 7) / 8) * sizeof(double2)));
  Args a{};
  a.M = N;
  a.N = V;
  a.splits = 1;
  a.target = tg.target;
  a.idx = tg.idx;
  a.K = tg.K;
  a.a2 = kLog2e / tg.T;
  a.stats = stats;
  a.slog = slog;
  a.ticket = ticket;
  if ((rc = launch<kStats, SPARSE>(mh, mw, mw, a, D, st))) return rc;
  // Rows per block: eight with up to 128 slots each where a row has many parts (16 rows of 1000
  // parts: 7 us, 17 with 32 rows per block), 256 where it has up to four (65536 rows of two parts:
  // 14 us with 32 rows per block, most of it the 2048 blocks' sum).
  const int want = parts > tg.K ? parts : tg.K;
  FinishArgs f{stats, parts, N, V, tg.K, 1, reduction, tg.target, tg.ignore, tg.idx, prob, ent, slog, a.a2, tg.T * tg.T,
               row_scale, lse2, loss, inv_count, part, ticket};
  const int rb = want > 32 ? 8 : want > 4 ? 32 : 256;
  while (f.slots < want && f.slots * rb < 1024) f.slots *= 2;
  const unsigned blocks = (unsigned)((N + rb - 1) / rb);
  if (rb == 8) finish_kernel<SPARSE, 8><<<blocks, rb * f.slots, 0, st>>>(f);
  else if (rb == 256) finish_kernel<SPARSE, 256><<<blocks, rb * f.slots, 0, st>>>(f);
  else finish_kernel<SPARSE, 32><<<blocks, rb * f.slots, 0, st>>>(f);
  return check_launch("finish_kernel");
}

template <bool SPARSE>
static int backward(const void* hidden, const void* weight, int N, int V, int D, const Targets& tg, const float* lse2,
                    const float* gval, const float* row_scale, const float* inv_count, const float* gout, int gstride,
                    void* dhidden, void* dweight, void* ws, cudaStream_t st) {
  int rc = make_context_current();
  if (rc) return rc;
  const Plan p = plan(N, V, D);
  char* g = (char*)ws;
  float* dh = (float*)(g + p.g);
  float* dw = (float*)(g + p.g + p.dh);
  CUtensorMap mh, mw, mdh, mdw, mg, mgo;
  if ((rc = map_load(&mh, hidden, N, D, D)) || (rc = map_load(&mw, weight, V, D, D))) return rc;
  if ((rc = p.dh_planes ? map_store(&mdh, dh, true, p.dh_splits, N, D, D) : map_store(&mdh, dhidden, false, 1, N, D, D)))
    return rc;
  for (int i = 0; i < p.pieces; ++i) {
    const long long v0 = i * p.C;
    const int cols = (int)(V - v0 < p.C ? V - v0 : p.C);
    if ((rc = map_load(&mg, g, N, cols, p.C)) || (rc = map_store(&mgo, g, false, 1, N, cols, p.C))) return rc;
    Args a{};
    a.M = N;
    a.N = cols;
    a.splits = 1;
    a.b_off = (int)v0;
    a.target = tg.target;
    a.idx = tg.idx;
    a.K = tg.K;
    a.a2 = kLog2e / tg.T;
    a.gval = gval;
    a.lse2 = lse2;
    a.row_scale = row_scale;
    a.inv_count = inv_count;
    a.gout = gout;
    a.gstride = gstride;
    a.cscale = tg.T;
    if ((rc = launch<kGrad, SPARSE>(mh, mw, mgo, a, D, st))) return rc;

    Args x{};
    x.M = N;
    x.N = D;
    const int kb = (cols + kTK - 1) / kTK;
    x.splits = p.dh_splits < kb ? p.dh_splits : kb;      // a short last piece may leave planes as they are
    x.b_off = (int)v0;
    x.out = !p.dh_planes ? kOutBf16 : i ? kOutPlaneAdd : kOutPlane;
    if ((rc = launch<kDH, false>(mg, mw, mdh, x, cols, st))) return rc;

    Args y{};
    y.M = cols;
    y.N = D;
    y.splits = p.dw_splits;
    y.out = p.dw_splits > 1 ? kOutPlane : kOutBf16;
    char* dw_out = (char*)dweight + (size_t)v0 * D * 2;
    if ((rc = p.dw_splits > 1 ? map_store(&mdw, dw, true, p.dw_splits, cols, D, D)
                              : map_store(&mdw, dw_out, false, 1, cols, D, D)))
      return rc;
    if ((rc = launch<kDW, false>(mg, mh, mdw, y, N, st))) return rc;
    if (p.dw_splits > 1 && (rc = sum_planes(dw, p.dw_splits, (size_t)cols * D, dw_out, st))) return rc;
  }
  return p.dh_planes ? sum_planes(dh, p.dh_splits, (size_t)N * D, dhidden, st) : LH_OK;
}

}  // namespace ll

size_t linear_loss_workspace_size(int N, int V, int D, int K, int backward) {
  return backward ? ll::plan(N, V, D).total : ll::fwd_workspace(N, V, K);
}

int linear_xent_fwd(const void* hidden, const void* weight, const long long* target, long long ignore, int N, int V, int D,
                    int reduction, float* loss, float* lse2, float* tgrad, float* row_scale, float* inv_count, void* ws,
                    cudaStream_t st) {
  const ll::Targets tg{target, ignore, nullptr, 1, 1.f};
  return ll::forward<false>(hidden, weight, N, V, D, tg, nullptr, nullptr, reduction, loss, lse2, tgrad, row_scale, inv_count, ws, st);
}

int linear_xent_bwd(const void* hidden, const void* weight, const long long* target, int N, int V, int D, const float* lse2,
                    const float* tgrad, const float* row_scale, const float* inv_count, const float* gout, int gstride,
                    void* dhidden, void* dweight, void* ws, cudaStream_t st) {
  const ll::Targets tg{target, 0, nullptr, 1, 1.f};
  return ll::backward<false>(hidden, weight, N, V, D, tg, lse2, tgrad, row_scale, inv_count, gout, gstride, dhidden,
                             dweight, ws, st);
}

int linear_distill_fwd(const void* hidden, const void* weight, const void* tv, int tv_dtype, const long long* ti, int N,
                       int V, int D, int K, float T, int reduction, float* loss, float* lse2, int* idx, float* tgrad,
                       float* row_scale, float* inv_count, void* ws, cudaStream_t st) {
  float* ent = (float*)((char*)ws + ll::stats_bytes(N, V));
  float* prob = (float*)((char*)ent + ll::up((size_t)N * sizeof(float)));
  const unsigned blocks = (unsigned)((N + 3) / 4);
  if (tv_dtype == LH_DTYPE_BF16)
    ll::teacher_kernel<<<blocks, 128, 4 * K * sizeof(int), st>>>((const __nv_bfloat16*)tv, ti, N, V, K, 1.f / T, idx, prob,
                                                                ent, row_scale);
  else
    ll::teacher_kernel<<<blocks, 128, 4 * K * sizeof(int), st>>>((const float*)tv, ti, N, V, K, 1.f / T, idx, prob, ent,
                                                                row_scale);
  int rc = check_launch("teacher_kernel");
  if (rc) return rc;
  const ll::Targets tg{nullptr, 0, idx, K, T};
  return ll::forward<true>(hidden, weight, N, V, D, tg, prob, ent, reduction, loss, lse2, tgrad, row_scale, inv_count, ws, st);
}

int linear_distill_bwd(const void* hidden, const void* weight, int N, int V, int D, int K, float T, const float* lse2,
                       const int* idx, const float* tgrad, const float* row_scale,
                       const float* inv_count, const float* gout, int gstride, void* dhidden, void* dweight, void* ws,
                       cudaStream_t st) {
  const ll::Targets tg{nullptr, 0, idx, K, T};
  return ll::backward<true>(hidden, weight, N, V, D, tg, lse2, tgrad, row_scale, inv_count, gout, gstride, dhidden,
                            dweight, ws, st);
}

int loss_status(int reset) {
  int h = 0;
  cudaMemcpyFromSymbol(&h, g_loss_status, sizeof(int));
  if (reset) { int z = 0; cudaMemcpyToSymbol(g_loss_status, &z, sizeof(int)); }
  return h;
}

}  // namespace lh
