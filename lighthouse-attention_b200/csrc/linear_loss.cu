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
// error of up to 2^-8 is that of the bf16 gradients it ends in (up to 32 rows: two
// terms, 2^-16; see kTwo).  Two terms everywhere would double the products of dH and
// dW, half of a training call.  All sums are fp32.
// Where the loss is reduced, c is the same for all rows: G / c is what is rounded, and
// dH and dW are multiplied by c in fp32.  The targets' entries, the largest ones, are
// then near -1, which bf16 holds, where G's would all be off by c's own rounding (434 x
// 967 x 296, mean: dH off by 0.0025 of itself, 0.0021 so; 0.0017 is dH's rounding).
//
// Where a row's vocabulary is one tile (V <= 256) and the loss is reduced, the forward
// knows a row's lse when its tile ends, and writes G / c there: the backward has one
// product and a reading of hidden less.
//
// Rows without a target (ignored positions, rows without a teacher) are left out of
// all products where those are long enough to pay for it: the rows that count are
// packed, and the kernels take their number from device memory.  Elsewhere their rows
// of G are zeros, and should one of them hold an infinity or a NaN, which a zero does
// not take out of a product, dW is formed with a copy of hidden that has zeros there.
// Whatever such a row holds, it reaches nothing.
//
// One persistent GEMM kernel does all four products: a pair of SMs
// (tcgen05.mma.cta_group::2) per 256 x 256 tile, so that each SM loads 128 rows
// of either operand and both accumulators (2 x 256 TMEM columns) alternate
// between the MMAs of one tile and the epilogue of the one before.  Roles: warp
// 0 TMA producer, warp 1 MMA issuer (leader's), warps 4-11 epilogue (thread = row
// = TMEM lane, two warps per row block, half the columns each).  Operands are
// K-major or MN-major as they lie in memory: no transposed copy exists.  Where a
// product has few tiles, its K range is split and the parts meet in fp32 planes
// which planes_kernel sums in a fixed order.
// Every mbarrier wait is bounded; on expiry the CTAs leave and a status flag is set.  Launches that find the
// flag set compute nothing; losses, and gradients that miss a tile, are NaN then.
#include <cudaTypedefs.h>

#include <atomic>
#include <type_traits>

#include "lh_common.cuh"
#include "sm100.cuh"

namespace lh {

using namespace sm100;

__device__ int g_loss_status;    // set to 1 when a bounded wait gave up
// One thread of a block asks: 16000 warps that read one address take 3 us.
__device__ __forceinline__ bool gave_up() { return *reinterpret_cast<volatile int*>(&g_loss_status) != 0; }

namespace ll {

constexpr int kTM = 256, kTN = 256, kTK = 64;    // tile of a pair of SMs
constexpr int kBox = 64 * 64 * 2;                // one 64 x 64 bf16 TMA box, 128-byte rows
constexpr int kOpBytes = 2 * kBox;               // 128 rows of an operand: one CTA's share of a stage
constexpr int kThreads = 384;
constexpr int kOutBuf = 4096;                    // 32 rows x 128 bytes: one store of an epilogue warp
constexpr int kPairs = 74;
constexpr int kNone = 0x7fffffff;
constexpr float kLn2 = 0.69314718055994531f;

enum Mode { kStats, kWhole, kGrad, kDH, kDW };      // kWhole: kStats and kGrad of rows of one tile
enum Out { kOutBf16, kOutPlane, kOutPlaneAdd };

// With few rows (kFew at most) the roles turn: the 256 rows of a tile are weights (or
// columns of dH) and its kFew columns are rows of hidden, so that the MMAs do an eighth
// of the work and the stages hold weights, which are what has to be read.
constexpr int kFew = 64;
// Up to kTwo rows, G is the sum of two bf16 terms, the second one's rows kTwo behind, off by 2^-16: the columns of
// the MMAs and the rows of a K step are there anyway (16 x 32000 x 4096, forward and backward: 243 us, 234 with one
// term; 32 x 128000 x 2048: 426, 421), and a gradient of so few positions is a handful of entries, whose roundings
// do not cancel over it.  Beyond, one term: the whole of dH and dW is off by 0.0019 to 0.0024 of itself (0.0017 is
// the rounding of the results), and a single row of dH, or one of dW that comes from one position, by up to 2^-8
// from its largest entry of G besides its own rounding.  The rule looks at the rows that are there, not at those
// that count, as the launches cannot know them.
constexpr int kTwo = kFew / 2;
// A stage holds two steps of 64: its eight MMAs are issued without a stop, as each wait for a
// stage and each commit of one leaves the tensor pipe empty for about 100 cycles, whatever waits
// (4096 x 32000 x 4096, forward: 790 us with six stages of one step, 830 with a wait or a commit
// per step and the other per two; 760 with three stages of two; 855 with two of three, which
// leaves the loads too little room).  One store's staging buffer per epilogue warp: two, and a
// step less of operands, are 1 to 2 % slower.
constexpr int kSubs = 2;
// Adding products the tensor core cuts the sum towards zero, which makes a logit of D products smaller by
// about 1e-9 D of itself, by twice that where its large products come first, by nothing where they come
// last or the sum is exact: no factor takes that out.  So the forward sums a logit in parts of kPart steps,
// which the epilogue adds in registers, rounding to nearest; what is lost no longer grows with D.  (65536 x
// 256 x 1024, the mean's error, the forward alone and with the backward: 2.7e-6, 50 and 150 us in one part,
// 1.3e-6, 50 and 152 in parts of 8 steps, 0.9e-6, 50 and 154 of 6, 0.6e-6, 54 and 162 of 4, whose accumulators
// the epilogue does not keep up with: the forward of 1999 x 50261 x 768 takes 100, 98, 98 and 113 us.)  The
// backward's logits are one sum: their exponentials are rounded to 2^-9.
constexpr int kPart = 6;
// Registers per thread of warps 0-3 and of the epilogue's in that forward; together the launch's 384 x 168 (a launch
// with less would wait for ever: launch() asks how many the kernel was compiled to).
constexpr int kRegsRoles = 40, kRegsEpilogue = 232;
__host__ __device__ constexpr int stages(bool few) { return few ? 5 : 3; }
__host__ __device__ constexpr int b_bytes(bool few) { return few ? kFew / 2 * 128 : kOpBytes; }
constexpr int smem_bytes(bool few) {
  return 1024 + stages(few) * kSubs * (kOpBytes + b_bytes(few)) + (few ? 0 : 8 * kOutBuf) + 512;
}

// Walk of the tiles: split, group of gm row blocks, column block, row block in the group.
struct Sched {
  int M, tiles_m, gm, kb, splits, total, packed;
  FastDiv div[4];                 // by the tiles of a split, of a group, of its columns, of the last group's
  __host__ __device__ uint32_t divisor(int i, int tiles_n) const {
    const uint32_t d = i == 0 ? tiles_m * tiles_n : i == 1 ? gm * tiles_n : i == 2 ? gm : gm ? tiles_m % gm : 0;
    return d ? d : 1;
  }
};

struct Smem {
  uint64_t full[5], empty[5], acc_full[2], acc_empty[2], drain;
  Sched sched;
  uint32_t tmem_base;
  int abort;
};
static_assert(sizeof(Smem) <= 512, "barriers do not fit their space");
static_assert(smem_bytes(false) <= 232448 && smem_bytes(true) <= 232448, "stages do not fit shared memory");

constexpr int kSplitTable = 2 * kPairs;
struct Args {
  int M, N;                       // rows and columns of the result
  int tiles_n, splits, kb, gm;
  Sched sched;                    // of all rows
  int n_rows;                     // rows of hidden
  const int* rows;                // NULL, or: number of packed rows, their rows of hidden, (and back)
  uint8_t split_of[kSplitTable];  // kDH: parts of the K range by the number of row blocks, 1 beyond the table
  int b_off;                      // first row of the weights, B's operand (few rows: A's): vocabulary piece
  int out;                        // kDH, kDW: Out
  // targets: int64 (K = 1, SPARSE false) or sorted int32 (n_rows, K), K a multiple of four then
  const long long* target;
  const int* idx;
  int K;
  float a2;                       // exponent_scale()
  float2* stats;                  // kStats: (2 tiles_n, n_rows) maximum and sum of a row's 128 columns
  float* slog;                    // kStats: logits of the targets (n_rows, K) out
  unsigned* ticket;               // forward: set to 0 for finish_kernel
  int* dirty;                     // forward: set to 0 for finish_kernel; kDW: B is tmP where it is not 0
  const float* gval;              // kGrad: exp(s - lse) - p at the targets (n_rows, K)
  const float* prob;              // kWhole: p at the targets (n_rows, K), not read where SPARSE is false
  long long ignore;               // kWhole, SPARSE false
  const float* lse2;              // kGrad: log2-sum-exp2 of s a2
  const float *gout, *row_scale, *inv_count;       // gout NULL: c is row_scale (kGrad), or 1 (kDH, kDW)
  float cscale;
  int two;                        // few rows: G has two terms
  void* result;                   // kDH, kDW: what the tiles go to (bf16, or fp32 planes); few rows, kGrad: G (few_pitch)
  long long few_pitch;
};

// Position of the first of a row's K sorted targets that is >= v.
__device__ __forceinline__ int lower_bound(const int* idx, int K, int v) {
  int lo = 0, hi = K;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (idx[mid] < v) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}
// A row's K values (K a multiple of four) read one after the other: four at a time, the
// next four on their way meanwhile (single loads leave a row waiting for each target).
template <class V4, class V>
struct Window {
  const V4* p;
  V4 now, behind;
  __device__ __forceinline__ void open(const V* row, int K, int at, V none) {
    p = reinterpret_cast<const V4*>(row);
    const V4 empty{none, none, none, none};
    const int g = at >> 2;
    now = at < K ? p[g] : empty;
    behind = (g + 1) * 4 < K ? p[g + 1] : empty;
    for (int k = at & 3; k; --k) shift();
  }
  __device__ __forceinline__ void shift() { now.x = now.y; now.y = now.z; now.z = now.w; }
  // to position `at`, the one behind the last
  __device__ __forceinline__ void step(int K, int at, V none) {
    if (at & 3) { shift(); return; }
    now = behind;
    if (at + 4 < K) behind = p[(at >> 2) + 1];
    else behind = V4{none, none, none, none};
  }
};

// Barriers of the two warps that hold the halves of a row block's columns.
__device__ __forceinline__ void pair_sync(int id) {
  __syncwarp();
  asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory");
}
__device__ __forceinline__ bool pair_all(int id, bool v) {
  uint32_t r;
  __syncwarp();
  asm volatile("{.reg .pred p, q; setp.ne.u32 p, %1, 0; bar.red.and.pred q, %2, 64, p; selp.u32 %0, 1, 0, q;}"
               : "=r"(r) : "r"((uint32_t)v), "r"(id) : "memory");
  return r;
}

// A row's sum of exponentials is relative to 2^scaled(m, a2), m its maximum so far: where the
// maximum moves, the sum is multiplied by 2^(scaled(old) - scaled(new)), which is one where it
// stays.  (With the unrounded m a2 in the place of one of the two, every join would multiply the
// sum by the rounding of m a2 once more: 1e-5 of a row whose largest logit is 20, 7e-5 at 90.)
__device__ __forceinline__ float scaled(float m, float a2) { return m == -INFINITY ? 0.f : __fmul_rn(m, a2); }

// 32 values per lane, one per column -> in lane e the result of column e over the warp.
template <class Op>
__device__ __forceinline__ float reduce_columns(float (&v)[32], int lane, Op op) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = up ? v[i + o] : v[i], give = up ? v[i] : v[i + o];
      v[i] = op(keep, __shfl_xor_sync(~0u, give, o));
    }
  }
  return v[0];
}

template <int MODE, bool SPARSE, bool FEW>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
loss_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmP,
                 const __grid_constant__ Args a) {
  // tmP: the packed rows, in the place of hidden (A of kStats and kGrad, B of kDW)
  constexpr bool kParts = MODE == kStats || MODE == kWhole;
  constexpr bool kAMn = MODE == kDW || (FEW && MODE == kDH), kBMn = !FEW && (MODE == kDH || MODE == kDW);
  constexpr int kStages = stages(FEW), kBBytes = b_bytes(FEW);
  constexpr int kCols = FEW ? kFew : kTN;          // columns of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = base;
  uint8_t* sB = base + kStages * kSubs * kOpBytes;
  uint8_t* sO = base + kStages * kSubs * (kOpBytes + kBBytes);
  Smem* sm = reinterpret_cast<Smem*>(sO + (FEW ? 0 : 8 * kOutBuf));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    for (int s = 0; s < kStages; ++s) { mbar_init(&sm->full[s], 1); mbar_init(&sm->empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&sm->acc_full[b], 1); mbar_init(&sm->acc_empty[b], 16); }
    mbar_init(&sm->drain, 1);
    fence_mbar_init();
  }
  if (warp == 2) tmem_alloc_pair(&sm->tmem_base, 512);
  __syncwarp();
  after_previous();                // nothing above touches global memory
  if (warp == 3) {
    // The walk of the host's numbers, or of the packed rows' (each divisor by a lane of its own).
    const int live = a.rows ? *a.rows : a.n_rows;
    if (live == a.n_rows) {
      if (lane == 0) sm->sched = a.sched;
    } else {
      Sched c;
      c.M = MODE == kDW ? a.M : live;
      c.kb = MODE == kDW ? (live + kTK - 1) / kTK : a.kb;
      c.packed = 1;
      c.tiles_m = (c.M + kTM - 1) / kTM;
      c.gm = max(1, min(a.gm, c.tiles_m));
      c.splits = a.splits;
      if (MODE == kDH) c.splits = max(1, min(a.splits, c.tiles_m < kSplitTable ? (int)a.split_of[c.tiles_m] : 1));
      c.total = c.tiles_m * a.tiles_n * c.splits;
      const FastDiv mine(c.divisor(lane & 3, a.tiles_n));
      if (lane < 4) sm->sched.div[lane] = mine;
      if (lane == 0) {
        sm->sched.M = c.M; sm->sched.tiles_m = c.tiles_m; sm->sched.gm = c.gm; sm->sched.kb = c.kb;
        sm->sched.splits = c.splits; sm->sched.total = c.total; sm->sched.packed = 1;
      }
    }
    if (lane == 0) {
      if ((MODE == kStats || MODE == kWhole) && blockIdx.x == 0) { *a.ticket = 0; *a.dirty = 0; }
      // an earlier launch gave up a wait: do nothing until the host resets
      sm->abort = gave_up() ? 2 : 0;
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync();
  tc_fence_after();
  const uint32_t tbase = sm->tmem_base;
  volatile int* abort = &sm->abort;
  const Sched& sched = sm->sched;
  const int total = sched.total, M = sched.M;
  auto upstream = [&]() {                                // c of a reduced loss
    const float up = *a.gout;
    return up == 0.f ? 0.f : a.cscale * up * *a.inv_count;
  };

  // tile t -> split, row block, column block
  auto decode = [&](int t, int& m, int& n, int& k0, int& k1, int& split) {
    uint32_t sp, r, g, x, y;
    sched.div[0].divmod(t, sp, r);
    sched.div[1].divmod(r, g, r);
    sched.div[(int)((g + 1) * sched.gm) <= sched.tiles_m ? 2 : 3].divmod(r, x, y);
    m = g * sched.gm + y;
    n = x;
    split = sp;
    const int q = sched.kb / sched.splits, rem = sched.kb - q * sched.splits;
    k0 = split * q + min(split, rem);
    k1 = k0 + q + (split < rem ? 1 : 0);
  };

  // A thread of the epilogue holds its half row of logits: registers of warps 0-3 go there.
  if (warp < 4) {
    if constexpr (kParts && !FEW) regs_shrink<kRegsRoles>();
    if (warp == 0 && *abort == 0) {
      // ---------------------------------------------------------- TMA producer
      // (The whole warp runs this role and the next one, one lane of it issues: with a single lane in a
      // branch the operands of each copy and MMA pass through vector registers; 1 to 3 % of the time.)
      const CUtensorMap* mapA = kAMn || MODE == kDH || !sched.packed ? &tmA : &tmP;
      const CUtensorMap* mapB = MODE == kDW && (sched.packed || a.two || (a.dirty && *a.dirty)) ? &tmP : &tmB;
      uint32_t it = 0;
      bool ok = true;
      for (int t = pair; t < total && ok; t += n_pairs) {
        int m, n, k0, k1, split;
        decode(t, m, n, k0, k1, split);
        const int ra = m * kTM + rank * 128, rb = n * kCols + rank * (kCols / 2);
        for (int kg = k0; kg < k1; kg += kSubs, ++it) {
          const int s = it % kStages;
          const uint32_t round = it / kStages;
          if (round > 0) ok = mbar_wait(&sm->empty[s], (round - 1) & 1, abort);
          if (__any_sync(~0u, !ok)) { ok = false; break; }
          if (elect_one()) {
            const int n_sub = min(kSubs, k1 - kg);
            if (rank == 0) mbar_expect_tx(&sm->full[s], n_sub * 2 * (kOpBytes + kBBytes));
            const uint32_t bar = leader_addr(&sm->full[s]);
#pragma unroll
            for (int u = 0; u < kSubs; ++u) {
              if (u < n_sub) {
                const int k = kg + u;
                uint8_t* pa = sA + (s * kSubs + u) * kOpBytes;
                uint8_t* pb = sB + (s * kSubs + u) * kBBytes;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  const int a_row = ra + 64 * j + (FEW && !kAMn ? a.b_off : 0), a_k = k * kTK + (FEW && kAMn ? a.b_off : 0);
                  if (kAMn) tma_load_2d_pair(pa + j * kBox, mapA, bar, a_row, a_k);
                  else tma_load_2d_pair(pa + j * kBox, mapA, bar, a_k, a_row);
                }
                if constexpr (FEW) {
                  tma_load_2d_pair(pb, mapB, bar, k * kTK, rb);
                } else {
#pragma unroll
                  for (int j = 0; j < 2; ++j) {
                    if (kBMn) tma_load_2d_pair(pb + j * kBox, mapB, bar, rb + 64 * j, a.b_off + k * kTK);
                    else tma_load_2d_pair(pb + j * kBox, mapB, bar, k * kTK, a.b_off + rb + 64 * j);
                  }
                }
              }
            }
          }
          __syncwarp();
        }
      }
      // no copy is in flight when the CTAs leave, whatever the other roles waited for (the
      // leader's barriers count the copies of both)
      if (rank == 0 && lane == 0)
        for (uint32_t i = it > kStages ? it - kStages : 0; i < it; ++i)
          for (uint32_t p = 0; p < kSpinLimit && !mbar_try_wait(&sm->full[i % kStages], (i / kStages) & 1); ++p) {}
    } else if (warp == 1 && rank == 0 && *abort == 0) {
      // ---------------------------------------------------------- MMA issuer
      constexpr uint32_t idesc = idesc_bf16_f32(kTM, kCols, kAMn, kBMn);
      uint32_t it = 0;
      int li = 0;                                        // accumulators so far
      bool ok = true;
      // (Looking at the next stage's barrier, or waiting for the next accumulator, before a stage's
      // MMAs are issued makes the kernel 3 to 8 % slower, not faster.)
      const int q = sched.kb / sched.splits, rem = sched.kb - q * sched.splits;
      for (int t = pair; t < total && ok; t += n_pairs) {
        const int steps = q + ((int)sched.div[0].div(t) < rem ? 1 : 0);
        int from = 0;
        do {                                             // a part, or all steps
          const int to = kParts ? min(from + kPart, steps) : steps, b = li & 1;
          const uint32_t acc = tbase + b * kCols;
          if (li >= 2) ok = mbar_wait(&sm->acc_empty[b], ((li >> 1) - 1) & 1, abort);
          if (__any_sync(~0u, !ok)) { ok = false; break; }
          tc_fence_after();
          for (int kg = from; kg < to; kg += kSubs, ++it) {
            const int s = it % kStages;
            ok = mbar_wait(&sm->full[s], (it / kStages) & 1, abort);
            if (__any_sync(~0u, !ok)) { ok = false; break; }
            tc_fence_after();
            const int n_sub = min(kSubs, to - kg);
            if (elect_one()) {
#pragma unroll
              for (int u = 0; u < kSubs; ++u) {
                if (u < n_sub) {
                  const uint32_t pa = smem_u32(sA + (s * kSubs + u) * kOpBytes), pb = smem_u32(sB + (s * kSubs + u) * kBBytes);
#pragma unroll
                  for (int kk = 0; kk < kTK / 16; ++kk)
                    mma_ss_pair(acc,
                                kAMn ? smem_desc_sw128(pa + kk * 2048, kBox, 1024) : smem_desc_sw128(pa + kk * 32, 16, 1024),
                                kBMn ? smem_desc_sw128(pb + kk * 2048, kBox, 1024) : smem_desc_sw128(pb + kk * 32, 16, 1024),
                                idesc, (kg + u > from || kk > 0) ? 1u : 0u);
                }
              }
              mma_commit_pair(&sm->empty[s]);
              if (kg + kSubs >= to) mma_commit_pair(&sm->acc_full[b]);
            }
            __syncwarp();
          }
          if (steps == 0 && elect_one()) mma_commit_pair(&sm->acc_full[b]);
          __syncwarp();
          ++li;
          from = to;
        } while (ok && from < steps);
      }
      if (__any_sync(~0u, *abort) && elect_one()) {      // the MMAs issued so far end before TMEM is freed
        mma_commit_pair(&sm->drain);
        for (uint32_t p = 0; p < kSpinLimit && !mbar_try_wait(&sm->drain, 0); ++p) {}
      }
    }
  } else {
    if constexpr (kParts && !FEW) regs_grow<kRegsEpilogue>();
    if (*abort != 0) {
      // nothing to do
    } else if constexpr (FEW) {
      // ---------------------------------------------------------- epilogue, few rows
      // TMEM lane = row of the weights (column of dH), 32 columns per warp = rows of hidden; what
      // belongs to a row of hidden is held by the lane of its number and handed out by shuffles
      const int quad = warp & 3, half = warp >= 8 ? 1 : 0;
      const uint32_t acc0 = tbase + ((uint32_t)(quad * 32) << 16) + half * 32;
      const uint32_t acc_empty0 = leader_addr(&sm->acc_empty[0]), acc_empty1 = leader_addr(&sm->acc_empty[1]);
      const int row = half * 32 + lane;
      const bool live = row < a.N;
      const int rows = min(32, a.N - half * 32);         // of this warp, may be negative
      float mx = -INFINITY, sum = 0.f, c = 0.f, lse2 = 0.f;
      const float alpha = MODE == kDH && a.gout ? upstream() : 1.f;
      long long target = -1;
      if constexpr (MODE == kStats || MODE == kGrad) {
        if (live && !SPARSE) target = a.target[row];
        if (MODE == kGrad && live) {
          const float up = a.gout ? a.cscale * a.gout[row] : 1.f;
          if (up != 0.f) c = up * a.row_scale[row];
          lse2 = a.lse2[row];
        }
      }
      int li = 0;                                        // accumulators so far
      const int parts = kParts ? (sched.kb + kPart - 1) / kPart : 1;
      for (int t = pair; t < total; t += n_pairs) {
        int m, n, k0, k1, split;
        decode(t, m, n, k0, k1, split);
        const int v0 = m * kTM + rank * 128 + quad * 32;
        const int left = min(32, M - v0);                // rows of the weights, may be negative
        const bool two = MODE == kDH && a.two;           // the other half's columns are the same rows' other term
        uint32_t x[32], y[32];
        bool ok = true;
        for (int p = 0; p < parts; ++p, ++li) {
          const int b = li & 1;
          ok = mbar_wait(&sm->acc_full[b], (li >> 1) & 1, abort);
          if (__any_sync(~0u, !ok)) { ok = false; break; }
          tc_fence_after();
          if (!kParts || p == 0) tmem_ld32(acc0 + b * kCols, x);
          else tmem_ld32(acc0 + b * kCols, y);
          if (two) tmem_ld32(acc0 + b * kCols + (half ? -kTwo : kTwo), y);
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_leader(b ? acc_empty1 : acc_empty0);
          if (kParts && p > 0) {
#pragma unroll
            for (int e = 0; e < 32; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) + __uint_as_float(y[e]));
          }
        }
        if (!ok) break;
        if (left <= 0 || (rows <= 0 && !two)) continue;
        if constexpr (MODE == kDH) {
          const int row0 = two ? 0 : half * 32;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            if (two) x[e] = __float_as_uint(__uint_as_float(x[e]) + __uint_as_float(y[e]));
            if ((two ? e < a.N && e / 16 == half : e < rows) && lane < left) {
              const size_t at = (size_t)(row0 + e) * a.M + v0 + lane;
              const float d = alpha == 0.f ? 0.f : alpha * __uint_as_float(x[e]);
              if (a.out == kOutBf16) reinterpret_cast<__nv_bfloat16*>(a.result)[at] = __float2bfloat16_rn(d);
              else reinterpret_cast<float*>(a.result)[(size_t)split * a.N * a.M + at] = d;
            }
          }
        } else {
          auto put_g = [&](int e, float v) {             // G of row e
            __nv_bfloat16* g = reinterpret_cast<__nv_bfloat16*>(a.result) + (half * 32 + e) * a.few_pitch + v0 + lane;
            const __nv_bfloat16 first = __float2bfloat16_rn(v);
            *g = first;
            const float rest = v - __bfloat162float(first);      // not a number where v is infinite
            if (a.two) g[kTwo * a.few_pitch] = __float2bfloat16_rn(fabsf(v) < INFINITY && fabsf(rest) < INFINITY ? rest : 0.f);
          };
          // dense part
          if constexpr (MODE == kGrad) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float ce = __shfl_sync(~0u, c, e), le = __shfl_sync(~0u, lse2, e);
              // (rows up to kTwo that are none are zeros: kDW's step takes them)
              if ((e < rows || a.two) && lane < left)
                put_g(e, e >= rows || ce == 0.f ? 0.f : ce * ex2(fmaf(__uint_as_float(x[e]), a.a2, -le)));
            }
          }
          // the rows' targets among these weights
          const int gv0 = v0 + (MODE == kGrad ? a.b_off : 0);
          int cur = 0, next = kNone;
          if (live) {
            if constexpr (SPARSE) {
              cur = lower_bound(a.idx + row * a.K, a.K, gv0);
              if (cur < a.K) next = a.idx[row * a.K + cur];
              if (next != kNone) next -= gv0;
            } else if (target >= gv0 && target < gv0 + 32) {
              next = (int)(target - gv0);
            }
          }
          for (unsigned hit; (hit = __ballot_sync(~0u, next < left)) != 0;) {
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              if (hit >> e & 1) {
                const int at = __shfl_sync(~0u, next, e), k = __shfl_sync(~0u, cur, e);
                const float ce = MODE == kGrad ? __shfl_sync(~0u, c, e) : 0.f;
                if (lane == at) {
                  const size_t kept = (size_t)(half * 32 + e) * a.K + k;
                  if constexpr (MODE == kStats) a.slog[kept] = __uint_as_float(x[e]);
                  else if (ce != 0.f) put_g(e, ce * a.gval[kept]);
                }
              }
            }
            if (next < left) {
              next = kNone;
              if (SPARSE && ++cur < a.K) {
                next = a.idx[row * a.K + cur];
                if (next != kNone) next -= gv0;
              }
            }
          }
          if constexpr (MODE == kStats) {
            float v[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = lane < left ? __uint_as_float(x[e]) : -INFINITY;
            const float mn = fmaxf(mx, reduce_columns(v, lane, [](float p, float q) { return fmaxf(p, q); }));
            const float mb = scaled(mn, a.a2);
            sum *= mx == -INFINITY ? 0.f : ex2(scaled(mx, a.a2) - mb);
            mx = mn;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float be = __shfl_sync(~0u, mb, e);
              v[e] = lane < left ? ex2(fmaf(__uint_as_float(x[e]), a.a2, -be)) : 0.f;
            }
            sum += reduce_columns(v, lane, [](float p, float q) { return p + q; });
          }
        }
      }
      if (MODE == kStats && live) a.stats[(size_t)(blockIdx.x * 4 + quad) * a.n_rows + row] = make_float2(mx, sum);
    } else {
      // ---------------------------------------------------------- epilogue
      // warps 4-7 take columns 0-127 of the tile, warps 8-11 the rest
      const int quad = warp & 3, half = warp >= 8 ? 1 : 0;
      constexpr int kHalf = kTN / 2;
      const uint32_t lane_base = tbase + ((uint32_t)(quad * 32) << 16) + half * kHalf;
      uint8_t* stage = sO + (quad + 4 * half) * kOutBuf;
      const uint32_t acc_empty0 = leader_addr(&sm->acc_empty[0]), acc_empty1 = leader_addr(&sm->acc_empty[1]);
      const float alpha = (MODE == kDH || MODE == kDW) && a.gout ? upstream() : 1.f;
      int li = 0;                                        // accumulators so far
      // 16 bytes to chunk c of this thread's row of a staging tile (128-byte swizzle)
      auto put = [&](uint8_t* p, int c, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
        *reinterpret_cast<uint4*>(p + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(x, y, z, w);
      };
      for (int t = pair; t < total; t += n_pairs) {
        int m, n, k0, k1, split;
        decode(t, m, n, k0, k1, split);
        const int row0 = m * kTM + rank * 128 + quad * 32, row = row0 + lane, n0 = n * kTN + half * kHalf;
        const int cols = min(kHalf, a.N - n0);           // of this warp's half, may be negative
        const bool live = row < M;
        const int orow = live && a.rows ? a.rows[1 + row] : row;      // row of hidden
        // next target of this row at or behind the half's first column, as a column of the half
        int cur = 0, next = kNone;
        const int g0 = MODE == kGrad ? a.b_off + n0 : n0;
        const size_t kept0 = (size_t)orow * a.K;         // the row's place among the targets' values
        Window<int4, int> win;
        Window<float4, float> val;                       // kGrad, kWhole (for G): the targets' gval, prob
        using yes = std::true_type;
        using no = std::false_type;
        auto advance = [&](auto values) {
          ++cur;
          win.step(a.K, cur, kNone);
          if constexpr (decltype(values)::value) val.step(a.K, cur, 0.f);
          next = win.now.x == kNone ? kNone : win.now.x - g0;
        };
        float c = 0.f, lse2 = 0.f;
        auto first = [&](auto values) {                  // of the targets in this half
          cur = lower_bound(a.idx + kept0, a.K, g0);
          win.open(a.idx + kept0, a.K, cur, kNone);
          if constexpr (decltype(values)::value) val.open((MODE == kGrad ? a.gval : a.prob) + kept0, a.K, cur, 0.f);
          next = win.now.x == kNone ? kNone : win.now.x - g0;
        };
        auto targets = [&]() {
          if (live && cols > 0) {
            if constexpr (SPARSE) {
              first(std::integral_constant<bool, MODE == kGrad>());
              if (MODE == kWhole) c = a.row_scale[orow];
            } else {
              const long long tv = a.target[orow] - g0;
              if (MODE == kWhole) c = tv + g0 == a.ignore ? 0.f : tv + g0 >= 0 && tv + g0 < a.N ? 1.f : __int_as_float(0x7fc00000);
              if (tv >= 0 && tv < kHalf) {
                next = (int)tv;
                if (MODE == kGrad) val.now.x = a.gval[orow];
              }
            }
            if constexpr (MODE == kGrad) {
              const float up = a.gout ? a.cscale * a.gout[orow] : 1.f;
              if (up != 0.f) c = up * a.row_scale[orow];
              lse2 = a.lse2[orow];
            }
          }
        };
        if (MODE == kGrad) targets();
        auto filled = [&]() {                            // the next accumulator, unless a wait gave up
          const bool ok = mbar_wait(&sm->acc_full[li & 1], (li >> 1) & 1, abort);
          if (__any_sync(~0u, !ok)) return false;
          tc_fence_after();
          return true;
        };
        auto release = [&]() {                           // its TMEM has been read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_leader(li & 1 ? acc_empty1 : acc_empty0);
          ++li;
        };
        // 64 columns of G to the staging, in bf16; zeros for a row without a gradient, whatever its logits are
        auto g_rows = [&](bool some, auto g) {
          if (!some) {
#pragma unroll
            for (int ch = 0; ch < 8; ++ch) put(stage, ch, 0, 0, 0, 0);
            return;
          }
          auto two = [&](int e) { const float2 v = g(e); return pack_bf16(v.x, v.y); };
#pragma unroll
          for (int ch = 0; ch < 8; ++ch) put(stage, ch, two(8 * ch), two(8 * ch + 2), two(8 * ch + 4), two(8 * ch + 6));
        };
        auto put_at = [&](int at, float v) {             // one of the 64 columns again
          *reinterpret_cast<__nv_bfloat16*>(stage + lane * 128 + (((at >> 3) ^ (lane & 7)) << 4) + (at & 7) * 2) =
              __float2bfloat16_rn(v);
        };
        auto store = [&](int c0) {                       // the staging to columns n0 + c0 of the result
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            if ((MODE == kDH || MODE == kDW) && a.out == kOutPlaneAdd) tma_reduce_add_3d(&tmO, stage, n0 + c0, row0, split);
            else tma_store_3d(&tmO, stage, n0 + c0, row0, split);
            bulk_commit();
          }
        };
        if constexpr (kParts) {
          float s[kHalf];                                // logits of this row
          bool ok = filled();
          if (ok) {
            uint32_t x[kHalf / 32][32];
#pragma unroll
            for (int c = 0; c < kHalf / 32; ++c) tmem_ld32(lane_base + (li & 1) * kTN + c * 32, x[c]);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < kHalf; ++e) s[e] = __uint_as_float(x[e / 32][e % 32]);
            release();
            targets();                                   // their loads meet the wait for the next part
          }
          for (int k = kPart; ok && k < sched.kb; k += kPart) {
            if (!(ok = filled())) break;
#pragma unroll
            for (int c0 = 0; c0 < kHalf; c0 += 32) {
              uint32_t x[32];
              tmem_ld32(lane_base + (li & 1) * kTN + c0, x);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float2 t = fadd2(make_float2(s[c0 + e], s[c0 + e + 1]),
                                       make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])));
                s[c0 + e] = t.x;
                s[c0 + e + 1] = t.y;
              }
            }
            release();
          }
          if (MODE == kWhole) ok = pair_all(1 + quad, ok);      // the two warps of a row go on together or not at all
          if (!ok) break;
          if (MODE == kWhole) {                          // the last tile's stores have read the staging
            if (lane == 0) bulk_wait_read_all();
            __syncwarp();
          }
          float st = 0.f;                                // the target's logit
#pragma unroll
          for (int c0 = 0; c0 < kHalf; c0 += 32) {
            // logits of the targets among these columns, by way of this thread's row in shared memory
            if (__any_sync(~0u, next < c0 + 32)) {
#pragma unroll
              for (int ch = 0; ch < 8; ++ch) {
                auto u = [&](int e) { return __float_as_uint(s[c0 + 4 * ch + e]); };
                put(stage, ch, u(0), u(1), u(2), u(3));
              }
              while (next < c0 + 32) {
                const int at = next - c0;
                st = *reinterpret_cast<const float*>(stage + lane * 128 + (((at >> 2) ^ (lane & 7)) << 4) + (at & 3) * 4);
                a.slog[kept0 + cur] = st;
                if constexpr (SPARSE) advance(no());
                else next = kNone;
              }
            }
          }
          if (cols < kHalf) {
#pragma unroll
            for (int e = 0; e < kHalf; ++e)
              if (e >= cols) s[e] = -INFINITY;
          }
          // maximum of the half row, then its exponentials, which take the logits' place
          float mp[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < kHalf; e += 2) mp[(e >> 1) & 3] = fmax3(mp[(e >> 1) & 3], s[e], s[e + 1]);
          const float mx = fmaxf(fmaxf(mp[0], mp[1]), fmaxf(mp[2], mp[3])), mb = scaled(mx, a.a2);
          float2 sp[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) sp[u] = make_float2(0.f, 0.f);
#pragma unroll
          for (int e = 0; e < kHalf; e += 2) {
            const float2 arg = ffma2(make_float2(s[e], s[e + 1]), make_float2(a.a2, a.a2), make_float2(-mb, -mb));
            s[e] = ex2(arg.x);
            s[e + 1] = ex2(arg.y);
            sp[(e >> 1) & 3] = fadd2(sp[(e >> 1) & 3], make_float2(s[e], s[e + 1]));
          }
          const float2 r = fadd2(fadd2(sp[0], sp[1]), fadd2(sp[2], sp[3]));
          const float sum = r.x + r.y;
          if (live) a.stats[(size_t)(2 * n + half) * a.n_rows + row] = make_float2(mx, sum);
          if constexpr (MODE == kWhole) {
            // the row's other half, then G / c = (exp(s - lse) - p) row_scale
            __syncwarp();
            reinterpret_cast<float2*>(stage)[lane] = make_float2(mx, sum);
            pair_sync(1 + quad);
            const float2 o = reinterpret_cast<const float2*>(sO + (quad + 4 * (1 - half)) * kOutBuf)[lane];
            pair_sync(1 + quad);
            const float top = fmaxf(mx, o.x), tb = scaled(top, a.a2);
            const float all = (mx == -INFINITY ? sum : sum * ex2(scaled(mx, a.a2) - tb)) +
                              (o.x == -INFINITY ? o.y : o.y * ex2(scaled(o.x, a.a2) - tb));
            lse2 = tb + log2f(all);
            // c / sum of the exponentials; a half of -infinities only has none (NaN where the whole row has none)
            const float f = c * (mx == -INFINITY ? 0.f * lse2 : ex2(mb - lse2));
            if constexpr (SPARSE) {
              if (live && cols > 0) first(yes());
            } else if (live && cols > 0) {
              const long long tv = a.target[orow] - g0;
              next = tv >= 0 && tv < kHalf ? (int)tv : kNone;
            }
#pragma unroll
            for (int c0 = 0; c0 < kHalf; c0 += 64) {
              if (c0 >= cols || row0 >= min(a.n_rows, (M + 63) / 64 * 64)) continue;
              if (lane == 0) bulk_wait_read_all();
              __syncwarp();
              g_rows(c != 0.f, [&](int e) { return fmul2(make_float2(s[c0 + e], s[c0 + e + 1]), make_float2(f, f)); });
              while (c != 0.f && next < c0 + 64) {
                const int at = next;
                float p = 1.f;
                if constexpr (SPARSE) {
                  st = a.slog[kept0 + cur];              // this thread's own
                  p = 0.f;
                  do { p += val.now.x; advance(yes()); } while (next == at);    // the same index adds up
                } else {
                  next = kNone;
                }
                put_at(at - c0, c * (ex2(fmaf(st, a.a2, -lse2)) - p));
              }
              store(c0);
            }
          }
        } else {
          if (!filled()) break;
          const uint32_t acc = lane_base + (li & 1) * kTN;
          const int width = MODE == kGrad || a.out == kOutBf16 ? 64 : 32;      // columns of one store
#pragma unroll 1
          for (int c0 = 0; c0 < kHalf; c0 += width) {
            uint32_t x[32], y[32];
            tmem_ld32(acc + c0, x);
            if (width == 64) tmem_ld32(acc + c0 + 32, y);
            tmem_ld_wait();
            if (c0 + width == kHalf) release();
            // kGrad writes zeros up to the end of the 64 rows that the last step of kDW takes
            if (c0 >= cols || row0 >= (MODE == kGrad ? min(a.n_rows, (M + 63) / 64 * 64) : M)) continue;
            if (MODE == kDW && k0 == k1) {       // no rows at all in this part
#pragma unroll
              for (int e = 0; e < 32; ++e) x[e] = y[e] = 0;
            }
            if constexpr (MODE == kDH || MODE == kDW) {
              if (a.gout) {
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  x[e] = alpha == 0.f ? 0u : __float_as_uint(alpha * __uint_as_float(x[e]));
                  if (width == 64) y[e] = alpha == 0.f ? 0u : __float_as_uint(alpha * __uint_as_float(y[e]));
                }
              }
            }
            uint8_t* p = stage;
            if (lane == 0) bulk_wait_read_all();
            __syncwarp();
            if constexpr (MODE == kGrad) {
              g_rows(c != 0.f, [&](int e) {
                const uint32_t* u = e < 32 ? x + e : y + e - 32;
                const float2 arg = ffma2(make_float2(__uint_as_float(u[0]), __uint_as_float(u[1])), make_float2(a.a2, a.a2),
                                         make_float2(-lse2, -lse2));
                return fmul2(make_float2(ex2(arg.x), ex2(arg.y)), make_float2(c, c));
              });
              while (c != 0.f && next < c0 + 64) {       // the row's targets among these columns (the same one twice: twice alike)
                put_at(next - c0, c * val.now.x);
                if constexpr (SPARSE) advance(yes());
                else next = kNone;
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
            store(c0);
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
  if constexpr (MODE == kDH || MODE == kDW) {
    // NaN in this CTA's rows of its tiles
    if (sm->abort) {
      const float nan = __int_as_float(0x7fc00000);
      for (int t = pair; t < total; t += n_pairs) {
        int m, n, k0, k1, split;
        decode(t, m, n, k0, k1, split);
        for (int i = threadIdx.x; i < 128 * kCols; i += kThreads) {
          const int r = m * kTM + rank * 128 + i / kCols, v = n * kCols + i % kCols;
          if (r >= M || v >= a.N) continue;
          const size_t at = FEW ? (size_t)v * a.M + r : (size_t)r * a.N + v;
          if (a.out == kOutBf16) reinterpret_cast<__nv_bfloat16*>(a.result)[at] = __float2bfloat16_rn(nan);
          else reinterpret_cast<float*>(a.result)[(size_t)split * (MODE == kDW ? a.M : a.n_rows) * (FEW ? a.M : a.N) + at] = nan;
        }
      }
    }
  }
}

// ---------------------------------------------------------------- small kernels
// One warp per row: the K teacher entries sorted by vocabulary index (absent ones, and
// those that fill a row up to Kp, a multiple of four, behind), their probabilities
// softmax(t / T) and sum p log p.  An entry's place is the number of smaller keys, the
// key being its index with its position in the low eight bits (V <= 2^22, K <= 256).
//   row_scale: 1, 0 for a row without entries, NaN for one with an index >= V or
//   a teacher logit that is NaN or +infinity
template <class T>
__global__ void __launch_bounds__(128)
teacher_kernel(const T* tv, const long long* ti, int N, int V, int K, float inv_t,
               int* idx, float* prob, float* ent, float* row_scale) {
  after_previous();
  extern __shared__ int4 sh[];
  const int Kp = (K + 3) & ~3;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* key = reinterpret_cast<int*>(sh) + warp * Kp;
  const int row = blockIdx.x * 4 + warp;
  if (row >= N) return;
  const T* tr = tv + (size_t)row * K;
  const long long* ir = ti + (size_t)row * K;
  idx += (size_t)row * Kp;
  prob += (size_t)row * Kp;
  constexpr int kAbsent = 0x7f000000;              // above every key of an entry
  bool bad = false;
  float mx = -INFINITY;
  for (int k = lane; k < Kp; k += 32) {
    bool here = false;
    long long i = -1;
    if (k < K) {
      i = ir[k];
      here = i >= 0 && i < V;
      const float x = (float)tr[k] * inv_t;
      bad |= i >= V || (here && x != x);
      if (here) mx = fmaxf(mx, x);
    }
    key[k] = here ? (int)i << 8 | k : kAbsent + k;
  }
  __syncwarp();
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
  bad = __any_sync(~0u, bad);
  float z = 0.f;
  for (int k = lane; k < K; k += 32)
    if (key[k] < kAbsent && mx != -INFINITY) z += expf((float)tr[k] * inv_t - mx);
#pragma unroll
  for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(~0u, z, o);
  const bool some = mx != -INFINITY;
  const float logz = logf(z);
  float e = 0.f;
  bool any_nan = false;
  const int4* keys = reinterpret_cast<const int4*>(key);
  for (int k = lane; k < Kp; k += 32) {
    const int me = key[k];
    int r = 0;
    for (int j = 0; j < Kp / 4; ++j) {
      const int4 o = keys[j];
      r += (o.x < me) + (o.y < me) + (o.z < me) + (o.w < me);
    }
    float p = 0.f;
    const bool here = me < kAbsent && some;
    if (here) {
      const float x = (float)tr[k] * inv_t - mx - logz;
      p = expf(x);
      any_nan |= p != p;
      if (p > 0.f) e = fmaf(p, x, e);
    }
    idx[r] = here ? me >> 8 : kNone;
    prob[r] = p;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) e += __shfl_xor_sync(~0u, e, o);
  any_nan = __any_sync(~0u, any_nan);
  if (lane == 0) {
    ent[row] = e;
    row_scale[row] = bad || any_nan ? __int_as_float(0x7fc00000) : some ? 1.f : 0.f;
  }
}

// ---- the rows that count, packed: rows = {their number, row of hidden of each, (n_rows)
// place of each row of hidden or -1 (n_rows)}.  Blocks of 1024 rows.
template <bool SPARSE>
__device__ __forceinline__ bool row_counts(const long long* target, long long ignore, const float* row_scale, int i) {
  return SPARSE ? row_scale[i] != 0.f : target[i] != ignore;
}
// Counts per block; what the losses of the other rows are.
template <bool SPARSE>
__global__ void __launch_bounds__(1024)
mark_kernel(const long long* target, long long ignore, float* row_scale, float* lse2,
            float* loss_rows, int N, int* counts) {
  after_previous();
  const int i = blockIdx.x * 1024 + threadIdx.x;
  const bool yes = i < N && row_counts<SPARSE>(target, ignore, row_scale, i);
  if (i < N && !yes) {
    row_scale[i] = 0.f;
    lse2[i] = 0.f;
    if (loss_rows) loss_rows[i] = 0.f;
  }
  const int n = __syncthreads_count(yes);
  if (threadIdx.x == 0) counts[blockIdx.x] = n;
}
template <bool SPARSE>
__global__ void __launch_bounds__(1024)
index_kernel(const long long* target, long long ignore, const float* row_scale, int N,
             const int* counts, int* rows) {
  after_previous();
  __shared__ int sums[2][32];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  int before = 0, all = 0;
  for (int b = tid; b < (int)gridDim.x; b += 1024) {
    const int c = counts[b];
    all += c;
    if (b < (int)blockIdx.x) before += c;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    before += __shfl_xor_sync(~0u, before, o);
    all += __shfl_xor_sync(~0u, all, o);
  }
  if (lane == 0) { sums[0][w] = before; sums[1][w] = all; }
  __syncthreads();
  before = all = 0;
  for (int k = 0; k < 32; ++k) { before += sums[0][k]; all += sums[1][k]; }
  if (blockIdx.x == 0 && tid == 0) rows[0] = all;
  const int i = blockIdx.x * 1024 + tid;
  const bool yes = i < N && row_counts<SPARSE>(target, ignore, row_scale, i);
  const unsigned mask = __ballot_sync(~0u, yes);
  __syncthreads();
  if (lane == 0) sums[0][w] = __popc(mask);
  __syncthreads();
  int at = before + __popc(mask & ((1u << lane) - 1));
  for (int k = 0; k < w; ++k) at += sums[0][k];
  if (yes) rows[1 + at] = i;
  if (i < N) rows[1 + N + i] = yes ? at : -1;
}
// One warp per packed row; zeros behind the last up to a multiple of 64 rows, the
// depth of kDW's steps.  Nothing to do where every row counts.
__global__ void __launch_bounds__(256)
pack_kernel(const uint4* hidden, const int* rows, int N, int chunks, uint4* out) {
  after_previous();
  const int live = rows[0], lane = threadIdx.x & 31;
  const int j = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (live == N || j >= min(N, (live + 63) / 64 * 64)) return;
  uint4* o = out + (size_t)j * chunks;
  if (j < live) {
    const uint4* h = hidden + (size_t)rows[1 + j] * chunks;
    for (int c = lane; c < chunks; c += 32) o[c] = h[c];
  } else {
    for (int c = lane; c < chunks; c += 32) o[c] = make_uint4(0, 0, 0, 0);
  }
}

// hidden with zeros in the rows that do not count, where one of those is not finite.  With
// two: in any case, and up to kTwo rows, twice.
__global__ void __launch_bounds__(256)
clean_kernel(const uint4* hidden, const float* row_scale, const int* dirty, int N, int chunks, int two, uint4* out) {
  after_previous();
  if (!two && *dirty == 0) return;
  const int lane = threadIdx.x & 31, rows = two ? 2 * kTwo : N;
  for (int j = blockIdx.x * 8 + (threadIdx.x >> 5); j < rows; j += gridDim.x * 8) {
    const int row = two ? j % kTwo : j;
    const bool yes = row < N && row_scale[row] != 0.f;
    const uint4* h = hidden + (size_t)row * chunks;
    uint4* o = out + (size_t)j * chunks;
    for (int c = lane; c < chunks; c += 32) o[c] = yes ? h[c] : make_uint4(0, 0, 0, 0);
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
  const int* rows;                   // as in Args
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
  int D;
  const uint4* scan;                      // hidden: *dirty is 1 if a row that does not count is not finite
  int* dirty;                             // NULL where the rows are packed
};

template <bool SPARSE, int RB>
__global__ void __launch_bounds__(1024)
finish_kernel(const FinishArgs a) {
  after_previous();
  __shared__ float2 sh[1024];
  __shared__ double2 tot[32];
  __shared__ bool last, lost;                      // lost: the statistics are not there, NaN
  const int tid = threadIdx.x, r = tid % RB, slot = tid / RB, N = a.N, K = a.K;
  const int j = blockIdx.x * RB + r;
  const bool live = j < (a.rows ? a.rows[0] : N);
  const int row = a.rows && live ? a.rows[1 + j] : j;
  auto join = [&](float2 u, float2 v) {
    const float mn = fmaxf(u.x, v.x), mb = scaled(mn, a.a2);
    return make_float2(mn, (u.x == -INFINITY ? u.y : u.y * ex2(scaled(u.x, a.a2) - mb)) +
                               (v.x == -INFINITY ? v.y : v.y * ex2(scaled(v.x, a.a2) - mb)));
  };
  float2 st = make_float2(-INFINITY, 0.f);
  if (live) {
#pragma unroll 4
    for (int t = slot; t < a.parts; t += a.slots) st = join(st, a.stats[(size_t)t * N + j]);
  }
  sh[tid] = st;
  if (tid == 0) lost = gave_up();
  __syncthreads();
  for (int o = a.slots >> 1; o; o >>= 1) {
    if (slot < o) sh[tid] = join(sh[tid], sh[tid + o * RB]);
    __syncthreads();
  }
  // lse2 = top + rest; a loss takes its logit off top first, so that what is left of a row with one
  // large logit does not carry lse2's rounding
  const float top = scaled(sh[r].x, a.a2), rest = log2f(sh[r].y), l2 = top + rest;
  float loss = 0.f, scale = 0.f;
  if constexpr (SPARSE) {
    // the entries of a row by the threads of consecutive numbers, which read them together
    __shared__ float2 lse_sh[RB];
    if (slot == 0) lse_sh[r] = make_float2(top, rest);
    __syncthreads();
    const int r2 = tid / a.slots, k0 = tid % a.slots, j2 = blockIdx.x * RB + r2;
    float x = 0.f;
    if (j2 < (a.rows ? a.rows[0] : N)) {
      const size_t row0 = (size_t)(a.rows ? a.rows[1 + j2] : j2) * K;
      const int* idx = a.idx + row0;
      const float2 lr = lse_sh[r2];
      for (int k = k0; k < K; k += a.slots) {
        const int me = idx[k];
        if (me == kNone) break;
        const float p = a.prob[row0 + k], q = fmaf(-a.slog[row0 + k], a.a2, lr.x) + lr.y;   // -log2 of the student's
        if (p > 0.f) x = fmaf(p, q * kLn2, x);
        float same = p;                            // entries with the same index add up
        for (int i = k - 1; i >= 0 && idx[i] == me; --i) same += a.prob[row0 + i];
        for (int i = k + 1; i < K && idx[i] == me; ++i) same += a.prob[row0 + i];
        a.slog[row0 + k] = ex2(-q) - same;
      }
    }
    sh[tid].x = x;                                 // sh was last read before the last __syncthreads
    __syncthreads();
    for (int o = a.slots >> 1; o; o >>= 1) {
      if (k0 < o) sh[tid].x += sh[tid + o].x;
      __syncthreads();
    }
    if (live && slot == 0) {
      scale = a.row_scale[row];
      if (lost && scale != 0.f) a.row_scale[row] = scale = __int_as_float(0x7fc00000);
      if (scale != 0.f) loss = scale * a.t2 * (a.ent[row] + sh[r * a.slots].x);
    }
  } else if (live && slot == 0) {
    const long long t = a.target[row];
    if (t != a.ignore) {
      const bool in = t >= 0 && t < a.V && !lost;
      scale = in ? 1.f : __int_as_float(0x7fc00000);
      const float q = in ? fmaf(-a.slog[row], a.a2, top) + rest : scale;      // -log2 of the target's probability
      loss = q < 0.f ? 0.f : q * kLn2;             // a rounding may leave it below zero
      if (in) a.slog[row] = ex2(-q) - 1.f;
    }
    a.row_scale[row] = scale;
  }
  if (live && slot == 0) {
    a.lse2[row] = l2;
    if (a.reduction == LH_REDUCE_NONE) a.loss[row] = loss;
  }
  if (a.dirty) {                                   // a warp per row; the rows that count are not read
    const int lane = tid & 31, chunks = a.D / 8;
    bool odd = false;
    for (int w = tid >> 5; w < RB; w += blockDim.x >> 5) {
      const int jj = blockIdx.x * RB + w;
      if (jj >= N || (SPARSE ? a.row_scale[jj] != 0.f : a.target[jj] != a.ignore)) continue;
      for (int c = lane; c < chunks; c += 32) {
        const uint4 v = a.scan[(size_t)jj * chunks + c];
        for (uint32_t u : {v.x, v.y, v.z, v.w})
          odd |= (u & 0x7f80u) == 0x7f80u || (u & 0x7f800000u) == 0x7f800000u;
      }
    }
    if (odd) *a.dirty = 1;
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
    const volatile double2* v = a.part + i;
    s += v->x;
    c += v->y;
  }
  block_sum(s, c);
  if (tid == 0) {
    const double inv = a.reduction == LH_REDUCE_MEAN ? (c > 0 ? 1.0 / c : 0.0) : 1.0;
    *a.loss = lost ? __int_as_float(0x7fc00000) : (float)(c > 0 ? s * inv : 0.0);
    *a.inv_count = lost ? __int_as_float(0x7fc00000) : (float)inv;
  }
}

// out (bf16) = sum of the fp32 planes (n_rows x cols each), in their order.  With
// rows: the planes hold packed rows, split_of tells how many planes their number of
// row blocks had, and a row that does not count is 0.
struct PlanesArgs {
  const float* planes;
  int n, n_rows, cols;
  const int* rows;
  uint8_t split_of[kSplitTable];
  __nv_bfloat16* out;
};
__global__ void __launch_bounds__(256)
planes_kernel(const __grid_constant__ PlanesArgs a) {
  after_previous();
  const size_t plane = (size_t)a.n_rows * a.cols;
  const int chunks = a.cols / 8;
  int n = a.n;
  if (a.rows) {
    const int t = (a.rows[0] + kTM - 1) / kTM;
    n = min(n, t < kSplitTable ? (int)a.split_of[t] : 1);
  }
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < plane / 8; i += (size_t)gridDim.x * 256) {
    size_t from = i;                              // 8-element chunk of a plane
    bool live = true;
    if (a.rows) {
      const size_t row = i / chunks;
      const int at = a.rows[1 + a.n_rows + row];
      live = at >= 0;
      from = (size_t)at * chunks + (i - row * chunks);
    }
    float v[8] = {};
    if (live) {
      const float* p = a.planes + from * 8;
#pragma unroll 4
      for (int k = 0; k < n; ++k) {
        float u[8];
        plain16(p + k * plane, u);
        plain16(p + k * plane + 4, u + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += u[e];
      }
    }
    store16(a.out + i * 8, v);
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

// bf16 (rows, cols) with a row pitch in elements; boxes of 64 columns, 128-byte swizzle.
static int map_load(CUtensorMap* m, const void* p, long long rows, long long cols, long long pitch, unsigned box_rows = 64) {
  auto enc = encode_fn();
  if (!enc) { set_error("cuTensorMapEncodeTiled unavailable"); return LH_ERR_LAUNCH; }
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)pitch * 2};
  cuuint32_t box[2] = {64, box_rows}, es[2] = {1, 1};
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

template <int MODE, bool SPARSE, bool FEW = false>
static int launch(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mo, const CUtensorMap& mp, Args& a,
                  long long K, cudaStream_t st) {
  const int tiles_m = (a.M + kTM - 1) / kTM;
  a.tiles_n = FEW ? 1 : (a.N + kTN - 1) / kTN;
  a.kb = (int)((K + kTK - 1) / kTK);
  // Row blocks walked together: as many as keep their operand rows in about half of L2, at least
  // eight (eight by nine tiles are one wave of the 74 pairs).
  long long gm = (48ll << 20) / (kTM * 2ll * a.kb * kTK);
  if (gm < 8) gm = 8;
  a.gm = (int)(gm < tiles_m ? gm : tiles_m);
  Sched& c = a.sched;
  c.M = a.M;
  c.kb = a.kb;
  c.packed = 0;
  c.tiles_m = tiles_m;
  c.gm = a.gm;
  c.splits = a.splits;
  if (MODE == kDH && !FEW) {         // as the kernel has it for packed rows
    const int s = tiles_m < kSplitTable ? a.split_of[tiles_m] : 1;
    if (s < c.splits) c.splits = s > 1 ? s : 1;
  }
  c.total = (int)((long long)tiles_m * a.tiles_n * c.splits);
  const long long total = (long long)tiles_m * a.tiles_n * a.splits;      // at most: packed rows may have more parts
  for (int i = 0; i < 4; ++i) c.div[i] = FastDiv(c.divisor(i, a.tiles_n));
  const int pairs = (int)(total < kPairs ? total : kPairs);
  static std::atomic<uint64_t> allowed{0};           // devices on which the kernel may use its shared memory
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (e == cudaSuccess && (dev >= 64 || !(allowed.load() & bit))) {
    e = cudaFuncSetAttribute(loss_gemm_kernel<MODE, SPARSE, FEW>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(FEW));
    if (e == cudaSuccess && (MODE == kStats || MODE == kWhole) && !FEW) {
      cudaFuncAttributes fa;
      e = cudaFuncGetAttributes(&fa, loss_gemm_kernel<MODE, SPARSE, FEW>);
      if (e == cudaSuccess && fa.numRegs * kThreads < 128 * kRegsRoles + 256 * kRegsEpilogue) {
        set_error("linear loss: the kernel was compiled to %d registers, too few to share out", fa.numRegs);
        return LH_ERR_LAUNCH;
      }
    }
    if (e == cudaSuccess && dev < 64) allowed.fetch_or(bit);
  }
  if (e != cudaSuccess) { set_error("linear loss: %s", cudaGetErrorString(e)); return LH_ERR_LAUNCH; }
  return launch_behind("loss_gemm_kernel", loss_gemm_kernel<MODE, SPARSE, FEW>, 2 * pairs, kThreads, smem_bytes(FEW), st,
                       ma, mb, mo, mp, a);
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

static size_t up(size_t n) { return (n + 255) & ~size_t(255); }

// Whether the rows that count are packed: where the products are long against the
// three small kernels that do it (about 8 us; a product of 5e10 takes 40 us or more)
// and more than one row block is there to be saved.
static bool packs(long long N, long long V, long long D) { return N > kTM && 2.0 * N * V * D >= 5e10; }

struct Plan {
  long long C;                 // columns of a vocabulary piece, a multiple of 256
  int pieces, dh_splits, dw_splits;
  uint8_t split_of[kSplitTable];
  bool dh_planes, pack, two;
  size_t g, dh, dw, packed, total;     // bytes
};
constexpr long long kPieceBytes = 512ll << 20;

static Plan make_plan(long long N, long long V, long long D) {
  Plan p{};
  long long C = kPieceBytes / (2 * N) / kTN * kTN;
  if (C < kTN) C = kTN;
  const long long Vp = (V + kTN - 1) / kTN * kTN;
  p.pieces = (int)((Vp + C - 1) / C);
  p.C = ((Vp + p.pieces - 1) / p.pieces + kTN - 1) / kTN * kTN;      // pieces of about equal size
  p.pieces = (int)((Vp + p.C - 1) / p.C);
  const long long cols = p.C < V ? p.C : V, tiles = (N + kTM - 1) / kTM;
  const bool pack = p.pack = packs(N, V, D);
  // dH: the parts by the number of row blocks that are left; at most twice those of all rows
  p.dh_splits = tiles < kSplitTable ? pick_splits(N, D, cols) : 1;
  const int most = pack ? 2 * p.dh_splits : p.dh_splits;
  for (int t = 1; t < kSplitTable; ++t) {
    int s = t == tiles ? p.dh_splits : t < tiles && pack ? pick_splits((long long)t * kTM, D, cols) : 1;
    p.split_of[t] = (uint8_t)(s < most ? s : most);
  }
  for (int t = 1; t < kSplitTable && t <= tiles; ++t)
    if (p.split_of[t] > p.dh_splits) p.dh_splits = p.split_of[t];
  p.dw_splits = pick_splits(cols, D, N);
  p.dh_planes = pack || p.pieces > 1 || p.dh_splits > 1;
  p.two = N <= kTwo;
  const long long rows = p.two ? 2 * kTwo : N;
  p.g = up((size_t)rows * p.C * 2);
  p.dh = p.dh_planes ? up((size_t)p.dh_splits * N * D * 4) : 0;
  p.dw = p.dw_splits > 1 ? up((size_t)p.dw_splits * p.C * D * 4) : 0;
  p.packed = up((size_t)rows * D * 2);    // the packed rows, or clean_kernel's
  p.total = p.g + p.dh + p.dw + p.packed;
  return p;
}

// The search over splits takes a few microseconds, a call's check and its launches each want the
// plan: every thread keeps those of the last sizes.
static const Plan& plan(long long N, long long V, long long D) {
  struct Entry { long long N, V, D; Plan p; };
  static thread_local Entry seen[8] = {};
  static thread_local int at = 0;
  for (const Entry& e : seen)
    if (e.N == N && e.V == V && e.D == D) return e.p;
  Entry& e = seen[at];
  at = (at + 1) % 8;
  e = {N, V, D, make_plan(N, V, D)};
  return e.p;
}

// Places of a row's K entries: a multiple of four, for the loads of four.
static long long entries(long long K) { return (K + 3) & ~3ll; }

// Whether the forward may leave G / c: the rows are whole in one tile, and c is one number
// (65536 x 256 x 1024, forward and backward: 161 us, 190 where the backward forms the logits
// again; 16384 rows with 16 targets each: 90 us against 95).
static bool whole(long long N, long long V, int reduction) { return N > kFew && V <= kTN && reduction != LH_REDUCE_NONE; }

// What the forward leaves for the backward.
struct Kept {
  float *lse2, *row_scale, *inv_count, *tgrad;   // (N), (N), (1), (N, max(K, 1))
  int *idx, *rows, *dirty;                       // (N, K) sorted targets, (2 N + 1) packed rows, (1)
  void* g;                                       // NULL or G / c (N, kTN) bf16
  size_t bytes;
  Kept(void* base, long long N, long long V, long long K, int reduction, bool gradients) {
    char* p = (char*)base;
    auto take = [&](size_t n) { char* q = p; p += up(n); return q; };
    lse2 = (float*)take(4 * N);
    row_scale = (float*)take(4 * N);
    inv_count = (float*)take(4);
    tgrad = (float*)take(4 * N * (K ? entries(K) : 1));
    idx = (int*)take(4 * N * entries(K));
    rows = (int*)take(4 * (2 * N + 1));
    dirty = (int*)take(4);
    g = gradients && whole(N, V, reduction) ? take(N * kTN * 2) : nullptr;
    bytes = p - (char*)base;
  }
};

// With few rows, parts of a row: one per TMEM row block of every CTA that kStats has.
static int few_parts(long long V) {
  const long long tiles = (V + kTM - 1) / kTM;
  return 8 * (int)(tiles < kPairs ? tiles : kPairs);
}

// Workspace of the forward.
struct FwdSpace {
  float2* stats;
  double2* part;
  unsigned* ticket;
  int* counts;
  float *ent, *prob;           // distillation
  void* packed;
  size_t bytes;
  FwdSpace(void* base, long long N, long long V, long long D, long long K) {
    char* p = (char*)base;
    auto take = [&](size_t n) { char* q = p; p += up(n); return q; };
    stats = (float2*)take((size_t)(N <= kFew ? few_parts(V) : (V + kTN - 1) / kTN * 2) * N * sizeof(float2));
    part = (double2*)take((size_t)((N + 7) / 8) * sizeof(double2));
    ticket = (unsigned*)take(4);
    counts = (int*)take(4 * ((N + 1023) / 1024));
    ent = (float*)take(K ? 4 * N : 0);
    prob = (float*)take(4 * N * entries(K));
    packed = take(packs(N, V, D) ? (size_t)N * D * 2 : 0);
    bytes = p - (char*)base;
  }
};

// log2(e) / T: logits to exponents of 2.
static float exponent_scale(float T) { return (float)(1.4426950408889634 / T); }

static int sum_planes(const float* planes, const Plan* p, int n, int rows, int cols, const int* packed, void* out,
                      cudaStream_t st) {
  PlanesArgs a{planes, n, rows, cols, packed, {}, (__nv_bfloat16*)out};
  if (p)
    for (int t = 0; t < kSplitTable; ++t) a.split_of[t] = p->split_of[t];
  const size_t blocks = ((size_t)rows * (cols / 8) + 255) / 256;
  return launch_behind("planes_kernel", planes_kernel, (unsigned)(blocks < 148 * 16 ? blocks : 148 * 16), 256, 0, st, a);
}

static int pack_rows(const void* hidden, const int* rows, int N, int D, void* out, cudaStream_t st) {
  return launch_behind("pack_kernel", pack_kernel, (N + 7) / 8, 256, 0, st, (const uint4*)hidden, rows, N, D / 8, (uint4*)out);
}

struct Problem {
  const void *hidden, *weight;
  int N, V, D;
  const long long* target;     // cross entropy
  long long ignore;
  int K;                       // distillation: entries of a row, 0 else
  float T;
};

template <bool SPARSE>
static int forward(const Problem& q, int reduction, float* loss, const Kept& kp, const FwdSpace& ws, cudaStream_t st) {
  int rc = make_context_current();
  if (rc) return rc;
  const int N = q.N, V = q.V, D = q.D, K = q.K ? (int)entries(q.K) : 1;
  CUtensorMap mh, mw, mp, mg;
  if ((rc = map_load(&mh, q.hidden, N, D, D)) || (rc = map_load(&mw, q.weight, V, D, D))) return rc;
  mp = mh;
  const int* rows = nullptr;
  if (packs(N, V, D)) {
    const int blocks = (N + 1023) / 1024;
    if ((rc = launch_behind("mark_kernel", mark_kernel<SPARSE>, blocks, 1024, 0, st, q.target, q.ignore, kp.row_scale, kp.lse2,
                            reduction == LH_REDUCE_NONE ? loss : nullptr, N, ws.counts)) ||
        (rc = launch_behind("index_kernel", index_kernel<SPARSE>, blocks, 1024, 0, st, q.target, q.ignore, kp.row_scale, N,
                            ws.counts, kp.rows)) ||
        (rc = pack_rows(q.hidden, kp.rows, N, D, ws.packed, st)) ||
        (rc = map_load(&mp, ws.packed, N, D, D)))
      return rc;
    rows = kp.rows;
  }
  const bool few = N <= kFew;
  const int parts = few ? few_parts(V) : (V + kTN - 1) / kTN * 2;
  Args a{};
  a.n_rows = N;
  a.M = few ? V : N;
  a.N = few ? N : V;
  a.splits = 1;
  a.rows = rows;
  a.target = q.target;
  a.idx = kp.idx;
  a.K = K;
  a.a2 = exponent_scale(q.T);
  a.stats = ws.stats;
  a.slog = kp.tgrad;
  a.ticket = ws.ticket;
  a.dirty = kp.dirty;
  if (few) {
    if ((rc = map_load(&mh, q.hidden, N, D, D, kFew / 2)) || (rc = launch<kStats, SPARSE, true>(mw, mh, mw, mw, a, D, st)))
      return rc;
  } else if (kp.g) {
    a.prob = ws.prob;
    a.ignore = q.ignore;
    a.row_scale = kp.row_scale;
    if ((rc = map_store(&mg, kp.g, false, 1, N, V, kTN)) || (rc = launch<kWhole, SPARSE>(mh, mw, mg, mp, a, D, st))) return rc;
  } else if ((rc = launch<kStats, SPARSE>(mh, mw, mw, mp, a, D, st))) {
    return rc;
  }
  // Rows per block: eight with 32 to 128 slots each where a row has many parts or entries, four
  // per slot (16 rows of 1000 parts: 7 us, 17 with 32 rows per block), 256 where it has up to four (65536 rows of two parts:
  // 14 us with 32 rows per block, most of it the 2048 blocks' sum).
  const int want = parts > K ? parts : K;
  FinishArgs f{ws.stats, rows, parts, N, V, K, 1, reduction, q.target, q.ignore, kp.idx, ws.prob, ws.ent, kp.tgrad, a.a2,
               q.T * q.T, kp.row_scale, kp.lse2, loss, kp.inv_count, ws.part, ws.ticket, D,
               (const uint4*)q.hidden, rows ? nullptr : kp.dirty};
  const int rb = want > 32 ? 8 : want > 4 ? 32 : 256;
  while (f.slots < (rb == 8 ? (want + 3) / 4 : want) && f.slots * rb < 1024) f.slots *= 2;
  if (rb == 8 && f.slots < 32) f.slots = 32;
  const unsigned blocks = (unsigned)((N + rb - 1) / rb);
  return launch_behind("finish_kernel", rb == 8 ? finish_kernel<SPARSE, 8> : rb == 256 ? finish_kernel<SPARSE, 256>
                                                                                   : finish_kernel<SPARSE, 32>,
                       blocks, rb * f.slots, 0, st, f);
}

template <bool SPARSE>
static int backward(const Problem& q, int reduction, const Kept& kp, const float* gout, void* dhidden, void* dweight,
                    void* ws, cudaStream_t st) {
  int rc = make_context_current();
  if (rc) return rc;
  const int N = q.N, V = q.V, D = q.D;
  const Plan& p = plan(N, V, D);
  char* g = kp.g ? (char*)kp.g : (char*)ws;
  float* dh = (float*)((char*)ws + p.g);
  float* dw = (float*)((char*)ws + p.g + p.dh);
  char* packed = (char*)ws + p.g + p.dh + p.dw;
  CUtensorMap mh, mw, mp, mdh, mdw, mg, mgo;
  if ((rc = map_load(&mh, q.hidden, N, D, D)) || (rc = map_load(&mw, q.weight, V, D, D))) return rc;
  if ((rc = p.dh_planes ? map_store(&mdh, dh, true, p.dh_splits, N, D, D)
           : dhidden   ? map_store(&mdh, dhidden, false, 1, N, D, D) : LH_OK))
    return rc;
  mp = mh;
  // few rows: always one piece (kFew rows of 2^22 columns take 512 MB)
  const bool few = N <= kFew;
  const int g_rows = p.two ? 2 * kTwo : N;
  CUtensorMap mh_few, mg_few;
  if (few && ((rc = map_load(&mh_few, q.hidden, N, D, D, kFew / 2)) || (rc = map_load(&mg_few, g, g_rows, V, p.C, kFew / 2))))
    return rc;
  const int* rows = nullptr;
  if (p.pack) {                      // kGrad's operand too
    rows = kp.rows;
    rc = pack_rows(q.hidden, rows, N, D, packed, st);
  } else if (dweight) {
    const unsigned blocks = (unsigned)((g_rows + 7) / 8);
    rc = launch_behind("clean_kernel", clean_kernel, blocks < 148 * 8 ? blocks : 148 * 8, 256, 0, st, (const uint4*)q.hidden,
                       kp.row_scale, kp.dirty, N, D / 8, (int)p.two, (uint4*)packed);
  }
  if (rc || (rc = map_load(&mp, packed, g_rows, D, D))) return rc;
  for (int i = 0; i < p.pieces; ++i) {
    const long long v0 = i * p.C;
    const int cols = (int)(V - v0 < p.C ? V - v0 : p.C);
    if ((rc = map_load(&mg, g, g_rows, cols, p.C)) || (!kp.g && (rc = map_store(&mgo, g, false, 1, N, cols, p.C)))) return rc;
    Args a{};
    a.n_rows = N;
    a.M = few ? cols : N;
    a.N = few ? N : cols;
    a.splits = 1;
    a.result = g;
    a.few_pitch = p.C;
    a.two = p.two;
    a.rows = rows;
    a.b_off = (int)v0;
    a.target = q.target;
    a.idx = kp.idx;
    a.K = q.K ? (int)entries(q.K) : 1;
    a.a2 = exponent_scale(q.T);
    a.gval = kp.tgrad;
    a.lse2 = kp.lse2;
    a.row_scale = kp.row_scale;
    a.gout = reduction == LH_REDUCE_NONE ? gout : nullptr;
    a.cscale = q.T;
    if (!kp.g && (rc = few ? launch<kGrad, SPARSE, true>(mw, mh_few, mw, mw, a, D, st)
                           : launch<kGrad, SPARSE>(mh, mw, mgo, mp, a, D, st)))
      return rc;
    auto scaled = [&](Args& z) {     // what comes of G / c
      if (reduction == LH_REDUCE_NONE) return;
      z.gout = gout;
      z.inv_count = kp.inv_count;
      z.cscale = q.T;
    };

    if (dhidden) {
      Args x{};
      x.n_rows = N;
      x.M = few ? D : N;
      x.N = few ? N : D;
      x.result = p.dh_planes ? (void*)dh : dhidden;
      const int kb = (cols + kTK - 1) / kTK;
      x.splits = p.dh_splits < kb ? p.dh_splits : kb;      // a short last piece may leave planes as they are
      for (int t = 0; t < kSplitTable; ++t) x.split_of[t] = p.split_of[t];
      scaled(x);
      x.two = p.two;
      x.rows = rows;
      x.b_off = (int)v0;
      x.out = !p.dh_planes ? kOutBf16 : i ? kOutPlaneAdd : kOutPlane;
      if ((rc = few ? launch<kDH, false, true>(mw, mg_few, mw, mw, x, cols, st)
                    : launch<kDH, false>(mg, mw, mdh, mg, x, cols, st)))
        return rc;
    }
    if (!dweight) continue;

    Args y{};
    y.M = cols;
    y.n_rows = N;
    y.N = D;
    y.splits = p.dw_splits;
    scaled(y);
    y.two = p.two;
    y.rows = rows;
    y.dirty = rows ? nullptr : kp.dirty;
    y.out = p.dw_splits > 1 ? kOutPlane : kOutBf16;
    char* dw_out = (char*)dweight + (size_t)v0 * D * 2;
    y.result = p.dw_splits > 1 ? (void*)dw : dw_out;
    if ((rc = p.dw_splits > 1 ? map_store(&mdw, dw, true, p.dw_splits, cols, D, D)
                              : map_store(&mdw, dw_out, false, 1, cols, D, D)))
      return rc;
    if ((rc = launch<kDW, false>(mg, mh, mdw, mp, y, g_rows, st))) return rc;
    if (p.dw_splits > 1 && (rc = sum_planes(dw, nullptr, p.dw_splits, cols, D, nullptr, dw_out, st))) return rc;
  }
  return dhidden && p.dh_planes ? sum_planes(dh, &p, p.dh_splits, N, D, rows, dhidden, st) : LH_OK;
}

}  // namespace ll

size_t linear_loss_workspace_size(int N, int V, int D, int K, int backward) {
  return backward ? ll::plan(N, V, D).total : ll::FwdSpace(nullptr, N, V, D, K).bytes;
}

size_t linear_loss_kept_size(int N, int V, int K, int reduction, int gradients) {
  return ll::Kept(nullptr, N, V, K, reduction, gradients).bytes;
}

int linear_xent_fwd(const void* hidden, const void* weight, const long long* target, long long ignore, int N, int V, int D,
                    int reduction, float* loss, void* kept, bool gradients, void* ws, cudaStream_t st) {
  return ll::forward<false>({hidden, weight, N, V, D, target, ignore, 0, 1.f}, reduction, loss,
                            ll::Kept(kept, N, V, 0, reduction, gradients), ll::FwdSpace(ws, N, V, D, 0), st);
}

int linear_xent_bwd(const void* hidden, const void* weight, const long long* target, int N, int V, int D, int reduction,
                    const void* kept, bool gradients, const float* gout, void* dhidden, void* dweight, void* ws,
                    cudaStream_t st) {
  return ll::backward<false>({hidden, weight, N, V, D, target, 0, 0, 1.f}, reduction,
                             ll::Kept(const_cast<void*>(kept), N, V, 0, reduction, gradients), gout, dhidden, dweight, ws, st);
}

int linear_distill_fwd(const void* hidden, const void* weight, const void* tv, int tv_dtype, const long long* ti, int N,
                       int V, int D, int K, float T, int reduction, float* loss, void* kept, bool gradients, void* ws,
                       cudaStream_t st) {
  const ll::Kept kp(kept, N, V, K, reduction, gradients);
  const ll::FwdSpace sp(ws, N, V, D, K);
  const unsigned blocks = (unsigned)((N + 3) / 4);
  const size_t smem = 4 * ll::entries(K) * sizeof(int);
  int rc = tv_dtype == LH_DTYPE_BF16
               ? launch_behind("teacher_kernel", ll::teacher_kernel<__nv_bfloat16>, blocks, 128, smem, st,
                                   (const __nv_bfloat16*)tv, ti, N, V, K, 1.f / T, kp.idx, sp.prob, sp.ent, kp.row_scale)
               : launch_behind("teacher_kernel", ll::teacher_kernel<float>, blocks, 128, smem, st, (const float*)tv, ti, N, V,
                                   K, 1.f / T, kp.idx, sp.prob, sp.ent, kp.row_scale);
  if (rc) return rc;
  return ll::forward<true>({hidden, weight, N, V, D, nullptr, 0, K, T}, reduction, loss, kp, sp, st);
}

int linear_distill_bwd(const void* hidden, const void* weight, int N, int V, int D, int K, float T, int reduction,
                       const void* kept, bool gradients, const float* gout, void* dhidden, void* dweight, void* ws,
                    cudaStream_t st) {
  return ll::backward<true>({hidden, weight, N, V, D, nullptr, 0, K, T}, reduction,
                            ll::Kept(const_cast<void*>(kept), N, V, K, reduction, gradients), gout, dhidden, dweight, ws, st);
}

int loss_status(int reset) {
  int h = 0;
  cudaMemcpyFromSymbol(&h, g_loss_status, sizeof(int));
  if (reset) { const int z = reset < 0; cudaMemcpyToSymbol(g_loss_status, &z, sizeof(int)); }
  return h;
}

}  // namespace lh
