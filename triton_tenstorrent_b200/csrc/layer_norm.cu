// Layer norm over the last dimension, forward and backward, with the reduction of the weight's gradient.
//
//   mu = mean(x), rstd = 1 / sqrt(mean((x - mu)^2) + eps), h = (x - mu) rstd, y = h w + b
//   u = dy w,  dx = rstd (u - mean(u) - h mean(u h)),  dw = sum over rows of dy h,  db = sum over rows of dy
//
// Everything between a load and a store is fp32; each output is rounded once.  The variance is summed over centred values
// (never as E[x^2] - mu^2, which cancels when |mu| is large against the spread).
// Bound: HBM.  Forward: x read, y written; backward: x and dy read, dx written; w, b and the row statistics are small.
#include <initializer_list>
#include <type_traits>

#include "dtypes.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace b200k {

// Sum over the threads of a CTA; every thread gets the result.  `scratch` holds 32 floats and may be reused after the
// next __syncthreads.  The order of the additions depends on the thread count only.
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* scratch) {
  v = warp_sum(v);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  const int warps = blockDim.x >> 5;
  v = warp_sum(lane < warps ? scratch[lane] : 0.f);
  __syncthreads();
  return v;
}

// ---------------------------------------------------------------------------------------------
// Any row length: one CTA per row, the row walked once per pass (the later passes hit L1 / L2).
// ---------------------------------------------------------------------------------------------
// N sums over i = first, first + step, ... below end, to each of which f(i, part) adds a term.  32 terms at a time in fp32, these in fp64, so that a thread's
// share of a row of 2^31 elements or of 2^30 rows is off by 32 roundings and no more.  (bf16, forward / backward: 4096 x 20000 191 / 457 us, 64 x 2^20
// 1050 / 1555 us; term by term in fp32 221 / 529 and 1270 / 1997 us, and equal terms 330 roundings off in 2000.)
template <int N, typename F>
__device__ __forceinline__ void long_sums(int64_t first, int64_t end, int64_t step, float (&sum)[N], F&& f) {
  double total[N] = {};
  int64_t at = first;
  for (; at + 31 * step < end; at += 32 * step) {
    float part[N] = {};
#pragma unroll                                              // loads of many terms on their way at a time
    for (int j = 0; j < 32; ++j) f(at + j * step, part);
#pragma unroll
    for (int k = 0; k < N; ++k) total[k] += static_cast<double>(part[k]);
  }
#pragma unroll
  for (int k = 0; k < N; ++k) sum[k] = 0.f;
#pragma unroll 4
  for (; at < end; at += step) f(at, sum);
#pragma unroll
  for (int k = 0; k < N; ++k) sum[k] = static_cast<float>(total[k] + static_cast<double>(sum[k]));
}

template <typename T, typename W>
__global__ void __launch_bounds__(512) ln_fwd_loop_kernel(const T* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b,
                                                          T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd,
                                                          int64_t rows, int64_t cols, int64_t ldx, int64_t ldy, float eps) {
  __shared__ float scratch[32];
  const float inv_n = 1.f / static_cast<float>(cols);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * ldx;
    float s[1];
    long_sums(threadIdx.x, cols, blockDim.x, s, [&](int64_t c, float (&t)[1]) { t[0] += to_f32<T>(xr[c]); });
    const float mu = block_sum(s[0], scratch) * inv_n;
    long_sums(threadIdx.x, cols, blockDim.x, s, [&](int64_t c, float (&t)[1]) {
      const float d = to_f32<T>(xr[c]) - mu;
      t[0] += d * d;
    });
    const float rs = rsqrtf(block_sum(s[0], scratch) * inv_n + eps);
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      float v = (to_f32<T>(xr[c]) - mu) * rs;
      if (w != nullptr) v *= to_f32<W>(w[c]);
      if (b != nullptr) v += to_f32<W>(b[c]);
      y[r * ldy + c] = from_f32<T>(v);
    }
    if (threadIdx.x == 0) {
      if (mean != nullptr) mean[r] = mu;
      if (rstd != nullptr) rstd[r] = rs;
    }
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(512) ln_dx_loop_kernel(const T* __restrict__ dy, const T* __restrict__ x, const W* __restrict__ w,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ dx,
                                                         int64_t rows, int64_t cols, int64_t lddy, int64_t ldx, int64_t lddx) {
  __shared__ float scratch[32];
  const float inv_n = 1.f / static_cast<float>(cols);
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * ldx;
    const T* gr = dy + r * lddy;
    const float mu = mean[r], rs = rstd[r];
    auto u_at = [&](int64_t c) { return to_f32<T>(gr[c]) * (w != nullptr ? to_f32<W>(w[c]) : 1.f); };
    float s[2];
    long_sums(threadIdx.x, cols, blockDim.x, s, [&](int64_t c, float (&t)[2]) {
      const float u = u_at(c);
      t[0] += u;
      t[1] += u * ((to_f32<T>(xr[c]) - mu) * rs);
    });
    const float c1 = block_sum(s[0], scratch) * inv_n;
    const float c2 = block_sum(s[1], scratch) * inv_n;
    for (int64_t c = threadIdx.x; c < cols; c += blockDim.x) {
      const float u = u_at(c);
      const float h = (to_f32<T>(xr[c]) - mu) * rs;
      dx[r * lddx + c] = from_f32<T>(rs * (u - c1 - h * c2));
    }
  }
}

// Partial sums of dw and db: CTA (i, j) adds the rows of slice j of the columns of tile i, one column per thread.
// part[2][parts][cols]: first dw, then db.
template <typename T>
__global__ void __launch_bounds__(256) ln_dw_loop_kernel(const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ mean,
                                                         const float* __restrict__ rstd, float* __restrict__ part, int64_t rows,
                                                         int64_t cols, int64_t lddy, int64_t ldx) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= cols) return;
  const int parts = gridDim.y;
  float s[2];
  auto term = [&](int64_t r, float (&t)[2]) {
    const float g = to_f32<T>(dy[r * lddy + c]);
    t[0] += g * ((to_f32<T>(x[r * ldx + c]) - mean[r]) * rstd[r]);
    t[1] += g;
  };
  if (rows <= static_cast<int64_t>(parts) * 32) {
    s[0] = s[1] = 0.f;
    for (int64_t r = blockIdx.y; r < rows; r += parts) term(r, s);
  } else {
    long_sums(blockIdx.y, rows, parts, s, term);
  }
  part[static_cast<int64_t>(blockIdx.y) * cols + c] = s[0];
  part[static_cast<int64_t>(parts + blockIdx.y) * cols + c] = s[1];
}

// ---------------------------------------------------------------------------------------------
// Rows of up to TPR * PER * VEC elements, TPR threads to a row: a whole CTA, or (TPR = 32) a warp, LN_GROUPS of them in a CTA.  The rows to come are on
// their way into a ring in shared memory meanwhile.
//
// A row is worked on in steps that wait for one another (load, row sum, second sum, store), and registers for enough rows at a time do not exist
// next to the backward's 2 N running sums; the ring keeps up to 60 KB (backward: 140; two stages at least) per SM on their way instead, whatever the arithmetic
// waits for.
// Rows come as untiled bulk copies of the 16-byte blocks that they touch, so that any length and alignment arrives at full rate; only the
// reads from shared memory and the stores go by VEC, the widest access that the operands' alignment allows.
// A CTA-wide row is fetched by the CTA's first thread, behind a barrier that the row sum needs anyway; a warp of its own for it, as the CTAs of
// narrow rows have, would cost the others registers (17 warps leave them 96 each, 16 warps 128: backward, 16384 x 4096 bf16, 82 against 64 us).
//
// Measured back to back (the backward with its join), inputs larger than L2, of 6460 GB/s: 16384 x 4096 bf16 forward 47 us (5.7 TB/s), backward 70 us
// (5.8 TB/s); 65536 x 4096 168 and 246 us (6.4, 6.5 TB/s); 8192 x 8192 bf16 with fp32 weights 48 and 75 us.  Rows on odd boundaries (16384 x 4095
// bf16: 79 and 87 us) are bound by their 2-byte stores and the LSU.
// ---------------------------------------------------------------------------------------------
constexpr int LN_GROUPS = 8;          // rows at a time of a CTA whose warps take a row each
constexpr int LN_MAX_STAGES = 8;
template <int TPR>
__host__ __device__ constexpr int ln_groups() { return TPR == 32 ? LN_GROUPS : 1; }
template <int TPR>
__host__ __device__ constexpr int ln_threads() { return TPR * ln_groups<TPR>() + (TPR == 32 ? 32 : 0); }      // with the fetching warp
// CTAs of one SM; E: elements a thread, SIZE: bytes of one.  The backward writes a partial sum per CTA, so that it takes fewer
// (65536 x 1024 bf16: 91 us with 4, 77 with 6, 75 with 8; fp32: 124, 136, 139).
template <int TPR, int E, bool BWD, int SIZE>
__host__ __device__ constexpr int ln_per_sm() {
  return TPR == 32 ? (BWD && E > 8 ? 2 : 3) : TPR == 128 ? (BWD ? (E <= 8 && SIZE == 2 ? 6 : 4) : E > 8 ? 5 : SIZE == 2 ? 8 : 6) : TPR == 256 ? (BWD ? 2 : 3) : 1;
}
// Rows that the forward works on at a time.  A second one fills the waits of the first, and halves the barriers: where one CTA has the SM (8192 x 8192), where
// a warp mostly waits (rows of up to 256; 512 to 1024 16-bit elements: 65536 x 1024 65 us one at a time on 6 CTAs, 58 on 8, 50 two at a time), and
// where w and b are read again for every row (4096 x 16384 bf16: 64 against 57 us).  fp32 rows and weights gain nothing there (65536 x 1024 fp32 92 against
// 94, 4096 x 16384 bf16 with fp32 weights 77 against 80).
template <int TPR, int E, int SIZE, int WSIZE>
__host__ __device__ constexpr int ln_batch() {
  return TPR == 512 ? (E <= 16 || SIZE + WSIZE == 4 ? 2 : 1) : TPR == 128 ? (E <= 8 && SIZE == 2 ? 2 : 1) : TPR == 32 && E <= 8 ? 2 : 1;
}

// Whether access k of a thread can lie behind the row's end.  A CTA-wide row fills more than half of its shape (ln_shape), so the first half of the
// accesses cannot.
template <int TPR, int PER>
__device__ __forceinline__ bool ln_inside(int k, int c, int cols) { return (TPR > 32 && k < PER / 2) || c < cols; }

struct LnRing {
  int stage_rows, stages, row_bytes;   // rows of a stage; row_bytes: a row's place in it, a multiple of 16
  int weight_bytes;                    // before the ring: a copy of w, where a thread's part does not fit its registers
};

// One operand's rows, and where its memory ends (nothing outside [base, end) is read).
struct LnSource {
  const char* base;
  int64_t pitch;        // bytes
  const char* end;
};
// Where in its 16-byte block row r begins.
__device__ __forceinline__ uint32_t ln_offset(const LnSource& s, int r) {
  return (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(s.base)) + static_cast<uint32_t>(r) * static_cast<uint32_t>(s.pitch)) & 15u;
}
// The 16-byte blocks of the row at `a` that lie inside the operand: [*from, *from + bytes).
__device__ __forceinline__ uint32_t ln_span(const LnSource& s, const char* a, int row_len, const char** from) {
  uintptr_t lo = reinterpret_cast<uintptr_t>(a) & ~uintptr_t(15);
  uintptr_t hi = (reinterpret_cast<uintptr_t>(a) + row_len + 15) & ~uintptr_t(15);
  if (lo < reinterpret_cast<uintptr_t>(s.base)) lo += 16;
  if (hi > reinterpret_cast<uintptr_t>(s.end)) hi -= 16;
  *from = reinterpret_cast<const char*>(lo);
  return hi > lo ? static_cast<uint32_t>(hi - lo) : 0u;
}
// What ln_span left out (less than 16 bytes at the operand's first and last row), element by element.
template <typename T>
__device__ __noinline__ void ln_patch(const char* a, int row_len, const char* from, uint32_t bytes, char* dst) {
  const char* z = a + row_len;
  const char* head = bytes == 0 || from < a ? a : from;                       // [a, head) and [tail, z) are missing
  const char* tail = bytes == 0 || from + bytes < a ? a : from + bytes;
  for (const char* q = a; q < head; q += sizeof(T)) *reinterpret_cast<T*>(dst + (q - a)) = *reinterpret_cast<const T*>(q);
  for (const char* q = tail; q < z; q += sizeof(T)) *reinterpret_cast<T*>(dst + (q - a)) = *reinterpret_cast<const T*>(q);
}

// One thread fetches `count` rows (one or two, from r on) of each operand into a stage.  ALIGNED: rows are whole 16-byte blocks.
template <typename T, bool ALIGNED, int NSRC>
__device__ __forceinline__ void ln_fetch_rows(const LnSource (&src)[NSRC], const LnRing& ring, int row_len, int r, int count, char* stage, uint64_t* bar) {
  if constexpr (ALIGNED) {
    mbar_expect_tx(bar, static_cast<uint32_t>(NSRC * count * row_len));
    for (int i = 0; i < count; ++i)
#pragma unroll
      for (int k = 0; k < NSRC; ++k) bulk_load(stage + (i * NSRC + k) * row_len, src[k].base + (r + i) * src[k].pitch, row_len, bar);
  } else {
    uint32_t bytes[2][NSRC], total = 0;
    const char* from[2][NSRC];
    char* dst[2][NSRC];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < NSRC; ++k) {
        bytes[i][k] = 0;
        if (i < count) {
          const char* a = src[k].base + (r + i) * src[k].pitch;
          bytes[i][k] = ln_span(src[k], a, row_len, &from[i][k]);
          char* row = stage + (i * NSRC + k) * ring.row_bytes + (reinterpret_cast<uintptr_t>(a) & 15u);
          dst[i][k] = row + (from[i][k] - a);
          if (from[i][k] > a || from[i][k] + bytes[i][k] < a + row_len) ln_patch<T>(a, row_len, from[i][k], bytes[i][k], row);
          total += bytes[i][k];
        }
      }
    mbar_expect_tx(bar, total);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < NSRC; ++k)
        if (i < count && bytes[i][k] > 0) bulk_load(dst[i][k], from[i][k], bytes[i][k], bar);
  }
}

// The fetching warp: blocks of stage_rows rows, a lane per row.
template <typename T, int NSRC>
__device__ __forceinline__ void ln_fetch_all(const LnSource (&src)[NSRC], const LnRing& ring, int rows, int row_len, char* ring_mem, uint64_t* full,
                                             uint64_t* empty, const WaitCtx& ctx) {
  const int lane = threadIdx.x & 31;
  const int blocks = (rows + ring.stage_rows - 1) / ring.stage_rows;
  const int stage_bytes = NSRC * ring.stage_rows * ring.row_bytes;
  int stage = 0;
  uint32_t phase = 0;
  for (int blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    if (!mbar_wait(&empty[stage], phase ^ 1u, ctx, 73)) return;
    const int r = blk * ring.stage_rows + lane;
    const bool mine = lane < ring.stage_rows && r < rows;
    char* dst[NSRC];
    const char* from[NSRC];
    uint32_t bytes[NSRC], total = 0;
#pragma unroll
    for (int i = 0; i < NSRC; ++i) {
      bytes[i] = 0;
      if (mine) {
        const char* a = src[i].base + r * src[i].pitch;
        bytes[i] = ln_span(src[i], a, row_len, &from[i]);
        char* row = ring_mem + stage * stage_bytes + (lane * NSRC + i) * ring.row_bytes + (reinterpret_cast<uintptr_t>(a) & 15u);
        dst[i] = row + (from[i] - a);
        if (from[i] > a || from[i] + bytes[i] < a + row_len) ln_patch<T>(a, row_len, from[i], bytes[i], row);
      }
      total += bytes[i];
    }
    if (ring.stage_rows > 1) total = __reduce_add_sync(0xFFFFFFFFu, total);
    __syncwarp();
    if (lane == 0) mbar_expect_tx(&full[stage], total);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NSRC; ++i)
      if (mine && bytes[i] > 0) bulk_load(dst[i], from[i], bytes[i], &full[stage]);
    if (++stage == ring.stages) { stage = 0; phase ^= 1u; }
  }
}

// Sums over the TPR threads of a row; every thread gets them.  A CTA-wide sum takes a slot of `scratch` of its own per call in a row of calls (two
// suffice: a barrier lies between the reads of one call and the writes of the call after the next).  Across warps the partial sums are joined by
// shuffles too: with 16 warps, reading all of them in every thread costs 48 instructions a warp and row against 11.
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float2 v, float (*scratch)[32], int slot) {
  const int lane = threadIdx.x & 31;
  // the lower half of the warp goes on with x, the upper half with y
  const bool upper = lane >= 16;
  float t = (upper ? v.y : v.x) + __shfl_xor_sync(0xFFFFFFFFu, upper ? v.x : v.y, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
  if constexpr (TPR > 32) {
    constexpr int WARPS = TPR / 32;
    static_assert(WARPS <= 16, "half a warp joins them");
    if ((lane & 15) == 0) scratch[slot][(threadIdx.x >> 5) + (lane & 16)] = t;
    named_bar_sync(1, TPR);
    t = scratch[slot][(lane & (WARPS - 1)) + (lane & 16)];
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
  }
  return make_float2(__shfl_sync(0xFFFFFFFFu, t, 0), __shfl_sync(0xFFFFFFFFu, t, 16));
}
template <int TPR>
__device__ __forceinline__ float row_sum(float t, float (*scratch)[32], int slot) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
  if constexpr (TPR > 32) {
    constexpr int WARPS = TPR / 32;
    if (lane == 0) scratch[slot][threadIdx.x >> 5] = t;
    named_bar_sync(1, TPR);
    t = scratch[slot][lane & (WARPS - 1)];
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
  }
  return t;
}
// The sums of one row (in x) or of two.
template <int TPR, int BATCH>
__device__ __forceinline__ float2 batch_sum(float2 v, float (*scratch)[32], int slot) {
  if constexpr (BATCH == 2) return row_sum2<TPR>(v, scratch, slot);
  return make_float2(row_sum<TPR>(v.x, scratch, slot), 0.f);
}

// One access of w or b, or what stands for it where there is none.
template <typename W, int VEC>
__device__ __forceinline__ void ln_weight(const W* w, int c, int cols, float dflt, typename Lanes<VEC>::V (&f)[Lanes<VEC>::N]) {
  if (w != nullptr && c < cols) {
    load_lanes<W, VEC>(w + c, f);
  } else {
#pragma unroll
    for (int j = 0; j < Lanes<VEC>::N; ++j) f[j] = vsplat<typename Lanes<VEC>::V>(dflt);
  }
}

// BATCH: ln_batch.
template <typename T, typename W, int VEC, int PER, int TPR, int BATCH>
__global__ void __launch_bounds__(ln_threads<TPR>(), ln_per_sm<TPR, PER * VEC, false, sizeof(T)>())
ln_fwd_kernel(const LnSource sx, const W* __restrict__ w, const W* __restrict__ b, T* __restrict__ y, float* __restrict__ mean,
              float* __restrict__ rstd, int rows, int cols, int64_t ldy, float eps, const LnRing ring, uint32_t* status) {
  constexpr int GROUPS = ln_groups<TPR>();
  constexpr bool HOLD = PER * VEC <= 16;      // w and b stay in registers
  using V = typename Lanes<VEC>::V;
  constexpr int N = Lanes<VEC>::N;
  extern __shared__ __align__(16) char ring_mem[];
  __shared__ uint64_t full[LN_MAX_STAGES], empty[LN_MAX_STAGES];
  __shared__ float scratch[2][32];
  __shared__ uint32_t abort_flag;
  if (threadIdx.x < LN_MAX_STAGES) {
    mbar_init(&full[threadIdx.x], 1);
    mbar_init(&empty[threadIdx.x], GROUPS);
  }
  if (threadIdx.x == 0) abort_flag = 0;
  fence_mbar_init();
  __syncthreads();
  const WaitCtx ctx{&abort_flag, status};
  const int group = threadIdx.x / TPR;
  constexpr bool SELF = TPR > 32, ALIGNED = VEC * sizeof(T) == 16;
  const int row_len = cols * static_cast<int>(sizeof(T));
  const LnSource src[1] = {sx};
  if (!SELF && group == GROUPS) {
    ln_fetch_all<T, 1>(src, ring, rows, row_len, ring_mem, full, empty, ctx);
  } else {
    const int lane = threadIdx.x % TPR;
    V fw[HOLD ? PER : 1][N], fb[HOLD ? PER : 1][N];
    if constexpr (HOLD) {
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        ln_weight<W, VEC>(w, (lane + k * TPR) * VEC, cols, 1.f, fw[k]);
        ln_weight<W, VEC>(b, (lane + k * TPR) * VEC, cols, 0.f, fb[k]);
      }
    }
    const float inv_n = 1.f / static_cast<float>(cols);
    const int stage_rows = TPR == 32 ? ring.stage_rows : BATCH;
    const int64_t ahead = static_cast<int64_t>(gridDim.x) * BATCH * ring.stages;      // from a stage's rows to its next ones
    if (SELF && threadIdx.x == 0)
      for (int i = 0; i < ring.stages; ++i) {
        const int64_t r = (blockIdx.x + static_cast<int64_t>(i) * gridDim.x) * BATCH;
        if (r < rows) ln_fetch_rows<T, ALIGNED, 1>(src, ring, row_len, static_cast<int>(r), min(BATCH, rows - static_cast<int>(r)), ring_mem + i * BATCH * ring.row_bytes, &full[i]);
      }
    const char* const my_ring = ring_mem + lane * VEC * static_cast<int>(sizeof(T));
    T* const my_y = y + lane * VEC;
    int stage = 0, stage_at = 0;
    uint32_t phase = 0;
    for (int top = blockIdx.x * stage_rows; top < rows; top += gridDim.x * stage_rows) {
      // a wait that gives up is on record; the rows are then worked through all the same, so that every barrier below is met
      mbar_wait(&full[stage], phase, ctx, 71);
      for (int i = group * BATCH; i < stage_rows; i += GROUPS * BATCH) {
        const int r = top + i;
        if (TPR == 32 && r >= rows) break;
        const bool two = BATCH == 2 && r + 1 < rows;
        V f[BATCH][PER][N];
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int h = 0; h < BATCH; ++h) {
          const int at = h == 1 && two ? 1 : 0;      // without a second row the first one is read again: its results are dropped
          const char* row = my_ring + stage_at + (i + at) * ring.row_bytes + (VEC * sizeof(T) == 16 ? 0 : ln_offset(sx, r + at));
          V t = vsplat<V>(0.f);
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            if (ln_inside<TPR, PER>(k, (lane + k * TPR) * VEC, cols)) {
              load_lanes<T, VEC>(reinterpret_cast<const T*>(row) + k * TPR * VEC, f[h][k]);
#pragma unroll
              for (int j = 0; j < N; ++j) t = vadd(t, f[h][k][j]);
            }
          }
          (h == 0 ? s.x : s.y) = vsum(t);
        }
        s = batch_sum<TPR, BATCH>(s, scratch, 0);
        if (TPR > 32 && lane == 0) {                                 // every thread holds its part of the stage's rows in registers
          if (top + ahead < rows) {
            const int n = static_cast<int>(top + ahead);
            ln_fetch_rows<T, ALIGNED, 1>(src, ring, row_len, n, min(BATCH, rows - n), ring_mem + stage_at, &full[stage]);
          }
        }
        const float mu[2] = {s.x * inv_n, s.y * inv_n};
        s = make_float2(0.f, 0.f);
#pragma unroll
        for (int h = 0; h < BATCH; ++h) {
          V t = vsplat<V>(0.f);
          const V minus = vsplat<V>(-mu[h]);
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            if (ln_inside<TPR, PER>(k, (lane + k * TPR) * VEC, cols)) {
#pragma unroll
              for (int j = 0; j < N; ++j) {
                f[h][k][j] = vadd(f[h][k][j], minus);
                t = vfma(f[h][k][j], f[h][k][j], t);
              }
            }
          }
          (h == 0 ? s.x : s.y) = vsum(t);
        }
        s = batch_sum<TPR, BATCH>(s, scratch, 1);
        const float rs[2] = {rsqrtf(s.x * inv_n + eps), rsqrtf(s.y * inv_n + eps)};
#pragma unroll
        for (int h = 0; h < BATCH; ++h) {
          if (h == 0 || two) {
            T* out = my_y + (r + h) * ldy;
            const V scale = vsplat<V>(rs[h]);
#pragma unroll
            for (int k = 0; k < PER; ++k) {
              const int c = (lane + k * TPR) * VEC;
              if (!ln_inside<TPR, PER>(k, c, cols)) continue;
              if constexpr (!HOLD) {
                ln_weight<W, VEC>(w, c, cols, 1.f, fw[0]);
                ln_weight<W, VEC>(b, c, cols, 0.f, fb[0]);
              }
#pragma unroll
              for (int j = 0; j < N; ++j) f[h][k][j] = vfma(vmul(f[h][k][j], scale), fw[HOLD ? k : 0][j], fb[HOLD ? k : 0][j]);
              store_lanes<T, VEC>(out + k * TPR * VEC, f[h][k]);
            }
            if (lane == 0) {
              if (mean != nullptr) mean[r + h] = mu[h];
              if (rstd != nullptr) rstd[r + h] = rs[h];
            }
          }
        }
      }
      if (TPR == 32) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
      }
      stage_at += stage_rows * ring.row_bytes;
      if (++stage == ring.stages) { stage = stage_at = 0; phase ^= 1u; }
    }
  }
  drain_after_abort(&abort_flag);
}

// Backward.  The columns' sums of dy h and dy stay in registers until the end: one partial sum per CTA (part[2][gridDim.x][cols], first dw's).
template <typename T, typename W, int VEC, int PER, int TPR>
__global__ void __launch_bounds__(ln_threads<TPR>(), ln_per_sm<TPR, PER * VEC, true, sizeof(T)>())
ln_bwd_kernel(const LnSource sg, const LnSource sx, const W* __restrict__ w, const float* __restrict__ mean, const float* __restrict__ rstd,
              T* __restrict__ dx, float* __restrict__ part, int rows, int cols, int64_t lddx, const LnRing ring, uint32_t* status) {
  constexpr int GROUPS = ln_groups<TPR>();
  // Up to 16 elements a thread, w stays in registers, and u and h do between the row sum and dx.  With 32, half as many warps share a row's fixed work
  // (about 80 instructions a warp); w is read from shared memory, and x and dy once more from the ring.
  constexpr bool HOLD = PER * VEC <= 16;
  using V = typename Lanes<VEC>::V;
  constexpr int N = Lanes<VEC>::N;
  extern __shared__ __align__(16) char ring_mem[];
  __shared__ uint64_t full[LN_MAX_STAGES], empty[LN_MAX_STAGES];
  __shared__ float scratch[2][32];
  __shared__ uint32_t abort_flag;
  if (threadIdx.x < LN_MAX_STAGES) {
    mbar_init(&full[threadIdx.x], 1);
    mbar_init(&empty[threadIdx.x], GROUPS);
  }
  if (threadIdx.x == 0) abort_flag = 0;
  fence_mbar_init();
  __syncthreads();
  const WaitCtx ctx{&abort_flag, status};
  const int group = threadIdx.x / TPR;
  constexpr bool SELF = TPR > 32, ALIGNED = VEC * sizeof(T) == 16;
  const int row_len = cols * static_cast<int>(sizeof(T));
  const LnSource src[2] = {sg, sx};
  if (!SELF && group == GROUPS) {
    ln_fetch_all<T, 2>(src, ring, rows, row_len, ring_mem + ring.weight_bytes, full, empty, ctx);
  } else {
    const int lane = threadIdx.x % TPR;
    W* const held_w = reinterpret_cast<W*>(ring_mem);
    if constexpr (!HOLD) {                  // each thread copies what it will read itself
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int c = (lane + k * TPR) * VEC;
        V t[N];
        ln_weight<W, VEC>(w, c, cols, 1.f, t);
        if (c < cols) store_lanes<W, VEC>(held_w + c, t);
      }
    }
    V fw[HOLD ? PER : 1][N], aw[PER][N], ab[PER][N];
    if constexpr (!HOLD) {
#pragma unroll
      for (int j = 0; j < N; ++j) fw[0][j] = vsplat<V>(0.f);     // behind the row's end it meets a zero dy
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if constexpr (HOLD) ln_weight<W, VEC>(w, (lane + k * TPR) * VEC, cols, 1.f, fw[k]);
#pragma unroll
      for (int j = 0; j < N; ++j) aw[k][j] = ab[k][j] = vsplat<V>(0.f);
    }
    const float inv_n = 1.f / static_cast<float>(cols);
    const int stage_rows = TPR == 32 ? ring.stage_rows : 1;
    // Rows that are under way beside the one worked on.  When that one is not held in registers, its stage is only free when the next row's barrier is
    // passed, so that one stage less is.
    const int under_way = HOLD || ring.stages == 1 ? ring.stages : ring.stages - 1;
    const int64_t ahead = static_cast<int64_t>(gridDim.x) * under_way;
    char* const stages = ring_mem + ring.weight_bytes;
    if (SELF && threadIdx.x == 0)
      for (int i = 0; i < under_way; ++i) {
        const int64_t n = blockIdx.x + static_cast<int64_t>(i) * gridDim.x;
        if (n < rows) ln_fetch_rows<T, ALIGNED, 2>(src, ring, row_len, static_cast<int>(n), 1, stages + 2 * i * ring.row_bytes, &full[i]);
      }
    const char* const my_ring = ring_mem + ring.weight_bytes + lane * VEC * static_cast<int>(sizeof(T));
    T* const my_dx = dx + lane * VEC;
    int stage = 0, stage_at = 0, slot = 0;
    uint32_t phase = 0;
    int r = blockIdx.x * stage_rows + group;
    float mu = r < rows ? mean[r] : 0.f, rs = r < rows ? rstd[r] : 0.f;
    for (int top = blockIdx.x * stage_rows; top < rows; top += gridDim.x * stage_rows) {
      mbar_wait(&full[stage], phase, ctx, 72);
      for (int i = group; i < stage_rows; i += GROUPS) {
        r = top + i;
        if (TPR == 32 && r >= rows) break;
        // h = x rstd - mean rstd: the product rounded once is as far off as the mean itself, which is rounded too
        const V shift = vsplat<V>(-mu * rs), q = vsplat<V>(rs);
        const float rs_now = rs;
        {                                                       // the next row's statistics
          const int n = i + GROUPS < stage_rows ? r + GROUPS : top + gridDim.x * stage_rows + group;
          if (n < rows) {
            mu = mean[n];
            rs = rstd[n];
          }
        }
        const char* row = my_ring + stage_at + 2 * i * ring.row_bytes;
        const T* row_g = reinterpret_cast<const T*>(row + (VEC * sizeof(T) == 16 ? 0 : ln_offset(sg, r)));
        const T* row_x = reinterpret_cast<const T*>(row + ring.row_bytes + (VEC * sizeof(T) == 16 ? 0 : ln_offset(sx, r)));
        // dy and h of one access; zeros behind the row's end, so that nothing there enters a sum
        auto terms = [&](int k, V (&g)[N], V (&h)[N]) {
          const int c = (lane + k * TPR) * VEC;
          if (ln_inside<TPR, PER>(k, c, cols)) {
            load_lanes<T, VEC>(row_g + k * TPR * VEC, g);
            load_lanes<T, VEC>(row_x + k * TPR * VEC, h);
          } else {
#pragma unroll
            for (int j = 0; j < N; ++j) g[j] = h[j] = vsplat<V>(0.f);
          }
          if constexpr (!HOLD) {
            if (ln_inside<TPR, PER>(k, c, cols)) load_lanes<W, VEC>(held_w + c, fw[0]);
          }
#pragma unroll
          for (int j = 0; j < N; ++j) h[j] = vfma(h[j], q, shift);
        };
        V g[HOLD ? PER : 1][N], h[HOLD ? PER : 1][N];
        V s1 = vsplat<V>(0.f), s2 = vsplat<V>(0.f);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          V (&gk)[N] = g[HOLD ? k : 0];
          V (&hk)[N] = h[HOLD ? k : 0];
          terms(k, gk, hk);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            aw[k][j] = vfma(gk[j], hk[j], aw[k][j]);
            ab[k][j] = vadd(ab[k][j], gk[j]);
            gk[j] = vmul(gk[j], fw[HOLD ? k : 0][j]);            // u
            s1 = vadd(s1, gk[j]);
            s2 = vfma(gk[j], hk[j], s2);
          }
        }
        float2 s = make_float2(vsum(s1), vsum(s2));
        s = row_sum2<TPR>(s, scratch, slot);
        slot ^= 1;
        if (SELF && threadIdx.x == 0 && top + ahead < rows) {   // behind the barrier every thread is past the row before, or holds this one
          if (HOLD) {
            ln_fetch_rows<T, ALIGNED, 2>(src, ring, row_len, static_cast<int>(top + ahead), 1, stages + stage_at, &full[stage]);
          } else if (ring.stages > 1) {
            const int before = stage == 0 ? ring.stages - 1 : stage - 1;
            ln_fetch_rows<T, ALIGNED, 2>(src, ring, row_len, static_cast<int>(top + ahead), 1, stages + 2 * before * ring.row_bytes, &full[before]);
          }
        }
        if (dx != nullptr) {
          const V c1 = vsplat<V>(-s.x * inv_n * rs_now), c2 = vsplat<V>(-s.y * inv_n * rs_now);
          T* out = my_dx + r * lddx;
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            const int c = (lane + k * TPR) * VEC;
            V (&gk)[N] = g[HOLD ? k : 0];
            V (&hk)[N] = h[HOLD ? k : 0];
            if constexpr (!HOLD) {                                // read once more instead of held
              terms(k, gk, hk);
#pragma unroll
              for (int j = 0; j < N; ++j) gk[j] = vmul(gk[j], fw[0][j]);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) gk[j] = vfma(hk[j], c2, vfma(gk[j], q, c1));
            if (ln_inside<TPR, PER>(k, c, cols)) store_lanes<T, VEC>(out + k * TPR * VEC, gk);
          }
        }
      }
      if (TPR == 32) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[stage]);
      } else if (!HOLD && ring.stages == 1) {
        named_bar_sync(2, TPR);                                 // the only stage is free
        if (threadIdx.x == 0 && top + ahead < rows) ln_fetch_rows<T, ALIGNED, 2>(src, ring, row_len, static_cast<int>(top + ahead), 1, stages, &full[0]);
      }
      stage_at += 2 * stage_rows * ring.row_bytes;
      if (++stage == ring.stages) { stage = stage_at = 0; phase ^= 1u; }
    }
    grid_launch_dependents();
    if (part != nullptr) {
      float* out_w = part + static_cast<int64_t>(blockIdx.x) * cols;
      float* out_b = part + static_cast<int64_t>(gridDim.x + blockIdx.x) * cols;
      if constexpr (GROUPS == 1) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int c = (lane + k * TPR) * VEC;
          if (c < cols) {
            store_lanes<float, VEC>(out_w + c, aw[k]);
            store_lanes<float, VEC>(out_b + c, ab[k]);
          }
        }
      } else {
        // the warps' sums one after the other, in a fixed order
        __shared__ __align__(16) float sums_w[TPR * PER * VEC], sums_b[TPR * PER * VEC];
        for (int g = 0; g < GROUPS; ++g) {
          if (group == g) {
#pragma unroll
            for (int k = 0; k < PER; ++k) {
              const int c = (lane + k * TPR) * VEC;
              V tw[N], tb[N];
              load_lanes<float, VEC>(sums_w + c, tw);
              load_lanes<float, VEC>(sums_b + c, tb);
#pragma unroll
              for (int j = 0; j < N; ++j) {
                tw[j] = g > 0 ? vadd(tw[j], aw[k][j]) : aw[k][j];
                tb[j] = g > 0 ? vadd(tb[j], ab[k][j]) : ab[k][j];
              }
              store_lanes<float, VEC>(sums_w + c, tw);
              store_lanes<float, VEC>(sums_b + c, tb);
            }
          }
          named_bar_sync(1, GROUPS * TPR);
        }
        for (int c = threadIdx.x; c < cols; c += GROUPS * TPR) {
          out_w[c] = sums_w[c];
          out_b[c] = sums_b[c];
        }
      }
    }
  }
  drain_after_abort(&abort_flag);
}

// dw[c] and db[c]: the sums over the parts, in a fixed order.
template <typename W>
__global__ void __launch_bounds__(1024) ln_dw_join_kernel(const float* __restrict__ part, W* __restrict__ dw, W* __restrict__ db, int parts,
                                                          int64_t cols) {
  __shared__ float sums[32][33];
  grid_wait();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  const float* p = part + static_cast<int64_t>(blockIdx.y) * parts * cols;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 4
    for (int i = slice; i < parts; i += 32) s += p[static_cast<int64_t>(i) * cols + c];
  }
  sums[slice][lane] = s;
  __syncthreads();
  // warp i now adds the 32 slices of column i
  s = warp_sum(sums[lane][slice]);
  W* out = blockIdx.y == 0 ? dw : db;
  const int64_t mine = static_cast<int64_t>(blockIdx.x) * 32 + slice;
  if (lane == 0 && mine < cols && out != nullptr) out[mine] = from_f32<W>(s);
}

// ---------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------
static int ln_parts(int64_t rows) { return static_cast<int>(rows < LN_MAX_PARTS ? rows : LN_MAX_PARTS); }

int64_t layer_norm_bwd_workspace(int64_t rows, int64_t cols) { return 2 * ln_parts(rows) * cols; }

// Largest power of two (at most 16) that divides every byte address and pitch given.
static int ln_alignment(std::initializer_list<uintptr_t> v) {
  uintptr_t all = 16;
  for (uintptr_t x : v) all |= x;
  return static_cast<int>(all & (~all + 1));
}
static LnSource ln_source(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t size) {
  const char* base = static_cast<const char*>(p);
  return LnSource{base, ld * size, base + ((rows - 1) * ld + cols) * size};
}
// The ring of a CTA: a few KB per stage (a row or a batch of them for a CTA-wide row, some for every warp otherwise), and two stages or what makes
// LN_AHEAD_FWD / LN_AHEAD_BWD bytes per SM, where the CTA's share of the shared memory holds them.  stages < 1: the rows are too long.
// More reads under way than HBM's latency asks for hold up the writes.  bf16, us by the stages of a CTA and what they hold per SM (the first is what the
// constants make):
//   forward   16384 x 4096   2 (48 KB) 47, 3 (72) 47, 4 (96) 50, 8 (192) 55        65536 x 4096   168, 190, 198, 204
//             32768 x 2048   3 (60 KB) 45, 4 (80) 48, 8 (160) 55                   4096 x 16384   2 (128 KB) 50, 3 (192) 60
//   backward  131072 x 512   4 (128 KB) 81, 2 (64) 97, 3 (96) 84, 6 (192) 89       16384 x 4096   4 (128 KB) 70, 2 (64) 71, 3 (96) 70, 6 (192) 72
// The backward reads twice as much as it writes and is slowed by fewer.
constexpr int LN_SMEM = 212 * 1024;     // shared memory that the CTAs of an SM divide
constexpr int LN_AHEAD_FWD = 60 * 1024, LN_AHEAD_BWD = 140 * 1024;
static LnRing ln_ring(int64_t cols, int size, int align, int operands, int groups, int per_sm, int batch, int weight_size) {
  LnRing r;
  r.row_bytes = static_cast<int>((cols * size + 15) / 16 * 16) + (align == 16 ? 0 : 16);
  r.stage_rows = groups == 1 ? batch : r.row_bytes * operands <= 256 ? 4 * groups : r.row_bytes * operands <= 1024 || batch == 2 ? 2 * groups : groups;
  r.weight_bytes = static_cast<int>((cols * weight_size + 15) / 16 * 16);
  const int64_t stage_bytes = static_cast<int64_t>(r.stage_rows) * r.row_bytes * operands;
  const int64_t most = (static_cast<int64_t>(LN_SMEM) / per_sm - r.weight_bytes) / stage_bytes;
  int64_t stages = (operands == 1 ? LN_AHEAD_FWD : LN_AHEAD_BWD) / per_sm / stage_bytes;
  if (stages < 2) stages = 2;
  if (stages > most) stages = most;
  r.stages = static_cast<int>(stages > LN_MAX_STAGES ? LN_MAX_STAGES : stages);
  return r;
}

template <typename T, typename W, int VEC, int PER, int TPR>
static int ln_fwd_rows(const LayerNormArgs& a, int align, const DeviceInfo* dev, cudaStream_t stream, bool* done) {
  constexpr int GROUPS = ln_groups<TPR>(), PER_SM = ln_per_sm<TPR, PER * VEC, false, sizeof(T)>(), BATCH = ln_batch<TPR, PER * VEC, sizeof(T), sizeof(W)>();
  const LnRing ring = ln_ring(a.cols, sizeof(T), align, 1, GROUPS, PER_SM, BATCH, 0);
  if (ring.stages < 1 || (TPR > 32 && a.cols <= TPR * VEC * (PER / 2))) return B200K_OK;   // the second is what ln_inside relies on
  auto kernel = ln_fwd_kernel<T, W, VEC, PER, TPR, BATCH>;
  const int smem = ring.stages * ring.stage_rows * ring.row_bytes;
  B200K_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LN_SMEM));
  const int64_t most = (a.rows + ring.stage_rows - 1) / ring.stage_rows, grid = static_cast<int64_t>(dev->sm_count) * PER_SM;
  kernel<<<static_cast<unsigned>(most < grid ? most : grid), ln_threads<TPR>(), smem, stream>>>(
      ln_source(a.x, a.rows, a.cols, a.ldx, sizeof(T)), static_cast<const W*>(a.w), static_cast<const W*>(a.b), static_cast<T*>(a.y), a.mean, a.rstd,
      static_cast<int>(a.rows), static_cast<int>(a.cols), a.ldy, a.eps, ring, dev->status_word);
  count_launch();
  B200K_CHECK_LAUNCH("ln_fwd_kernel");
  *done = true;
  return B200K_OK;
}

template <typename T, typename W, int VEC, int PER, int TPR>
static int ln_bwd_rows(const LayerNormArgs& a, int align, const DeviceInfo* dev, float* part, int* parts, cudaStream_t stream, bool* done) {
  constexpr int GROUPS = ln_groups<TPR>(), PER_SM = ln_per_sm<TPR, PER * VEC, true, sizeof(T)>();
  const LnRing ring = ln_ring(a.cols, sizeof(T), align, 2, GROUPS, PER_SM, 1, PER * VEC > 16 ? sizeof(W) : 0);
  if (ring.stages < 1 || (TPR > 32 && a.cols <= TPR * VEC * (PER / 2))) return B200K_OK;   // the second is what ln_inside relies on
  auto kernel = ln_bwd_kernel<T, W, VEC, PER, TPR>;
  const int smem = ring.weight_bytes + 2 * ring.stages * ring.stage_rows * ring.row_bytes;
  B200K_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LN_SMEM));
  int64_t grid = (a.rows + ring.stage_rows - 1) / ring.stage_rows;
  if (grid > static_cast<int64_t>(dev->sm_count) * PER_SM) grid = static_cast<int64_t>(dev->sm_count) * PER_SM;
  if (grid > LN_MAX_PARTS) grid = LN_MAX_PARTS;
  *parts = static_cast<int>(grid);
  kernel<<<static_cast<unsigned>(grid), ln_threads<TPR>(), smem, stream>>>(
      ln_source(a.dy, a.rows, a.cols, a.lddy, sizeof(T)), ln_source(a.x, a.rows, a.cols, a.ldx, sizeof(T)), static_cast<const W*>(a.w), a.mean,
      a.rstd, static_cast<T*>(a.dx), part, static_cast<int>(a.rows), static_cast<int>(a.cols), a.lddx, ring, dev->status_word);
  count_launch();
  B200K_CHECK_LAUNCH("ln_bwd_kernel");
  *done = true;
  return B200K_OK;
}

// Calls f with the kernel shape for rows of `cols` elements of `size` bytes whose operands share `align`: (VEC, PER, TPR) as integral constants.
// 16 elements a thread or less, 32 beyond 8192, where no more threads are to be had; false beyond 16384 elements.  A warp takes a row of up to 512; a
// CTA-wide shape is the smallest one that holds the row, so that more than half of it is filled.
template <int N>
using Int = std::integral_constant<int, N>;
template <int SIZE, typename F>
static bool ln_shape(int64_t cols, int align, F&& f) {
  constexpr int V = 16 / SIZE;
  if (align == 16) {
    const int64_t u = cols / V;
    if (u <= 32) f(Int<V>(), Int<1>(), Int<32>());
    else if (u <= 64) f(Int<V>(), Int<2>(), Int<32>());
    else if (u <= 512 / V) f(Int<V>(), Int<16 / V>(), Int<32>());       // fp32 alone: 64 accesses hold 512 16-bit elements
    else if (u <= 1024 / V) f(Int<V>(), Int<8 / V>(), Int<128>());
    else if (u <= 2 * 1024 / V) f(Int<V>(), Int<16 / V>(), Int<128>());
    else if (u <= 4 * 1024 / V) f(Int<V>(), Int<16 / V>(), Int<256>());
    else if (u <= 8 * 1024 / V) f(Int<V>(), Int<16 / V>(), Int<512>());
    else if (u <= 16 * 1024 / V) f(Int<V>(), Int<32 / V>(), Int<512>());
    else return false;
    return true;
  }
  if constexpr (SIZE == 2) if (align >= 4) {
    if (cols <= 256) f(Int<2>(), Int<4>(), Int<32>());
    else if (cols <= 512) f(Int<2>(), Int<8>(), Int<32>());
    else if (cols <= 1024) f(Int<2>(), Int<4>(), Int<128>());
    else if (cols <= 2048) f(Int<2>(), Int<8>(), Int<128>());
    else if (cols <= 4096) f(Int<2>(), Int<8>(), Int<256>());
    else if (cols <= 8192) f(Int<2>(), Int<8>(), Int<512>());
    else if (cols <= 16384) f(Int<2>(), Int<16>(), Int<512>());
    else return false;
    return true;
  }
  if (cols <= 256) f(Int<1>(), Int<8>(), Int<32>());
  else if (cols <= 512) f(Int<1>(), Int<16>(), Int<32>());
  else if (cols <= 1024) f(Int<1>(), Int<8>(), Int<128>());
  else if (cols <= 2048) f(Int<1>(), Int<16>(), Int<128>());
  else if (cols <= 4096) f(Int<1>(), Int<16>(), Int<256>());
  else if (cols <= 8192) f(Int<1>(), Int<16>(), Int<512>());
  else if (cols <= 16384) f(Int<1>(), Int<32>(), Int<512>());
  else return false;
  return true;
}

// The alignment of x's accesses that the weights allow too: VEC elements of x go with VEC elements of w.
template <typename T, typename W>
static int ln_common_alignment(int rows_align, const void* w, const void* b) {
  const int weights = ln_alignment({reinterpret_cast<uintptr_t>(w), reinterpret_cast<uintptr_t>(b)});
  const int allowed = weights == 16 ? 16 : weights * static_cast<int>(sizeof(T)) / static_cast<int>(sizeof(W));
  return rows_align < allowed ? rows_align : allowed;
}

template <typename T, typename W>
static int ln_fwd(const LayerNormArgs& a, const DeviceInfo* dev, cudaStream_t stream) {
  constexpr uintptr_t S = sizeof(T);
  const int align = ln_common_alignment<T, W>(ln_alignment({reinterpret_cast<uintptr_t>(a.x), reinterpret_cast<uintptr_t>(a.y), a.cols * S, a.ldx * S, a.ldy * S}), a.w, a.b);
  int rc = B200K_OK;
  bool done = false;
  if (a.rows < (int64_t(1) << 30)) ln_shape<S>(a.cols, align, [&](auto vec, auto per, auto tpr) { rc = ln_fwd_rows<T, W, vec(), per(), tpr()>(a, align, dev, stream, &done); });
  if (rc != B200K_OK || done) return rc;
  const unsigned grid = static_cast<unsigned>(a.rows < (1 << 30) ? a.rows : (1 << 30));
  ln_fwd_loop_kernel<T, W><<<grid, 512, 0, stream>>>(static_cast<const T*>(a.x), static_cast<const W*>(a.w), static_cast<const W*>(a.b),
                                                     static_cast<T*>(a.y), a.mean, a.rstd, a.rows, a.cols, a.ldx, a.ldy, a.eps);
  count_launch();
  B200K_CHECK_LAUNCH("ln_fwd_loop_kernel");
  return B200K_OK;
}

template <typename T, typename W>
static int ln_bwd_main(const LayerNormArgs& a, const DeviceInfo* dev, float* part, int* parts, cudaStream_t stream) {
  constexpr uintptr_t S = sizeof(T);
  const int align = ln_common_alignment<T, W>(ln_alignment({reinterpret_cast<uintptr_t>(a.x), reinterpret_cast<uintptr_t>(a.dy), reinterpret_cast<uintptr_t>(a.dx),
                                                            a.cols * S, a.ldx * S, a.lddy * S, a.dx == nullptr ? 0 : a.lddx * S}), a.w, nullptr);
  int rc = B200K_OK;
  bool done = false;
  if (a.rows < (int64_t(1) << 30)) ln_shape<S>(a.cols, align, [&](auto vec, auto per, auto tpr) { rc = ln_bwd_rows<T, W, vec(), per(), tpr()>(a, align, dev, part, parts, stream, &done); });
  if (rc != B200K_OK || done) return rc;
  const T* dy = static_cast<const T*>(a.dy);
  const T* x = static_cast<const T*>(a.x);
  if (a.dx != nullptr) {
    const unsigned grid = static_cast<unsigned>(a.rows < (1 << 30) ? a.rows : (1 << 30));
    ln_dx_loop_kernel<T, W><<<grid, 512, 0, stream>>>(dy, x, static_cast<const W*>(a.w), a.mean, a.rstd, static_cast<T*>(a.dx), a.rows, a.cols,
                                                      a.lddy, a.ldx, a.lddx);
    count_launch();
    B200K_CHECK_LAUNCH("ln_dx_loop_kernel");
  }
  if (part != nullptr) {
    *parts = ln_parts(a.rows);
    ln_dw_loop_kernel<T><<<dim3(static_cast<unsigned>((a.cols + 255) / 256), *parts), 256, 0, stream>>>(dy, x, a.mean, a.rstd, part, a.rows, a.cols,
                                                                                                      a.lddy, a.ldx);
    count_launch();
    B200K_CHECK_LAUNCH("ln_dw_loop_kernel");
  }
  return B200K_OK;
}

template <typename T, typename W>
static int ln_bwd(const LayerNormArgs& a, const DeviceInfo* dev, cudaStream_t stream) {
  const bool sums = a.dw != nullptr || a.db != nullptr;
  int parts = 0;
  if (a.rows > 0 && (sums || a.dx != nullptr)) {
    const int rc = ln_bwd_main<T, W>(a, dev, sums ? a.workspace : nullptr, &parts, stream);
    if (rc != B200K_OK) return rc;
  }
  if (sums) {
    B200K_CHECK_CUDA(launch_dependent(ln_dw_join_kernel<W>, dim3(static_cast<unsigned>((a.cols + 31) / 32), 2), dim3(1024), 0, stream, a.workspace,
                                      static_cast<W*>(a.dw), static_cast<W*>(a.db), parts, a.cols));
    count_launch();
    B200K_CHECK_LAUNCH("ln_dw_join_kernel");
  }
  return B200K_OK;
}

template <typename F>
static int ln_dispatch(const LayerNormArgs& a, F&& f) {
  const bool wide = a.wdtype == B200K_DTYPE_F32;
  switch (a.dtype) {
    case B200K_DTYPE_F32: return f(float(), float());
    case B200K_DTYPE_BF16: return wide ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
    default: return wide ? f(__half(), float()) : f(__half(), __half());
  }
}

static int ln_check(const LayerNormArgs& a, const char* what) {
  if (a.dtype < B200K_DTYPE_F32 || a.dtype > B200K_DTYPE_F16) return set_error(B200K_ERR_INVALID_ARG, "%s: bad element type %d", what, a.dtype);
  if (a.wdtype != a.dtype && a.wdtype != B200K_DTYPE_F32)
    return set_error(B200K_ERR_INVALID_ARG, "%s: weight and bias have the type of x or fp32 (got %d for x of type %d)", what, a.wdtype, a.dtype);
  if (a.rows < 0 || a.cols < 1 || a.cols > (int64_t(1) << 31) - 512)
    return set_error(B200K_ERR_INVALID_ARG, "%s: rows >= 0 and 1 <= cols < 2^31 - 512 expected (got %lld x %lld)", what, (long long)a.rows, (long long)a.cols);
  const uintptr_t size = a.dtype == B200K_DTYPE_F32 ? 4 : 2, wsize = a.wdtype == B200K_DTYPE_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.dy) | reinterpret_cast<uintptr_t>(a.dx)) & (size - 1) ||
      (reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.b) | reinterpret_cast<uintptr_t>(a.dw) | reinterpret_cast<uintptr_t>(a.db)) & (wsize - 1) ||
      (reinterpret_cast<uintptr_t>(a.mean) | reinterpret_cast<uintptr_t>(a.rstd)) & 3u || reinterpret_cast<uintptr_t>(a.workspace) & 15u)
    return set_error(B200K_ERR_INVALID_ARG, "%s: a pointer is not aligned to its element size, or the workspace not to 16 bytes", what);
  if (a.rows > 0 && a.cols > (int64_t(1) << 62) / a.rows) return set_error(B200K_ERR_INVALID_ARG, "%s: too many elements", what);
  return B200K_OK;
}

int layer_norm_fwd(const LayerNormArgs& a, cudaStream_t stream) {
  const int rc = ln_check(a, "layer_norm");
  if (rc != B200K_OK) return rc;
  if (!(a.eps >= 0.f)) return set_error(B200K_ERR_INVALID_ARG, "layer_norm: eps must be >= 0");
  if (a.rows == 0) return B200K_OK;
  if (a.x == nullptr || a.y == nullptr) return set_error(B200K_ERR_INVALID_ARG, "layer_norm: null pointer");
  if (a.ldx < 0 || a.ldy < a.cols) return set_error(B200K_ERR_INVALID_ARG, "layer_norm: bad row stride");
  const DeviceInfo* dev = current_device_info();
  if (dev == nullptr) return B200K_ERR_NO_DEVICE;
  return ln_dispatch(a, [&](auto t, auto w) { return ln_fwd<decltype(t), decltype(w)>(a, dev, stream); });
}

int layer_norm_bwd(const LayerNormArgs& a, cudaStream_t stream) {
  const int rc = ln_check(a, "layer_norm_backward");
  if (rc != B200K_OK) return rc;
  const bool sums = a.dw != nullptr || a.db != nullptr;
  if (a.rows > 0) {
    if (a.dy == nullptr || a.x == nullptr || a.mean == nullptr || a.rstd == nullptr)
      return set_error(B200K_ERR_INVALID_ARG, "layer_norm_backward: null pointer");
    if (a.ldx < 0 || a.lddy < 0 || (a.dx != nullptr && a.lddx < a.cols)) return set_error(B200K_ERR_INVALID_ARG, "layer_norm_backward: bad row stride");
    if (sums && (a.workspace == nullptr || a.workspace_floats < layer_norm_bwd_workspace(a.rows, a.cols)))
      return set_error(B200K_ERR_INVALID_ARG, "layer_norm_backward: a workspace of %lld floats is needed (got %lld)",
                       (long long)layer_norm_bwd_workspace(a.rows, a.cols), (long long)(a.workspace == nullptr ? 0 : a.workspace_floats));
  }
  const DeviceInfo* dev = current_device_info();
  if (dev == nullptr) return B200K_ERR_NO_DEVICE;
  return ln_dispatch(a, [&](auto t, auto w) { return ln_bwd<decltype(t), decltype(w)>(a, dev, stream); });
}

}  // namespace b200k
