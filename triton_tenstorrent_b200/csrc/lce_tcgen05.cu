// Cross entropy of a linear output layer, logits = h W^T over a vocabulary of V, forward and backward, without keeping the logits:
//
//   loss_i = lse_i - logits[i, y_i],   lse_i = log sum_v exp(logits[i, v])
//   dlogits[i, v] = g_i (exp(logits[i, v] - lse_i) - [v = y_i]),   dh = dlogits W,   dW = dlogits^T h
//
// Forward: one matrix product whose epilogue reduces each 256-column tile of the fp32 accumulators to a maximum and a sum of exponentials per
// row; a second kernel joins the tiles' pairs.  Backward, for one piece of the vocabulary after the other: the logits of the piece again,
// turned in the epilogue into dlogits in 16 bits; then dW of the piece (all tokens summed in one accumulator) and the piece's share of dh
// (summed over the pieces in fp32).  8 T V D floating-point operations (forward 2, backward 6 of which 2 are the recomputation).
//
// Tokens whose target is `ignore_index` are left out before the first product: a gather kernel moves the rows that count to the front of a
// copy of h and writes their number to device memory, where the products read it.  Work and time shrink with the tokens that carry a loss,
// and whatever stands in the rows of the others (padding, infinities) is never read by a product.
//
// The products run on CTA pairs (tcgen05, cta_group::2, 256 x 256 tiles, fp32 accumulators in tensor memory): warp 0 loads both operands by
// TMA into a six-stage ring, one thread of warp 1 issues the MMAs, the other warps run the epilogue of tile i during the main loop of tile i + 1.
// Bound: the tensor pipe; with few tokens the stream of W from HBM.  Measured, single launches at 2048 x 32000 x 4096 bf16: logits 340 us (1580 TFLOP/s, pipe
// active 88 %), dlogits 347, dW 332, dh 364; 8192 tokens, D = 4096, V = 128000, forward and backward back to back: 26.3 ms, 1310 TFLOP/s at the power cap.
#include <string.h>

#include "attn_common.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace b200k {

// Each step of 16 along K truncates the tensor cores' running sum towards zero, which takes 2^-25 of it on average: K = 4096 in one go leaves a logit of
// growing sums 3.8e-6 of itself too small, K = 8192 7.7e-6 (measured).  So the logits are summed over LCE_SEGMENT steps of 64 in tensor memory and these
// parts in fp32 registers, rounded to nearest: about 2^-22 of it (2.4e-7), whatever K is, and nothing where the products' sums are exact.  Eight epilogue
// warps hold a tile's sums, 128 columns of a row each (4096 x 65536 x 2048 bf16: 1 % slower than one go on four; parts of 1024 instead: 0.5 %).  The
// gradients' products, whose results are rounded to 16 bits, sum in one go on four.
constexpr int LCE_SEGMENT = 8;
__host__ __device__ constexpr bool lce_logits(int epi) { return epi <= 1; }                          // STATS, DLOGITS
__host__ __device__ constexpr int lce_epi_warps(int epi) { return lce_logits(epi) ? 8 : 4; }
__host__ __device__ constexpr int lce_threads(int epi) { return 64 + 32 * lce_epi_warps(epi); }
constexpr int LCE_STAGES = 6;
constexpr int LCE_BOX_BYTES = 64 * 128;                     // 64 rows of 128 bytes
constexpr int LCE_A_BYTES = 2 * LCE_BOX_BYTES;              // a CTA's 128 x 64 share of A
constexpr int LCE_B_BYTES = 2 * LCE_BOX_BYTES;              // its half of B: 128 x 64
constexpr int LCE_C_BUF_BYTES = 32 * 128;
constexpr int LCE_A_OFF = 0;
constexpr int LCE_B_OFF = LCE_STAGES * LCE_A_BYTES;
constexpr int LCE_C_OFF = LCE_B_OFF + LCE_STAGES * LCE_B_BYTES;
constexpr int LCE_BAR_OFF = LCE_C_OFF + 8 * LCE_C_BUF_BYTES;     // two staging buffers for each of four epilogue warps, one for each of eight
constexpr int LCE_SMEM = LCE_BAR_OFF + (2 * LCE_STAGES + 4) * 8 + 16 + 1024;
static_assert(LCE_SMEM <= 232448, "shared memory budget exceeded");

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
// dlogits are stored as dlogits / max|g| * 2^14 in fp16 (at most 2^14 in magnitude, and probabilities down to 2^-38 survive; unscaled ones below
// 2^-24 would be lost) and without the power of two in bf16, whose range is fp32's.
constexpr float LCE_F16_SCALE = 16384.f;

enum { LCE_STATS = 0, LCE_DLOGITS = 1, LCE_DW = 2, LCE_DH = 3 };

struct LceGemmParams {
  const int* count;        // tokens that carry a loss (device memory)
  int M, N, K;             // sizes of the launch; M of STATS, DLOGITS and DH and K of DW are bounds that `count` replaces
  int group_m;             // tile rows of a group (their A panel stays in L2 while the tile columns stream)
  int f16;
  uint32_t idesc, idesc_half;
  uint32_t* status;
  const int* target;       // per row that counts: its target (STATS, DLOGITS)
  const int64_t* token_target;   // STATS without a gather: per token
  int width;               // STATS on single CTAs: columns of a tile
  int col_base;            // first vocabulary entry of the piece
  float2* part;            // STATS: [tile column][rows] (maximum * log2 e, sum of exponentials)
  int64_t part_ld;
  float* target_logit;     // STATS
  const float* lse2;       // DLOGITS: lse * log2 e
  const float* row_scale;  // DLOGITS: factor of the row
  const float* alpha;      // DW, DH: factor of the result (device memory)
  const float* add;        // DH: fp32 sum over the earlier pieces, or null
  float* sum;              // DH: where the sum so far goes, max_splits buffers split_stride apart
  int64_t split_stride;
  int max_splits, last;    // DH: last = the last piece
  void* out;               // DH, last piece without splits: dh
  const int* token;        // DH: token of a row
};

// Parts that the K axis of the dh product is cut in: with fewer tiles than CTA pairs, or a last wave that is nearly empty, the parts of a tile go to
// different pairs, which leave fp32 sums that lce_dh_kernel adds.  Cost of s parts, in steps of 64 along K (0.28 us): waves of K / s steps, about 8
// steps for filling the pipeline and the epilogue of each, and a part's sums written and read (a tile: 0.3 steps of all pairs).  Cutting at all
// has to gain 3 %.  The whole warp calls it, a lane per s.
constexpr int LCE_MAX_SPLITS = 32;
__device__ __forceinline__ int lce_splits(int tiles, int pairs, int num_kb, int max_splits) {
  if (max_splits <= 1) return 1;
  const int s = static_cast<int>(lane_id()) + 1;
  auto cost = [&](int parts) { return static_cast<int64_t>((tiles * parts + pairs - 1) / pairs) * ((num_kb + parts - 1) / parts + 8); };
  const int64_t c = s == 1 ? cost(1) : cost(s) + cost(1) / 32 + static_cast<int64_t>(tiles) * s * 5 / 16;
  const uint32_t key = s > max_splits ? 0xFFFFFFFFu : static_cast<uint32_t>(min(c, static_cast<int64_t>((1 << 27) - 1))) << 5 | static_cast<uint32_t>(s - 1);
  return static_cast<int>(__reduce_min_sync(0xFFFFFFFFu, key) & 31u) + 1;
}

struct LceWork {
  int pid_m, pid_n, col0, width, split;
};
struct LceSchedule {
  int num_pid_m, num_pid_n, group_m, full_work, num_work, splits;
};
// Tiles in groups of group_m rows, odd groups backwards; the tiles of a last wave that occupy at most half of the pairs are cut in two column
// halves (the order and the split of the matmul kernel).
__device__ __forceinline__ LceSchedule lce_schedule(int M, int N, int group_m, int pairs, int splits) {
  LceSchedule s;
  s.num_pid_m = (M + 255) >> 8;
  s.num_pid_n = (N + 255) >> 8;
  s.group_m = group_m;
  s.splits = splits;
  const int tiles = s.num_pid_m * s.num_pid_n;
  const int rest = tiles % pairs;
  s.full_work = s.num_work = tiles * splits;
  if (splits == 1 && rest > 0 && 2 * rest <= pairs) {
    s.full_work = tiles - rest;
    s.num_work = tiles + rest;
  }
  return s;
}
__device__ __forceinline__ LceWork lce_work(const LceSchedule& s, int w) {
  LceWork r;
  int tile = w, half = 0;
  r.width = 256;
  r.split = 0;
  if (s.splits > 1) {                  // the tiles of one part of K after the other
    const int tiles = s.num_pid_m * s.num_pid_n;
    r.split = w / tiles;
    tile = w - r.split * tiles;
  } else if (w >= s.full_work) {
    tile = s.full_work + ((w - s.full_work) >> 1);
    half = (w - s.full_work) & 1;
    r.width = 128;
  }
  const int per_group = s.group_m * s.num_pid_n;
  const int group = tile / per_group;
  const int first = group * s.group_m;
  const int size = min(s.num_pid_m - first, s.group_m);
  const int in = tile - group * per_group;
  r.pid_m = first + in % size;
  r.pid_n = in / size;
  if (group & 1) r.pid_n = s.num_pid_n - 1 - r.pid_n;
  r.col0 = r.pid_n * 256 + half * 128;
  return r;
}

__device__ __forceinline__ uint32_t lce_pack2(float lo, float hi, int f16) { return f16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi); }

// 64 columns of a warp's 32 rows, packed to 16 bits, through the warp's BUFS staging buffers in turn to the tensor map.
template <int BUFS>
__device__ __forceinline__ void lce_store_chunk(const CUtensorMap* map, const float (&f)[64], int f16, int row0, int col0, int rows, int cols,
                                                uint8_t* stage, int& buf, uint32_t lane) {
  if (lane == 0) tma_store_wait_read<BUFS - 1>();   // the buffer's store of BUFS chunks ago
  __syncwarp();
  uint8_t* dst = stage + buf * LCE_C_BUF_BYTES;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint4 v = make_uint4(lce_pack2(f[8 * j], f[8 * j + 1], f16), lce_pack2(f[8 * j + 2], f[8 * j + 3], f16),
                               lce_pack2(f[8 * j + 4], f[8 * j + 5], f16), lce_pack2(f[8 * j + 6], f[8 * j + 7], f16));
    *reinterpret_cast<uint4*>(dst + lane * 128 + ((j ^ (lane & 7)) << 4)) = v;
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    if (row0 < rows && col0 < cols) tma_store_2d(map, dst, col0, row0);
    tma_store_commit();
  }
  if (BUFS == 2) buf ^= 1;
}

// 64 columns of a row of logits into its running maximum (in units of log2) and sum of 2^(x - maximum); `in`: the target's place among them, `limit`:
// the first column that does not count.
__device__ __forceinline__ void lce_stats_chunk(float (&f)[64], int in, int col0, int limit, float* target_logit, float& run_max, float& run_sum) {
  if (in >= 0 && in < 64 && col0 + in < limit) {
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < 64; ++j) t = j == in ? f[j] : t;
    *target_logit = t;
  }
  if (col0 + 64 > limit) {
#pragma unroll
    for (int j = 0; j < 64; ++j) f[j] = col0 + j < limit ? f[j] : -INFINITY;
  }
  float m = f[0];
#pragma unroll
  for (int j = 1; j < 63; j += 2) m = fmax3(m, f[j], f[j + 1]);
  m = fmaxf(m, f[63]);
  const float new_max = fmaxf(run_max, m * LOG2E);
  const float shift = new_max == -INFINITY ? 0.f : new_max;     // a row of -inf: the sum stays 0
  float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
  for (int j = 0; j < 64; j += 4) {
    s0 += ex2_approx(fmaf(f[j], LOG2E, -shift));
    s1 += ex2_approx(fmaf(f[j + 1], LOG2E, -shift));
    s2 += ex2_approx(fmaf(f[j + 2], LOG2E, -shift));
    s3 += ex2_approx(fmaf(f[j + 3], LOG2E, -shift));
  }
  run_sum = fmaf(run_sum, ex2_approx(run_max - shift), (s0 + s1) + (s2 + s3));
  run_max = new_max;
}

// Adds 128 columns of the part of a row's sums that lies in tensor memory (16 at a time: 32 more registers would be spilled next to the sums).
__device__ __forceinline__ void lce_add_segment(uint32_t taddr, float (&f)[2][64]) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint32_t v[16];
    tmem_ld_x16(taddr + c * 16, v);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j) f[c / 4][(c & 3) * 16 + j] += __uint_as_float(v[j]);
  }
}

// A target as the kernels compare it with columns: outside the vocabulary, or ignored, it matches none.
constexpr int LCE_NO_TARGET = -(1 << 29);
__device__ __forceinline__ int lce_target(int64_t y, int V) { return y >= 0 && y < V ? static_cast<int>(y) : LCE_NO_TARGET; }

// A_MN / B_MN: the operand's tile is contiguous along M / N in memory (else along K).
template <int EPI, bool A_MN, bool B_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(lce_threads(EPI), 1)
lce_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                const __grid_constant__ CUtensorMap tmap_c, const LceGemmParams p) {
  constexpr bool LOGITS = lce_logits(EPI);
  constexpr int EPI_WARPS = lce_epi_warps(EPI), BUFS = 8 / EPI_WARPS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_a = smem + LCE_A_OFF;
  uint8_t* smem_b = smem + LCE_B_OFF;
  uint8_t* smem_c = smem + LCE_C_OFF;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + LCE_BAR_OFF);   // used in the leader only
  uint64_t* empty_bar = full_bar + LCE_STAGES;                            // one set per CTA
  uint64_t* tmem_full_bar = empty_bar + LCE_STAGES;                       // one set per CTA
  uint64_t* tmem_empty_bar = tmem_full_bar + 2;                           // used in the leader only
  uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(tmem_empty_bar + 2);
  uint32_t* abort_smem = tmem_ptr_smem + 1;

  const int warp_idx = threadIdx.x >> 5;
  const uint32_t lane = lane_id();
  const uint32_t rank = cluster_ctarank();   // 0 = pair leader
  const int pair = blockIdx.x >> 1;
  const int num_pairs = gridDim.x >> 1;
  WaitCtx ctx{abort_smem, p.status};

  if (threadIdx.x == 0) {
    for (int s = 0; s < LCE_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full_bar[a], 1);
      mbar_init(&tmem_empty_bar[a], 2 * EPI_WARPS);
    }
    *abort_smem = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_b);
    if (EPI == LCE_DLOGITS || EPI == LCE_DW) prefetch_tmap(&tmap_c);
  }
  if (warp_idx == 1) {
    tmem_alloc_2cta(tmem_ptr_smem, 512);
    tmem_relinquish_2cta();
  }
  tc_fence_before();
  __syncthreads();
  cluster_arrive();   // both CTAs' barriers must exist before either CTA signals the other
  cluster_wait();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr_smem;
  grid_launch_dependents();
  grid_wait();

  const int count = p.count != nullptr ? *p.count : p.M;
  const int M = EPI == LCE_DW ? p.M : count;
  const int num_kb = ((EPI == LCE_DW ? count : p.K) + 63) >> 6;
  const int splits = EPI == LCE_DH ? lce_splits(((M + 255) >> 8) * ((p.N + 255) >> 8), num_pairs, num_kb, p.max_splits) : 1;
  const LceSchedule sched = lce_schedule(M, p.N, p.group_m, num_pairs, splits);
  // the steps along K of a work item
  auto kb_begin = [&](const LceWork& wk) { return EPI == LCE_DH ? static_cast<int>(static_cast<int64_t>(num_kb) * wk.split / splits) : 0; };
  auto kb_end = [&](const LceWork& wk) { return EPI == LCE_DH ? static_cast<int>(static_cast<int64_t>(num_kb) * (wk.split + 1) / splits) : num_kb; };

  if (warp_idx == 0) {
    // ---------------------------------------------------------------- TMA producer (both CTAs)
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    const uint64_t pol_a = l2_policy_evict_last();     // a group's A panel is read again by every tile column
    const uint64_t pol_b = l2_policy_evict_normal();
    for (int work = pair; ok && work < sched.num_work; work += num_pairs) {
      const LceWork wk = lce_work(sched, work);
      const int m0 = wk.pid_m * 256 + static_cast<int>(rank) * 128;
      const int n0 = wk.col0 + static_cast<int>(rank) * (wk.width / 2);
      const int b_boxes = wk.width / 128;
      const int kb1 = kb_end(wk);
      for (int kb = kb_begin(wk); kb < kb1; ++kb) {
        ok = mbar_wait(&empty_bar[stage], phase ^ 1u, ctx, 61);
        if (!ok) break;
        if (lane == 0) {
          const uint32_t leader_full = mapa_shared(smem_u32(&full_bar[stage]), 0);
          if (rank == 0) mbar_expect_tx(&full_bar[stage], 2 * (LCE_A_BYTES + b_boxes * LCE_BOX_BYTES));
          uint8_t* da = smem_a + stage * LCE_A_BYTES;
          uint8_t* db = smem_b + stage * LCE_B_BYTES;
#pragma unroll
          for (int i = 0; i < 2; ++i)
            tma_load_2d_2cta_hint(da + i * LCE_BOX_BYTES, &tmap_a, leader_full, A_MN ? m0 + i * 64 : kb * 64, A_MN ? kb * 64 : m0 + i * 64, pol_a);
          for (int i = 0; i < b_boxes; ++i)
            tma_load_2d_2cta_hint(db + i * LCE_BOX_BYTES, &tmap_b, leader_full, B_MN ? n0 + i * 64 : kb * 64, B_MN ? kb * 64 : n0 + i * 64, pol_b);
        }
        __syncwarp();
        if (++stage == LCE_STAGES) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp_idx == 1) {
    // ---------------------------------------------------------------- MMA issuer (leader only)
    if (rank == 0 && num_kb > 0) {
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;
      bool ok = true;
      for (int work = pair; ok && work < sched.num_work; work += num_pairs) {
        const uint32_t idesc = work >= sched.full_work ? p.idesc_half : p.idesc;
        int kb0 = 0, kb1 = num_kb;
        if (EPI == LCE_DH) {
          const LceWork wk = lce_work(sched, work);
          kb0 = kb_begin(wk);
          kb1 = kb_end(wk);
        }
        // a part of K (LOGITS: of LCE_SEGMENT steps) per accumulator
        for (int first = kb0; ok && first < kb1; ++it) {
          const int next = LOGITS ? min(first + LCE_SEGMENT, kb1) : kb1;
          const int acc = it & 1;
          ok = mbar_wait(&tmem_empty_bar[acc], ((it >> 1) & 1) ^ 1u, ctx, 62);
          if (!ok) break;
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + acc * 256;
          for (int kb = first; kb < next; ++kb) {
            ok = mbar_wait(&full_bar[stage], phase, ctx, 63);
            if (!ok) break;
            tc_fence_after();
            if (lane == 0) {
              const uint32_t a_addr = smem_u32(smem_a + stage * LCE_A_BYTES);
              const uint32_t b_addr = smem_u32(smem_b + stage * LCE_B_BYTES);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                // K-major: a k step is 32 bytes along the 128-byte rows; M/N-major: 16 rows down, 64-wide chunks one box apart
                const uint64_t a_desc = umma_smem_desc_sw128(a_addr + k * (A_MN ? 2048 : 32), A_MN ? LCE_BOX_BYTES : 16, 1024);
                const uint64_t b_desc = umma_smem_desc_sw128(b_addr + k * (B_MN ? 2048 : 32), B_MN ? LCE_BOX_BYTES : 16, 1024);
                umma_ss_2cta(d_tmem, a_desc, b_desc, idesc, (kb > first || k > 0) ? 1u : 0u);
              }
              const uint32_t e = smem_u32(&empty_bar[stage]);
              umma_commit_2cta(mapa_shared(e, 0));
              umma_commit_2cta(mapa_shared(e, 1));
              if (kb == next - 1) {
                const uint32_t f = smem_u32(&tmem_full_bar[acc]);
                umma_commit_2cta(mapa_shared(f, 0));
                umma_commit_2cta(mapa_shared(f, 1));
              }
            }
            __syncwarp();
            if (++stage == LCE_STAGES) { stage = 0; phase ^= 1u; }
          }
          first = next;
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue (warps 2.., both CTAs)
    const int q = warp_idx & 3;
    uint8_t* my_stage = smem_c + (warp_idx - 2) * BUFS * LCE_C_BUF_BYTES;
    int it = 0, buf = 0;
    bool ok = true;
    if constexpr (LOGITS) {
      const int side = (warp_idx - 2) >> 2;          // the warp's 128 columns of a tile
      for (int work = pair; ok && work < sched.num_work; work += num_pairs) {
        const LceWork wk = lce_work(sched, work);
        const int row0 = wk.pid_m * 256 + static_cast<int>(rank) * 128 + q * 32;
        const int row = row0 + static_cast<int>(lane);
        const int first_col = wk.col0 + side * 128;
        const bool live = row < M, mine = side * 128 < wk.width;
        // what the row needs, fetched while the main loop still runs
        int target = -1;
        float lse2 = 0.f, scale = 0.f;
        if (live) target = (EPI == LCE_STATS && p.token_target != nullptr ? lce_target(p.token_target[row], p.N) : p.target[row]) - p.col_base - first_col;
        if (EPI == LCE_DLOGITS && live) {
          lse2 = p.lse2[row];
          scale = p.row_scale[row];
        }
        float f[2][64];
#pragma unroll
        for (int j = 0; j < 64; ++j) f[0][j] = f[1][j] = 0.f;
        for (int first = 0; first < num_kb; first += LCE_SEGMENT, ++it) {
          const int acc = it & 1;
          ok = mbar_wait(&tmem_full_bar[acc], (it >> 1) & 1, ctx, 64);
          if (!ok) break;
          tc_fence_after();
          if (mine) lce_add_segment(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * 256 + side * 128, f);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(&tmem_empty_bar[acc]), 0));
        }
        if (!ok) break;
        if (!mine) continue;
        float run_max = -INFINITY, run_sum = 0.f;     // STATS: maximum in units of log2, sum of 2^(x - maximum)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col0 = first_col + c * 64;
          const int in = target - c * 64;              // the target's place in this chunk
          if constexpr (EPI == LCE_STATS) {
            lce_stats_chunk(f[c], in, col0, p.N, p.target_logit + row, run_max, run_sum);
          } else {
#pragma unroll
            for (int j = 0; j < 64; ++j) {
              const float e = ex2_approx(fmaf(f[c][j], LOG2E, -lse2)) - (j == in ? 1.f : 0.f);
              f[c][j] = live ? e * scale : 0.f;        // rows behind the last one that counts: zeros, for the K tail of dW
            }
            if (col0 + 64 > p.N) {                     // columns behind the piece: zeros, for the K tail of dh
#pragma unroll
              for (int j = 0; j < 64; ++j) f[c][j] = col0 + j < p.N ? f[c][j] : 0.f;
            }
            lce_store_chunk<BUFS>(&tmap_c, f[c], p.f16, row0, col0, p.M, p.N, my_stage, buf, lane);   // the map ends on a multiple of 8 columns
          }
        }
        if (EPI == LCE_STATS && live) p.part[static_cast<int64_t>(first_col >> 7) * p.part_ld + row] = make_float2(run_max, run_sum);
      }
    } else {
      const float alpha = *p.alpha;
      for (int work = pair; ok && work < sched.num_work; work += num_pairs, ++it) {
        const LceWork wk = lce_work(sched, work);
        const int row0 = wk.pid_m * 256 + static_cast<int>(rank) * 128 + q * 32;
        const int row = row0 + static_cast<int>(lane);
        const int chunks = wk.width / 64;
        const int acc = it & 1;
        const bool live = row < M;
        const uint32_t t_row = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * 256;
        const int token = EPI == LCE_DH && live ? p.token[row] : 0;      // fetched while the main loop still runs
        if (num_kb > 0) {
          ok = mbar_wait(&tmem_full_bar[acc], (it >> 1) & 1, ctx, 64);
          if (!ok) break;
          tc_fence_after();
        }
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          float f[64];
          if (num_kb > 0) {
            uint32_t v0[32], v1[32];
            tmem_ld_x32(t_row + c * 64, v0);
            tmem_ld_x32(t_row + c * 64 + 32, v1);
            tmem_wait_ld();
            if (c == chunks - 1) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(&tmem_empty_bar[acc]), 0));
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              f[j] = __uint_as_float(v0[j]);
              f[32 + j] = __uint_as_float(v1[j]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 64; ++j) f[j] = 0.f;
          }
          const int col0 = wk.col0 + c * 64;
          if constexpr (EPI == LCE_DW) {
#pragma unroll
            for (int j = 0; j < 64; ++j) f[j] *= alpha;
            lce_store_chunk<BUFS>(&tmap_c, f, p.f16, row0, col0, p.M, p.N, my_stage, buf, lane);
          } else {
            // K (= D) is a multiple of 8, so a row of the result ends on a multiple of 8 columns
            if (live) {
              const int cols = min(64, p.N - col0);
              const int64_t at = wk.split * p.split_stride + static_cast<int64_t>(row) * p.N + col0;
              if (p.add != nullptr) {
#pragma unroll
                for (int j = 0; j < 64; j += 4)
                  if (j < cols) {
                    const float4 a = *reinterpret_cast<const float4*>(p.add + at + j);
                    f[j] += a.x; f[j + 1] += a.y; f[j + 2] += a.z; f[j + 3] += a.w;
                  }
              }
              if (splits > 1 || !p.last) {
#pragma unroll
                for (int j = 0; j < 64; j += 4)
                  if (j < cols) *reinterpret_cast<float4*>(p.sum + at + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
              } else {
                uint16_t* out = static_cast<uint16_t*>(p.out) + static_cast<int64_t>(token) * p.N + col0;
#pragma unroll
                for (int j = 0; j < 64; j += 8)
                  if (j < cols)
                    *reinterpret_cast<uint4*>(out + j) =
                        make_uint4(lce_pack2(f[j] * alpha, f[j + 1] * alpha, p.f16), lce_pack2(f[j + 2] * alpha, f[j + 3] * alpha, p.f16),
                                   lce_pack2(f[j + 4] * alpha, f[j + 5] * alpha, p.f16), lce_pack2(f[j + 6] * alpha, f[j + 7] * alpha, p.f16));
              }
            }
          }
        }
      }
    }
    if (lane == 0) tma_store_wait_all<0>();
    __syncwarp();
  }

  // ------------------------------------------------------------------ teardown
  drain_after_abort(abort_smem);
  tc_fence_before();
  __syncthreads();
  cluster_arrive();   // neither CTA may exit while its partner can still signal its barriers
  cluster_wait();
  if (warp_idx == 1) {
    tc_fence_after();
    tmem_dealloc_2cta(tmem_base, 512);
  }
}

// ---------------------------------------------------------------------------------------------
// The statistics of at most 128 tokens: single CTAs (M = 128), one wave or more of tiles of `width` columns, chosen so that every SM gets the same
// number (lce_narrow_width).  The bound is the stream of W, which the pairs' 256-column tiles would spread unevenly over the SMs (61 tokens, 32000
// entries: 125 tiles on 74 pairs, 24 us).  The tokens are read where they are: with one tile row nothing is gained by leaving some out.
// ---------------------------------------------------------------------------------------------
constexpr int LCE1_STAGES = 4;
constexpr int LCE1_A_BYTES = 128 * 128, LCE1_B_BYTES = 256 * 128;
constexpr int LCE1_BAR_OFF = LCE1_STAGES * (LCE1_A_BYTES + LCE1_B_BYTES);
constexpr int LCE1_SMEM = LCE1_BAR_OFF + (2 * LCE1_STAGES + 4) * 8 + 16 + 1024;
static_assert(LCE1_SMEM <= 232448, "shared memory budget exceeded");

static int lce_narrow_width(int V, int sms) {
  const int64_t waves = (V + 256ll * sms - 1) / (256ll * sms);
  const int64_t width = (V + waves * sms - 1) / (waves * sms);
  return static_cast<int>((width + 15) / 16 * 16);
}

__global__ void __launch_bounds__(lce_threads(LCE_STATS), 1)
lce_stats_narrow_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const LceGemmParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem + LCE1_STAGES * LCE1_A_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + LCE1_BAR_OFF);
  uint64_t* empty_bar = full_bar + LCE1_STAGES;
  uint64_t* tmem_full_bar = empty_bar + LCE1_STAGES;
  uint64_t* tmem_empty_bar = tmem_full_bar + 2;
  uint32_t* tmem_ptr_smem = reinterpret_cast<uint32_t*>(tmem_empty_bar + 2);
  uint32_t* abort_smem = tmem_ptr_smem + 1;
  // What the warps of a tile's second 128 columns hand to those of the first, in three buffers in turn: the writers are two tiles ahead of a reader at
  // most, since a tile's accumulator is that of the tile two before it, which the readers empty after they have joined the one before that.
  __shared__ float2 second[3][128];
  __shared__ uint64_t second_bar[3];
  const int warp_idx = threadIdx.x >> 5;
  const uint32_t lane = lane_id();
  WaitCtx ctx{abort_smem, p.status};
  if (threadIdx.x == 0) {
    for (int i = 0; i < 3; ++i) mbar_init(&second_bar[i], lce_epi_warps(LCE_STATS) / 2);
    for (int s = 0; s < LCE1_STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full_bar[a], 1);
      mbar_init(&tmem_empty_bar[a], lce_epi_warps(LCE_STATS));
    }
    *abort_smem = 0;
    fence_mbar_init();
    prefetch_tmap(&tmap_a);
    prefetch_tmap(&tmap_b);
  }
  if (warp_idx == 1) {
    tmem_alloc(tmem_ptr_smem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr_smem;
  grid_launch_dependents();
  const int num_kb = (p.K + 63) >> 6;
  const int tiles = (p.N + p.width - 1) / p.width;

  if (warp_idx == 0) {
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x)
      for (int kb = 0; kb < num_kb; ++kb) {
        ok = mbar_wait(&empty_bar[stage], phase ^ 1u, ctx, 65);
        if (!ok) break;
        if (lane == 0) {
          mbar_expect_tx(&full_bar[stage], LCE1_A_BYTES + p.width * 128);
          tma_load_2d(smem_a + stage * LCE1_A_BYTES, &tmap_a, &full_bar[stage], kb * 64, 0);
          tma_load_2d(smem_b + stage * LCE1_B_BYTES, &tmap_b, &full_bar[stage], kb * 64, tile * p.width);
        }
        __syncwarp();
        if (++stage == LCE1_STAGES) { stage = 0; phase ^= 1u; }
      }
  } else if (warp_idx == 1) {
    int stage = 0, it = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
      for (int first = 0; ok && first < num_kb; first += LCE_SEGMENT, ++it) {
        const int next = min(first + LCE_SEGMENT, num_kb);
        const int acc = it & 1;
        ok = mbar_wait(&tmem_empty_bar[acc], ((it >> 1) & 1) ^ 1u, ctx, 66);
        if (!ok) break;
        tc_fence_after();
        for (int kb = first; kb < next; ++kb) {
          ok = mbar_wait(&full_bar[stage], phase, ctx, 67);
          if (!ok) break;
          tc_fence_after();
          if (lane == 0) {
            const uint32_t a_addr = smem_u32(smem_a + stage * LCE1_A_BYTES), b_addr = smem_u32(smem_b + stage * LCE1_B_BYTES);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_ss(tmem_base + acc * 256, umma_smem_desc_sw128(a_addr + k * 32, 16, 1024), umma_smem_desc_sw128(b_addr + k * 32, 16, 1024), p.idesc,
                      (kb > first || k > 0) ? 1u : 0u);
            umma_commit(&empty_bar[stage]);
            if (kb == next - 1) umma_commit(&tmem_full_bar[acc]);
          }
          __syncwarp();
          if (++stage == LCE1_STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else {
    const int q = warp_idx & 3;
    const int row = q * 32 + static_cast<int>(lane);
    const bool live = row < p.M;
    const int target = live ? lce_target(p.token_target[row], p.N) : LCE_NO_TARGET;
    const int side = (warp_idx - 2) >> 2;          // the warp's 128 columns of a tile
    int it = 0, buf = 0;
    uint32_t buf_phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
      const int first_col = tile * p.width + side * 128, limit = min(p.N, (tile + 1) * p.width);
      float f[2][64];
#pragma unroll
      for (int j = 0; j < 64; ++j) f[0][j] = f[1][j] = 0.f;
      for (int first = 0; first < num_kb; first += LCE_SEGMENT, ++it) {
        const int acc = it & 1;
        ok = mbar_wait(&tmem_full_bar[acc], (it >> 1) & 1, ctx, 68);
        if (!ok) break;
        tc_fence_after();
        lce_add_segment(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * 256 + side * 128, f);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tmem_empty_bar[acc]);
      }
      if (!ok) break;
      float run_max = -INFINITY, run_sum = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col0 = first_col + c * 64;
        if (col0 < limit) lce_stats_chunk(f[c], target - col0, col0, limit, p.target_logit + row, run_max, run_sum);
      }
      if (side == 1) {
        second[buf][row] = make_float2(run_max, run_sum);
        __syncwarp();
        if (lane == 0) mbar_arrive(&second_bar[buf]);
      } else {
        ok = mbar_wait(&second_bar[buf], buf_phase, ctx, 69);
        if (!ok) break;
        const float2 o = second[buf][row];
        const float top = fmaxf(run_max, o.x), shift = top == -INFINITY ? 0.f : top;
        run_sum = fmaf(run_sum, ex2_approx(run_max - shift), o.y * ex2_approx(o.x - shift));
        if (live) p.part[static_cast<int64_t>(tile) * p.part_ld + row] = make_float2(top, run_sum);
      }
      if (++buf == 3) { buf = 0; buf_phase ^= 1u; }
    }
  }
  drain_after_abort(abort_smem);
  tc_fence_before();
  __syncthreads();
  if (warp_idx == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// ---------------------------------------------------------------------------------------------
// Gather: the rows that count move to the front of `hc`, in order; the other rows of `hc` become zeros.
// ---------------------------------------------------------------------------------------------
constexpr int LCE_GATHER_ROWS = 8;      // a warp per row

struct LceGatherParams {
  const uint4* h;
  int64_t ldh8;            // row pitch of h in 16-byte units
  const int64_t* target;
  int64_t ignore;
  int T, D8, V;            // D8: 16-byte units of a row
  int cta_rows;            // rows of a CTA, a multiple of LCE_GATHER_ROWS
  uint4* hc;
  int* count;
  int* token;
  int* row_target;
  // forward
  float* losses;
  float* lse;
  // backward
  const float* lse_in;
  const float* d_loss;     // per token when gmax is not null, else one number
  const float* gmax;
  float* row_lse2;
  float* row_scale;
  uint4* dh;
  float* alpha;
  float unit;              // 1 or LCE_F16_SCALE
  int mean;
};

template <bool BACKWARD>
__global__ void __launch_bounds__(256) lce_gather_kernel(const LceGatherParams p) {
  grid_launch_dependents();
  grid_wait();
  __shared__ int warp_counts[8];
  __shared__ int place[LCE_GATHER_ROWS];       // row of hc; that of a row that does not count as -1 - row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = blockIdx.x * p.cta_rows, end = min(p.T, first + p.cta_rows);
  // tokens that count before this CTA's rows
  int n = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < first; i += 256) n += p.target[i] != p.ignore ? 1 : 0;
  n = __reduce_add_sync(0xFFFFFFFFu, n);
  if (lane == 0) warp_counts[warp] = n;
  __syncthreads();
  int before = 0;
  if (warp == 0) before = __reduce_add_sync(0xFFFFFFFFu, lane < 8 ? warp_counts[lane] : 0);
  for (int top = first; top < end; top += LCE_GATHER_ROWS) {
    if (warp == 0) {
      const int t = top + lane;
      const bool mine = lane < LCE_GATHER_ROWS && t < end;
      const int64_t y = mine ? p.target[t] : p.ignore;
      const bool counts = y != p.ignore;
      const unsigned mask = __ballot_sync(0xFFFFFFFFu, counts);
      const int at = before + __popc(mask & ((1u << lane) - 1u));   // rows that count before this one
      if (mine) {
        const int row = counts ? at : p.T - 1 - (t - at);           // the k-th row that does not count takes the k-th place from the back
        place[lane] = counts ? row : -1 - row;
        const int column = lce_target(y, p.V);
        const bool valid = column != LCE_NO_TARGET;
        p.row_target[row] = counts ? column : LCE_NO_TARGET;
        p.token[row] = t;
        if (BACKWARD) {
          p.row_lse2[row] = counts ? p.lse_in[t] * LOG2E : 0.f;
          float g = 1.f;
          if (p.gmax != nullptr) {
            const float m = *p.gmax;
            g = m > 0.f ? p.d_loss[t] / m : p.d_loss[t];
          }
          // a target outside the vocabulary: NaN, in the loss and in every gradient that it enters
          p.row_scale[row] = counts ? (valid ? g * p.unit : __int_as_float(0x7FC00000)) : 0.f;
        } else if (!counts) {
          p.losses[t] = 0.f;
          p.lse[t] = 0.f;
        }
      }
      before += __popc(mask);
    }
    __syncthreads();
    if (top + warp < end) {
      const int code = place[warp];
      const bool counts = code >= 0;
      uint4* dst = p.hc + static_cast<int64_t>(counts ? code : -1 - code) * p.D8;
      uint4* zeros = BACKWARD && !counts && p.dh != nullptr ? p.dh + static_cast<int64_t>(top + warp) * p.D8 : nullptr;
      const uint4* src = p.h + static_cast<int64_t>(top + warp) * p.ldh8;
      for (int i = lane; i < p.D8; i += 32 * 8) {
        uint4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = counts && i + 32 * k < p.D8 ? src[i + 32 * k] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (i + 32 * k < p.D8) {
            dst[i + 32 * k] = v[k];
            if (zeros != nullptr) zeros[i + 32 * k] = v[k];
          }
      }
    }
    __syncthreads();
  }
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) {
    *p.count = before;
    if (BACKWARD) {
      float a = p.gmax != nullptr ? (*p.gmax > 0.f ? *p.gmax : 1.f) : *p.d_loss;
      if (p.mean) a /= static_cast<float>(before > 0 ? before : 1);
      *p.alpha = a / p.unit;
    }
  }
}

// Largest magnitude of the tokens' gradients, of those that count and are finite.
__global__ void __launch_bounds__(1024) lce_gmax_kernel(const float* __restrict__ g, const int64_t* __restrict__ target, int64_t ignore, int T,
                                                        float* __restrict__ gmax) {
  __shared__ float warps[32];
  grid_launch_dependents();
  float m = 0.f;
  for (int i = threadIdx.x; i < T; i += 1024) {
    const float a = fabsf(g[i]);
    if (target[i] != ignore && a <= 3.4028234663852886e38f) m = fmaxf(m, a);
  }
  m = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(m)));
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x < 32) {
    m = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(warps[threadIdx.x])));
    if (threadIdx.x == 0) *gmax = m;
  }
}

// Joins the tiles' (maximum, sum) of 32 rows: 32 slices of the slots, one row per lane.  Without a gather (token == null) row and token are the same.
__global__ void __launch_bounds__(1024) lce_join_kernel(const float2* __restrict__ part, int64_t part_ld, int slots, const int* __restrict__ count, int T,
                                                        const float* __restrict__ target_logit, const int* __restrict__ token,
                                                        const int64_t* __restrict__ target, int64_t ignore, int V,
                                                        float* __restrict__ losses, float* __restrict__ lse) {
  __shared__ float2 joined[32][33];
  grid_launch_dependents();
  grid_wait();
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + lane;
  const bool live = row < (token != nullptr ? *count : T);
  float m = -INFINITY, s = 0.f;
  if (live) {
    for (int i = slice; i < slots; i += 4 * 32) {           // four slots at a time: their loads and exponentials do not wait for one another
      float2 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = i + 32 * k < slots ? part[static_cast<int64_t>(i + 32 * k) * part_ld + row] : make_float2(-INFINITY, 0.f);
      const float top = fmaxf(m, fmaxf(fmaxf(v[0].x, v[1].x), fmaxf(v[2].x, v[3].x)));
      const float shift = top == -INFINITY ? 0.f : top;
      s *= ex2_approx(m - shift);
#pragma unroll
      for (int k = 0; k < 4; ++k) s += v[k].y * ex2_approx(v[k].x - shift);
      m = top;
    }
  }
  joined[slice][lane] = make_float2(m, s);
  __syncthreads();
  // warp i joins the slices of row i
  const float2 v = joined[lane][slice];
  float top = v.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  float sum = v.y * ex2_approx(v.x - (top == -INFINITY ? 0.f : top));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  const int mine = blockIdx.x * 32 + slice;
  if (lane == 0 && mine < (token != nullptr ? *count : T)) {
    const int t = token != nullptr ? token[mine] : mine;
    const float lse2 = top + log2f(sum);
    const int64_t y = target[t];
    const bool counts = y != ignore, valid = y >= 0 && y < V;
    lse[t] = counts ? lse2 * LN2 : 0.f;
    losses[t] = !counts ? 0.f : valid ? fmaf(-target_logit[mine], LOG2E, lse2) * LN2 : __int_as_float(0x7FC00000);
  }
}

// Sum or mean of the losses, in an order that depends on T only.
__global__ void __launch_bounds__(1024) lce_reduce_kernel(const float* __restrict__ losses, const int64_t* __restrict__ target, int64_t ignore, int T,
                                                          int mean, float* __restrict__ loss) {
  __shared__ double warps[32];
  __shared__ int counts[32];
  grid_wait();
  double s = 0.0;
  int n = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < T; i += 1024) {
    s += static_cast<double>(losses[i]);
    n += target[i] != ignore ? 1 : 0;
  }
  n = __reduce_add_sync(0xFFFFFFFFu, n);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  if ((threadIdx.x & 31) == 0) {
    warps[threadIdx.x >> 5] = s;
    counts[threadIdx.x >> 5] = n;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warps[threadIdx.x];
    n = __reduce_add_sync(0xFFFFFFFFu, counts[threadIdx.x]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (threadIdx.x == 0) *loss = static_cast<float>(mean ? s / (n > 0 ? n : 1) : s);
  }
}

// dh from the fp32 sums of the parts of K, where the product was cut in several (a CTA per row that counts).
__global__ void __launch_bounds__(256) lce_dh_kernel(const LceGemmParams p, int pairs) {
  grid_launch_dependents();
  grid_wait();
  const int count = *p.count;
  const int row = blockIdx.x;
  if (row >= count) return;
  const int splits = lce_splits(((count + 255) >> 8) * ((p.N + 255) >> 8), pairs, (p.K + 63) >> 6, p.max_splits);
  if (splits == 1) return;
  const float alpha = *p.alpha;
  uint16_t* out = static_cast<uint16_t*>(p.out) + static_cast<int64_t>(p.token[row]) * p.N;
  for (int c = threadIdx.x * 4; c < p.N; c += 1024) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < splits; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(p.sum + k * p.split_stride + static_cast<int64_t>(row) * p.N + c);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    *reinterpret_cast<uint2*>(out + c) = make_uint2(lce_pack2(s.x * alpha, s.y * alpha, p.f16), lce_pack2(s.z * alpha, s.w * alpha, p.f16));
  }
}

// ---------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------
// Slots of the forward's workspace with few tokens: tiles of lce_narrow_width, at most one per SM and wave, and a wave is 256 columns per SM or all there is.
constexpr int LCE_NARROW_SLOTS = 512;
// Tokens up to which the forward reads h where it is (one tile row: leaving tokens out would save nothing), and up to which it runs on single CTAs.
constexpr int LCE_DIRECT_TOKENS = 256, LCE_NARROW_TOKENS = 128;

// Bytes of dlogits that a piece of the vocabulary may take.
constexpr int64_t LCE_PIECE_BYTES = int64_t(512) << 20;

static int lce_piece(int T, int V) {
  const int64_t most = LCE_PIECE_BYTES / (2 * static_cast<int64_t>(T)) / 256 * 256;
  const int64_t piece = most < 256 ? 256 : most;
  if (piece >= V) return V;
  const int64_t pieces = (V + piece - 1) / piece;
  return static_cast<int>(((V + pieces - 1) / pieces + 255) / 256 * 256);     // pieces of about one size
}

struct LceLayout {
  int64_t hc, token, row_target, count, alpha, gmax, a, b, part, dl, sum, total;   // byte offsets
  int slots, piece, pieces, max_splits;
  int64_t ld_dl;
};
static LceLayout lce_layout(int T, int D, int V, bool backward) {
  LceLayout l{};
  int64_t at = 0;
  auto take = [&at](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  l.count = take(4);
  l.alpha = take(4);
  l.gmax = take(4);
  l.token = take(4ll * T);
  l.row_target = take(4ll * T);
  l.a = take(4ll * T);           // forward: target logits; backward: lse * log2 e
  l.hc = take(2ll * T * D);
  if (!backward) {
    l.slots = 2 * ((V + 255) / 256);       // two per tile of 256; tiles of single CTAs are never narrower than 16 and no more than four per SM
    if (T <= LCE_NARROW_TOKENS && l.slots < LCE_NARROW_SLOTS) l.slots = LCE_NARROW_SLOTS;
    l.part = take(8ll * T * l.slots);
  } else {
    l.b = take(4ll * T);         // row factors
    l.piece = lce_piece(T, V);
    l.pieces = (V + l.piece - 1) / l.piece;
    l.ld_dl = (l.piece + 7) / 8 * 8;
    l.dl = take(2ll * T * l.ld_dl);
    // as many parts as could fill the pairs eight times over
    const int64_t tiles = static_cast<int64_t>((T + 255) / 256) * ((D + 255) / 256);
    const int64_t splits = 8 * 74 / tiles;
    // (several pieces carry one sum from piece to piece, and dW is never cut: with few tiles of dh or dW, as for a small D, some pairs then idle)
    l.max_splits = static_cast<int>(l.pieces > 1 || splits < 1 ? 1 : splits > LCE_MAX_SPLITS ? LCE_MAX_SPLITS : splits);
    if (l.pieces > 1 || l.max_splits > 1) l.sum = take(4ll * T * D * l.max_splits);
  }
  l.total = at;
  return l;
}

int64_t lce_workspace(int T, int D, int V, int backward) { return lce_layout(T, D, V, backward != 0).total; }

static int lce_check(const LceArgs& a, const char* what) {
  if (a.T < 0 || a.D < 8 || a.V < 1 || (a.D & 7)) return set_error(B200K_ERR_INVALID_ARG, "%s: T >= 0, V >= 1 and D a positive multiple of 8 expected (got %d, %d, %d)", what, a.T, a.V, a.D);
  if (a.V > (1 << 30) || a.T > (1 << 30) || a.D > (1 << 30)) return set_error(B200K_ERR_INVALID_ARG, "%s: at most 2^30 tokens, vocabulary entries and columns", what);
  if (a.dtype != B200K_DTYPE_BF16 && a.dtype != B200K_DTYPE_F16) return set_error(B200K_ERR_INVALID_ARG, "%s: bf16 or fp16 operands expected (got type %d)", what, a.dtype);
  if (a.reduction < B200K_REDUCE_NONE || a.reduction > B200K_REDUCE_SUM) return set_error(B200K_ERR_INVALID_ARG, "%s: bad reduction %d", what, a.reduction);
  if (static_cast<int64_t>((a.T + 255) / 256) * ((a.V + 255) / 256) > 0x3FFFFFFF || static_cast<int64_t>((a.V + 255) / 256) * ((a.D + 255) / 256) > 0x3FFFFFFF)
    return set_error(B200K_ERR_INVALID_ARG, "%s: too many tiles", what);
  if (a.T > 0) {
    if (a.h == nullptr || a.w == nullptr || a.target == nullptr) return set_error(B200K_ERR_INVALID_ARG, "%s: null pointer", what);
    if (a.ldh < a.D || a.ldw < a.D || (a.ldh & 7) || (a.ldw & 7))
      return set_error(B200K_ERR_INVALID_ARG, "%s: row pitches must be multiples of 8 elements and at least D (got %lld, %lld)", what, (long long)a.ldh, (long long)a.ldw);
    if ((reinterpret_cast<uintptr_t>(a.h) | reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.dh) | reinterpret_cast<uintptr_t>(a.dw)) & 15u)
      return set_error(B200K_ERR_INVALID_ARG, "%s: h, w and their gradients must be 16-byte aligned", what);
    if (reinterpret_cast<uintptr_t>(a.workspace) & 255u) return set_error(B200K_ERR_INVALID_ARG, "%s: the workspace must be 256-byte aligned", what);
  }
  return B200K_OK;
}

static int lce_check_workspace(const LceArgs& a, const LceLayout& l, const char* what) {
  if (a.workspace == nullptr || a.workspace_bytes < l.total)
    return set_error(B200K_ERR_INVALID_ARG, "%s: a workspace of %lld bytes is needed (got %lld)", what, (long long)l.total, (long long)(a.workspace == nullptr ? 0 : a.workspace_bytes));
  return B200K_OK;
}

// Rows of a gathering CTA: about a thousand CTAs, each of which counts the tokens before its own.
static int lce_gather_rows(int T) { return (T / 1024 / LCE_GATHER_ROWS + 1) * LCE_GATHER_ROWS; }

// CTA pairs of a launch: enough for every tile's halves, or for the parts of K.
static int lce_pairs(const LceGemmParams& p, const DeviceInfo* dev) {
  const int64_t tiles = static_cast<int64_t>((p.M + 255) / 256) * ((p.N + 255) / 256) * (p.max_splits > 2 ? p.max_splits : 2);
  const int max_pairs = dev->sm_count / 2;
  return static_cast<int>(tiles < max_pairs ? tiles : max_pairs);
}

template <int EPI, bool A_MN, bool B_MN>
static int lce_gemm(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, LceGemmParams p, const DeviceInfo* dev, cudaStream_t stream) {
  p.group_m = 8;
  p.idesc = umma_idesc_16bit_f32(256, 256, A_MN, B_MN, p.f16);
  p.idesc_half = umma_idesc_16bit_f32(256, 128, A_MN, B_MN, p.f16);
  p.status = dev->status_word;
  B200K_CHECK_CUDA(cudaFuncSetAttribute(lce_gemm_kernel<EPI, A_MN, B_MN>, cudaFuncAttributeMaxDynamicSharedMemorySize, LCE_SMEM));
  const int pairs = lce_pairs(p, dev);
  // the forward's with few tokens is the first of its chain
  if (p.count == nullptr) {
    lce_gemm_kernel<EPI, A_MN, B_MN><<<2 * pairs, lce_threads(EPI), LCE_SMEM, stream>>>(ta, tb, tc, p);
  } else {
    B200K_CHECK_CUDA(launch_dependent(lce_gemm_kernel<EPI, A_MN, B_MN>, dim3(2 * pairs), dim3(lce_threads(EPI)), LCE_SMEM, stream, ta, tb, tc, p));
  }
  count_launch();
  B200K_CHECK_LAUNCH("lce_gemm_kernel");
  return B200K_OK;
}

static const DeviceInfo* lce_device(const char* what) {
  const DeviceInfo* dev = current_device_info();
  if (dev != nullptr && dev->cc_major != 10) {
    set_error(B200K_ERR_NO_DEVICE, "%s: needs an sm_100 device (found sm_%d%d)", what, dev->cc_major, dev->cc_minor);
    return nullptr;
  }
  return dev;
}

int lce_fwd(const LceArgs& a, cudaStream_t stream) {
  const char* what = "linear_cross_entropy";
  int rc = lce_check(a, what);
  if (rc != B200K_OK) return rc;
  if (a.reduction != B200K_REDUCE_NONE && a.loss == nullptr) return set_error(B200K_ERR_INVALID_ARG, "%s: null loss", what);
  if (a.T == 0) {
    if (lce_device(what) == nullptr) return B200K_ERR_NO_DEVICE;
    if (a.reduction != B200K_REDUCE_NONE) B200K_CHECK_CUDA(cudaMemsetAsync(a.loss, 0, sizeof(float), stream));
    return B200K_OK;
  }
  const LceLayout l = lce_layout(a.T, a.D, a.V, false);
  if (a.losses == nullptr || a.lse == nullptr) return set_error(B200K_ERR_INVALID_ARG, "%s: null losses or lse", what);
  if ((rc = lce_check_workspace(a, l, what)) != B200K_OK) return rc;
  const DeviceInfo* dev = lce_device(what);
  if (dev == nullptr) return B200K_ERR_NO_DEVICE;
  char* ws = static_cast<char*>(a.workspace);
  float* target_logit = reinterpret_cast<float*>(ws + l.a);
  const bool direct = a.T <= LCE_DIRECT_TOKENS;
  LceGemmParams p{};
  p.M = a.T; p.N = a.V; p.K = a.D;
  p.f16 = a.dtype == B200K_DTYPE_F16;
  p.part = reinterpret_cast<float2*>(ws + l.part);
  p.part_ld = a.T;
  p.target_logit = target_logit;
  const void* rows = a.h;
  int64_t ld_rows = a.ldh;
  if (direct) {
    p.token_target = a.target;
  } else {
    LceGatherParams g{};
    g.h = static_cast<const uint4*>(a.h);
    g.ldh8 = a.ldh / 8;
    g.target = a.target;
    g.ignore = a.ignore_index;
    g.T = a.T; g.D8 = a.D / 8; g.V = a.V;
    g.hc = reinterpret_cast<uint4*>(ws + l.hc);
    g.count = reinterpret_cast<int*>(ws + l.count);
    g.token = reinterpret_cast<int*>(ws + l.token);
    g.row_target = reinterpret_cast<int*>(ws + l.row_target);
    g.losses = a.losses;
    g.lse = a.lse;
    g.cta_rows = lce_gather_rows(a.T);
    lce_gather_kernel<false><<<(a.T + g.cta_rows - 1) / g.cta_rows, 256, 0, stream>>>(g);
    count_launch();
    B200K_CHECK_LAUNCH("lce_gather_kernel");
    p.count = g.count;
    p.target = g.row_target;
    p.token = g.token;
    rows = ws + l.hc;
    ld_rows = a.D;
  }
  int slots = 2 * ((a.V + 255) / 256);
  CUtensorMap th, tw;
  if (a.T <= LCE_NARROW_TOKENS) {
    p.width = lce_narrow_width(a.V, dev->sm_count);
    slots = (a.V + p.width - 1) / p.width;
    if (slots > l.slots) return set_error(B200K_ERR_INVALID_ARG, "%s: workspace slots", what);
    if ((rc = make_tmap_bf16_2d(&th, rows, a.D, a.T, ld_rows, 64, 128)) != 0) return rc;
    if ((rc = make_tmap_bf16_2d(&tw, a.w, a.D, a.V, a.ldw, 64, p.width)) != 0) return rc;
    p.idesc = umma_idesc_16bit_f32(128, p.width, 0, 0, p.f16);
    p.status = dev->status_word;
    B200K_CHECK_CUDA(cudaFuncSetAttribute(lce_stats_narrow_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LCE1_SMEM));
    lce_stats_narrow_kernel<<<slots < dev->sm_count ? slots : dev->sm_count, lce_threads(LCE_STATS), LCE1_SMEM, stream>>>(th, tw, p);
    count_launch();
    B200K_CHECK_LAUNCH("lce_stats_narrow_kernel");
  } else {
    if ((rc = make_tmap_bf16_2d(&th, rows, a.D, a.T, ld_rows, 64, 64)) != 0) return rc;
    if ((rc = make_tmap_bf16_2d(&tw, a.w, a.D, a.V, a.ldw, 64, 64)) != 0) return rc;
    if ((rc = lce_gemm<LCE_STATS, false, false>(th, tw, th, p, dev, stream)) != 0) return rc;
  }
  B200K_CHECK_CUDA(launch_dependent(lce_join_kernel, dim3((a.T + 31) / 32), dim3(1024), 0, stream, p.part, p.part_ld, slots, p.count, a.T, target_logit,
                                    p.token, a.target, a.ignore_index, a.V, a.losses, a.lse));
  count_launch();
  B200K_CHECK_LAUNCH("lce_join_kernel");
  if (a.reduction != B200K_REDUCE_NONE) {
    B200K_CHECK_CUDA(launch_dependent(lce_reduce_kernel, dim3(1), dim3(1024), 0, stream, a.losses, a.target, a.ignore_index, a.T,
                                      a.reduction == B200K_REDUCE_MEAN ? 1 : 0, a.loss));
    count_launch();
    B200K_CHECK_LAUNCH("lce_reduce_kernel");
  }
  return B200K_OK;
}

int lce_bwd(const LceArgs& a, cudaStream_t stream) {
  const char* what = "linear_cross_entropy_backward";
  int rc = lce_check(a, what);
  if (rc != B200K_OK) return rc;
  if (a.T == 0) {
    if (lce_device(what) == nullptr) return B200K_ERR_NO_DEVICE;
    if (a.dw != nullptr) B200K_CHECK_CUDA(cudaMemsetAsync(a.dw, 0, 2ll * a.V * a.D, stream));
    return B200K_OK;
  }
  if (a.lse == nullptr || a.d_loss == nullptr) return set_error(B200K_ERR_INVALID_ARG, "%s: null lse or d_loss", what);
  const LceLayout l = lce_layout(a.T, a.D, a.V, true);
  if ((rc = lce_check_workspace(a, l, what)) != B200K_OK) return rc;
  const DeviceInfo* dev = lce_device(what);
  if (dev == nullptr) return B200K_ERR_NO_DEVICE;
  if (a.dh == nullptr && a.dw == nullptr) return B200K_OK;
  char* ws = static_cast<char*>(a.workspace);
  float* gmax = reinterpret_cast<float*>(ws + l.gmax);
  const bool each = a.reduction == B200K_REDUCE_NONE;
  if (each) {
    lce_gmax_kernel<<<1, 1024, 0, stream>>>(a.d_loss, a.target, a.ignore_index, a.T, gmax);
    count_launch();
    B200K_CHECK_LAUNCH("lce_gmax_kernel");
  }
  LceGatherParams g{};
  g.h = static_cast<const uint4*>(a.h);
  g.ldh8 = a.ldh / 8;
  g.target = a.target;
  g.ignore = a.ignore_index;
  g.T = a.T; g.D8 = a.D / 8; g.V = a.V;
  g.hc = reinterpret_cast<uint4*>(ws + l.hc);
  g.count = reinterpret_cast<int*>(ws + l.count);
  g.token = reinterpret_cast<int*>(ws + l.token);
  g.row_target = reinterpret_cast<int*>(ws + l.row_target);
  g.lse_in = a.lse;
  g.d_loss = a.d_loss;
  g.gmax = each ? gmax : nullptr;
  g.row_lse2 = reinterpret_cast<float*>(ws + l.a);
  g.row_scale = reinterpret_cast<float*>(ws + l.b);
  g.dh = static_cast<uint4*>(a.dh);
  g.alpha = reinterpret_cast<float*>(ws + l.alpha);
  g.unit = a.dtype == B200K_DTYPE_F16 ? LCE_F16_SCALE : 1.f;
  g.mean = a.reduction == B200K_REDUCE_MEAN;
  g.cta_rows = lce_gather_rows(a.T);
  if (each) {
    B200K_CHECK_CUDA(launch_dependent(lce_gather_kernel<true>, dim3((a.T + g.cta_rows - 1) / g.cta_rows), dim3(256), 0, stream, g));
  } else {
    lce_gather_kernel<true><<<(a.T + g.cta_rows - 1) / g.cta_rows, 256, 0, stream>>>(g);
  }
  count_launch();
  B200K_CHECK_LAUNCH("lce_gather_kernel");

  CUtensorMap th;
  if ((rc = make_tmap_bf16_2d(&th, ws + l.hc, a.D, a.T, a.D, 64, 64)) != 0) return rc;
  float* sum = l.pieces > 1 || l.max_splits > 1 ? reinterpret_cast<float*>(ws + l.sum) : nullptr;
  for (int k = 0; k < l.pieces; ++k) {
    const int v0 = k * l.piece;
    const int n = a.V - v0 < l.piece ? a.V - v0 : l.piece;
    const int cols = (n + 7) / 8 * 8;     // dlogits of the piece, its last columns zeros
    CUtensorMap tw, tdl, tdl_store, tdw;
    const uint16_t* w = static_cast<const uint16_t*>(a.w) + static_cast<int64_t>(v0) * a.ldw;
    if ((rc = make_tmap_bf16_2d(&tw, w, a.D, n, a.ldw, 64, 64)) != 0) return rc;
    if ((rc = make_tmap_bf16_2d(&tdl, ws + l.dl, cols, a.T, l.ld_dl, 64, 64)) != 0) return rc;
    if ((rc = make_tmap_bf16_2d(&tdl_store, ws + l.dl, cols, a.T, l.ld_dl, 64, 32)) != 0) return rc;
    LceGemmParams p{};
    p.count = g.count;
    p.f16 = a.dtype == B200K_DTYPE_F16;
    p.alpha = g.alpha;
    p.M = a.T; p.N = n; p.K = a.D;
    p.target = g.row_target;
    p.col_base = v0;
    p.lse2 = g.row_lse2;
    p.row_scale = g.row_scale;
    if ((rc = lce_gemm<LCE_DLOGITS, false, false>(th, tw, tdl_store, p, dev, stream)) != 0) return rc;
    if (a.dw != nullptr) {
      uint16_t* dw = static_cast<uint16_t*>(a.dw) + static_cast<int64_t>(v0) * a.D;
      if ((rc = make_tmap_bf16_2d(&tdw, dw, a.D, n, a.D, 64, 32)) != 0) return rc;
      p.M = n; p.N = a.D; p.K = a.T;
      if ((rc = lce_gemm<LCE_DW, true, true>(tdl, th, tdw, p, dev, stream)) != 0) return rc;
    }
    if (a.dh != nullptr) {
      p.M = a.T; p.N = a.D; p.K = n;
      p.max_splits = l.max_splits;
      p.add = k > 0 ? sum : nullptr;
      p.sum = sum;
      p.split_stride = static_cast<int64_t>(a.T) * a.D;
      p.last = k + 1 == l.pieces;
      p.out = a.dh;
      p.token = g.token;
      if ((rc = lce_gemm<LCE_DH, false, true>(tdl, tw, tw, p, dev, stream)) != 0) return rc;
      if (p.max_splits > 1) {
        B200K_CHECK_CUDA(launch_dependent(lce_dh_kernel, dim3(a.T), dim3(256), 0, stream, p, lce_pairs(p, dev)));
        count_launch();
        B200K_CHECK_LAUNCH("lce_dh_kernel");
      }
    }
  }
  return B200K_OK;
}

}  // namespace b200k
