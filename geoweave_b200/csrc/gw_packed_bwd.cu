// Backward pass of the attention over packed sequences on the tcgen05 tensor cores, 16-bit operands, head dim up to 128.
//
//   P = 2^(c S - lse log2 e),  D = rowsum(d_o * o),  dP = d_o v^T,  dS = P * (dP - D)
//   dq = scale dS k,   dk = scale sum dS^T q,   dv = sum P^T d_o
//
// Two kernels, so that every sum is made by one block in a fixed order and nothing needs atomics (results do not depend on
// timing): one owns 128 query rows and walks the keys (dq, and D on the way), one owns 128 key rows and walks the queries of all
// heads that read them (dk, dv).  S and dP are made in both: seven products instead of five, against 32-bit atomic traffic of
// one query tile for every pair of tiles.
//
// Each pair of tiles: S and dP from shared-memory operands into tensor memory; groups of four warps, 64 columns each,
// make P and dS in registers (a thread owns a row of its 64 columns) and put them back into tensor memory as 16-bit A operands of
// the accumulating products, whose B operand is the tile that is in shared memory already, read along its rows.  The key-side
// kernel works on the transposes (rows are keys), so neither P nor dS is ever transposed.
//
// P and dS are rounded to the inputs' type, the only one that may stand beside the tile of the other operand, once each: with bf16 dq and dk
// are off by 0.0024 of their norm, of which the last rounding alone makes 0.0017.  All else (S, dP, D, lse, the sums) is fp32.
#include <type_traits>

#include "gw_packed_mma.cuh"

namespace gw {
namespace {

struct BwdShared {
  uint64_t own_full, s_full, dp_full, s_read, dp_read, p_full, ds_full, ds_done, all_done;
  uint64_t a_full[4], a_empty[4], b_full[4], b_empty[4], st_full[4];
  uint64_t top_full[4];  // fp16, wide heads: both warps of a row have left their exponents
  PackedSeq seq;
  int64_t tiles, end;
  int found;
  float part[2][kTile];  // the two halves' sums of d_o * o
  uint8_t top[2][2][kTile];  // [tile & 1][half][row]: biased exponent of the largest raised |dS|
  uint32_t tmem_base;
  volatile int abort_flag;
};

// A block owns 128 rows and walks the other side in tiles of kWalk rows.  Narrow heads: 64, so that the accumulators need half of the
// tensor memory and two blocks share an SM; one's softmax, loads and output then run under the other's products.  Wide heads:
// 128, one block an SM.  Four warps for each 64 columns make P and dS, then one warp loads and one issues products.
template <int DP>
struct BwdShape {
  static constexpr int kWalk = DP == 64 ? 64 : 128;
  static constexpr int kHalves = kWalk / 64;
  static constexpr int kLoad = 4 * kHalves, kIssue = kLoad + 1;
  static constexpr int kThreads = (kIssue + 1) * 32;
  static constexpr int kBlocks = DP == 64 ? 2 : 1;
  // Rings of the walked side: kStages in the key-side kernel (q, d_o); in the query-side kernel K stays until dq has used it and V
  // only until dP is made.  At head dim 128, two stages of each against three of K and two of V, a training step: 7 prompts of 45 to
  // 4099 tokens, 4 key heads 558 -> 515 us; 8328 tokens, 16 heads 2558 -> 2166 us.  (Three and one: 538, 2400.)
  static constexpr int kStages = DP == 64 ? 4 : 2, kStagesK = DP == 64 ? 4 : 3, kStagesV = DP == 64 ? 4 : 2;
  static constexpr int kOwnBytes = DP / 64 * kBoxBytes, kWalkBytes = kWalk * DP * 2;
  static constexpr uint32_t kColumns = DP == 64 ? 256 : 512;
  static constexpr size_t kSmemBase = 1024 + 2 * kOwnBytes + sizeof(BwdShared);
  static constexpr size_t kSmemQ = kSmemBase + static_cast<size_t>(kStagesK + kStagesV) * kWalkBytes;  // query-side kernel
  static constexpr size_t kSmem = kSmemBase + static_cast<size_t>(2 * kStages) * kWalkBytes + kStages * 2 * kWalk * 4;  // key side: rows' sums
  static_assert(kSmem <= 232448 && kSmemQ <= 232448, "227 KB");
};

// dS as an fp16 operand.  It is as small as P times the incoming gradient, and fp16 has 15 powers of two below 1 (10 more with
// ever fewer bits) and 15 above: with d_o of 1e-3 a fifth of 8328 keys' dS became zero (dq off by 0.58 % of its norm, 0.05 % with the
// result rounded alone), and beyond 65 504 it was infinite.  So each row of the A operand, and with it the row's sums in tensor memory, is
// raised by a power of two of its own: at first 2^40; whenever a tile's largest value passes 2^15, the row's power falls so that this
// value lies at 2^7, and the sums so far are lowered to match.  What fp16 then takes off is 2^-11 of a value, or 2^-32 of the row's
// largest.  A multiplication by a power of two is exact, and so is the way back in fp32 at the end.  bf16 has fp32's range.
// Cost: the largest of 64 values a thread and tile (wide heads: an exponent shared by the two warps of a row); an fp16 training step of
// 8328 tokens, 16 heads of 64 1589 -> 1634 us, of 128 2214 -> 2293; ragged prompts, 4 key heads of 128 517 -> 541.
template <typename T>
constexpr bool kRaised = std::is_same<T, __half>::value;
constexpr int kFirstLift = 40, kGoal = 7, kMost = 15;

// Whole warp, behind the tile's masks: 64 of the row's values, raised by 2^lift.  Returns what they and the sums must be multiplied with
// (1 as a rule), and lowers `lift` to match.
template <int HALVES>
__device__ __forceinline__ float lift_row(const float (&x)[64], int& lift, bool live, BwdShared* sh, int half, int row, int tile, bool& ok) {
  float top[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 64; i += 4)
#pragma unroll
    for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], fabsf(x[i + e]));
  int exponent = static_cast<int>(__float_as_uint(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))) >> 23);
  if (HALVES == 2) {
    sh->top[tile & 1][half][row] = static_cast<uint8_t>(exponent);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&sh->top_full[row >> 5]);
    ok = ok && warp_wait(&sh->top_full[row >> 5], tile & 1, &sh->abort_flag);
    exponent = max(exponent, static_cast<int>(sh->top[tile & 1][half ^ 1][row]));
  }
  // infinite values stay what they are; rows behind the sequence hold its neighbour's and are not stored
  if (!live || exponent == 255 || exponent < 127 + kMost) return 1.f;
  lift += 127 + kGoal - exponent;
  return __int_as_float((127 + 127 + kGoal - exponent) << 23);
}

// Columns [from, to) of the row's sums in tensor memory times f
__device__ __forceinline__ void scale_sums(uint32_t addr, int from, int to, float f) {
#pragma unroll 1
  for (int b = from; b < to; b += 8) {
    uint32_t o[8];
    tmem_ld_x8(addr + b, o);
    tmem_wait_ld();
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
    tmem_store8(addr + b, o);
  }
  tmem_wait_st();
}

// Barriers, the block's tile and tensor memory; the same in both kernels.
template <int DP>
__device__ __forceinline__ uint32_t bwd_setup(BwdShared* sh, const PackedParams& p, bool key_side, int64_t rank, int warp, int lane) {
  using Shape = BwdShape<DP>;
  if (warp == Shape::kLoad) {
    PackedSeq s{};
    int64_t tiles = 0, end = 0;
    const bool found = packed_find_sorted(p, key_side, kTile, rank, &s, &tiles, &end);
    if (lane == 0) {
      sh->seq = s;
      sh->tiles = tiles;
      sh->end = end;
      sh->found = found;
      for (uint64_t* b : {&sh->own_full, &sh->s_full, &sh->dp_full, &sh->ds_done, &sh->all_done}) mbar_init(b, 1);
      for (uint64_t* b : {&sh->s_read, &sh->dp_read, &sh->p_full, &sh->ds_full}) mbar_init(b, Shape::kLoad);
      for (int i = 0; i < 4; ++i) {
        mbar_init(&sh->a_full[i], 1);
        mbar_init(&sh->a_empty[i], 1);
        mbar_init(&sh->b_full[i], 1);
        mbar_init(&sh->b_empty[i], 1);
        mbar_init(&sh->st_full[i], 1);
        mbar_init(&sh->top_full[i], 2);
      }
      sh->abort_flag = 0;
      mbar_fence_init();
      fence_proxy_async_smem();
    }
  }
  if (warp == Shape::kIssue) tmem_alloc(&sh->tmem_base, Shape::kColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return __shfl_sync(0xffffffffu, sh->tmem_base, 0);
}

// columns [from, to) of one row of an accumulator in this thread's TMEM lane, times lower, then times mul, as 16-bit values (zeros if
// !any); `base` is the tensor that the row `dst` belongs to; `more`, if any: values to be added in between, four columns every kTile
template <typename T>
__device__ __forceinline__ void store_acc(const void* base, T* dst, uint32_t addr, int from, int to, int D, float lower, float mul, bool live,
                                          bool any, const float4* more = nullptr) {
#pragma unroll 1
  for (int b = from; b < to; b += 32) {
    if (b >= D) break;
    float o[32];
    tmem_load32(addr + b, o);  // without a product: whatever is there, and unused
    tmem_wait_ld();
#pragma unroll
    for (int k = 0; k < 32; ++k) o[k] *= lower;
    if (more != nullptr) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float4 m = more[(b / 4 + c) * kTile];
        o[4 * c] += m.x;
        o[4 * c + 1] += m.y;
        o[4 * c + 2] += m.z;
        o[4 * c + 3] += m.w;
      }
    }
    uint32_t e[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) e[k] = any ? pack_half2<T>(o[2 * k] * mul, o[2 * k + 1] * mul) : 0u;
    if (live) store_row32(dst + b, e, D - b, row_sectors(base, D));
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(BwdShape<DP>::kThreads, BwdShape<DP>::kBlocks)
packed_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ CUtensorMap tmG, const PackedParams p, const int ab_format) {
  using Shape = BwdShape<DP>;
  constexpr int SK = Shape::kStagesK, SV = Shape::kStagesV;  // depths of the rings of K and V
  constexpr int TB = Shape::kOwnBytes, W = Shape::kWalk, WB = Shape::kWalkBytes;
  constexpr uint32_t kS = 0, kDp = W, kDs = 2 * W, kDq = Shape::kColumns - DP;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* q_smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* g_smem = q_smem + TB;
  unsigned char* k_smem = g_smem + TB;
  unsigned char* v_smem = k_smem + SK * WB;
  BwdShared* sh = reinterpret_cast<BwdShared*>(v_smem + SV * WB);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int head = blockIdx.x % p.H, kv = head / (p.H / p.Hk);
  const uint32_t tmem = bwd_setup<DP>(sh, p, false, blockIdx.x / p.H, warp, lane);
  if (!sh->found) {
    packed_zero_rows<T>(p.dq, nullptr, sh->end, p.total_q, p.H, head, p.D, blockIdx.x / p.H - sh->tiles, gridDim.x / p.H - sh->tiles,
                        blockDim.x);
  } else {
    const PackedSeq s = {uniform(sh->seq.q0), uniform(sh->seq.lq), uniform(sh->seq.k0), uniform(sh->seq.lk), uniform(sh->seq.tile)};
    const int off = s.lk - s.lq;
    const int r0 = s.tile * kTile;
    const int keys = p.causal ? max(0, min(s.lk, min(r0 + kTile, s.lq) + off)) : s.lk;
    const int n = (keys + W - 1) / W;

    if (warp == Shape::kLoad) {
      if (lane == 0 && n > 0) {
        bool ok = true;
        int jk = 0, jv = 0;  // key tiles whose K and V have been asked for
        mbar_arrive_expect_tx(&sh->own_full, 2 * TB);
        load_rows<DP>(q_smem, &tmQ, head, s.q0 + r0, &sh->own_full);
        load_rows<DP>(g_smem, &tmG, head, s.q0 + r0, &sh->own_full);
        while (jk < n) {  // V first: in the order in which stages come back, dP(j + 1) before dq(j)
          const int sv = jv % SV, sk = jk % SK;
          ok = mbar_wait_bounded(&sh->b_empty[sv], ((jv / SV) & 1u) ^ 1u);
          if (!ok || sh->abort_flag) break;
          mbar_arrive_expect_tx(&sh->b_full[sv], WB);
          load_rows<DP, W>(v_smem + sv * WB, &tmV, kv, s.k0 + jv * W, &sh->b_full[sv]);
          ++jv;
          ok = mbar_wait_bounded(&sh->a_empty[sk], ((jk / SK) & 1u) ^ 1u);
          if (!ok || sh->abort_flag) break;
          mbar_arrive_expect_tx(&sh->a_full[sk], WB);
          load_rows<DP, W>(k_smem + sk * WB, &tmK, kv, s.k0 + jk * W, &sh->a_full[sk]);
          ++jk;
        }
        if (!ok) sh->abort_flag = 1;
        if (sh->abort_flag) {  // let the copies in flight land before the shared memory is given up
          mbar_wait_limit(&sh->own_full, 0, kDrainLimitNs);
          for (int u = max(0, jk - SK); u < jk; ++u) mbar_wait_limit(&sh->a_full[u % SK], (u / SK) & 1u, kDrainLimitNs);
          for (int u = max(0, jv - SV); u < jv; ++u) mbar_wait_limit(&sh->b_full[u % SV], (u / SV) & 1u, kDrainLimitNs);
          report_status(p.status, GW_ERR_TIMEOUT);
        }
      }
    } else if (warp == Shape::kIssue) {
      const uint32_t idesc_s = make_idesc_mn(ab_format, kTile, W);
      const uint32_t idesc_o = make_idesc_mn(ab_format, kTile, DP) | kBMajorMN;
      const uint64_t qd = make_smem_desc(smem_u32(q_smem)), gd = make_smem_desc(smem_u32(g_smem));
      const uint64_t kd = make_smem_desc(smem_u32(k_smem)), vd = make_smem_desc(smem_u32(v_smem));
      const uint64_t kd_mn = make_smem_desc_mn(smem_u32(k_smem));
      bool ok = n == 0 || warp_wait(&sh->own_full, 0, &sh->abort_flag);
      auto products = [&](int j) {  // S and dP of key tile j, each as soon as the one before it has been read
        const int sk = j % SK, sv = j % SV;
        ok = warp_wait(&sh->a_full[sk], (j / SK) & 1, &sh->abort_flag);
        if (!ok) return;
        if ((j + 1) * W > s.lk) zero_rows_from<DP, W>(k_smem + sk * WB, s.lk - j * W);  // K is also dq's operand
        if (j > 0) ok = warp_wait(&sh->s_read, (j - 1) & 1, &sh->abort_flag);
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) {
          mma_rows<DP>(tmem + kS, qd, kd + sk * (WB >> 4), idesc_s);
          tc_commit(&sh->s_full);
        }
        ok = warp_wait(&sh->b_full[sv], (j / SV) & 1, &sh->abort_flag);
        if (j > 0) ok = ok && warp_wait(&sh->dp_read, (j - 1) & 1, &sh->abort_flag);
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) {
          mma_rows<DP>(tmem + kDp, gd, vd + sv * (WB >> 4), idesc_s);
          tc_commit(&sh->dp_full);
          tc_commit(&sh->b_empty[sv]);
        }
      };
      if (n > 0 && ok) products(0);
      for (int j = 0; j < n && ok; ++j) {
        const int st = j % SK;
        if (j + 1 < n) products(j + 1);
        ok = ok && warp_wait(&sh->ds_full, j & 1, &sh->abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < W / 16; ++i)
            tc_mma_f16_ts(tmem + kDq, tmem + kDs + i * 8, kd_mn + st * (WB >> 4) + i * (16 * 128 >> 4), idesc_o, (j > 0 || i > 0) ? 1u : 0u);
          tc_commit(&sh->a_empty[st]);
          tc_commit(&sh->ds_done);
        }
      }
      if (!ok) {
        sh->abort_flag = 1;
        if (lane == 0) report_status(p.status, GW_ERR_TIMEOUT);
      }
    } else {
      const int half = warp >> 2;
      const int row = r0 + (warp & 3) * 32 + lane;
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const bool live = row < s.lq;
      const int64_t token = s.q0 + row;
      // D of this row, from the saved output.  D's error is shared by the whole row of dS, where the errors of the 16-bit dS largely
      // cancel: with o as rounded it is up to half of the gradients' error over few keys, hence o_low.
      float delta = 0.f, neg_lse = -INFINITY;
      bool ok = true;
      const int64_t at = static_cast<int64_t>(head) * p.total_q + token;
      if (n > 0) {
        // 64 columns a thread (the other half's warps take the rest of a wide head); d_o is in shared memory
        const T* o = static_cast<const T*>(p.o) + (token * p.H + head) * p.D;
        const T* low = static_cast<const T*>(p.o_low) + (token * p.H + head) * p.D;
        uint4 ow[8], lw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int col = half * 64 + i * 8;
          const bool there = live && col < p.D;
          ow[i] = there ? *reinterpret_cast<const uint4*>(o + col) : make_uint4(0, 0, 0, 0);
          lw[i] = there && p.o_low != nullptr ? *reinterpret_cast<const uint4*>(low + col) : make_uint4(0, 0, 0, 0);
        }
        if (live) {
          const float lse = p.lse[at];
          neg_lse = lse == -INFINITY ? -INFINITY : -lse * kLog2e;
        }
        ok = warp_wait(&sh->own_full, 0, &sh->abort_flag);
        const int r = (warp & 3) * 32 + lane;
        const unsigned char* g = g_smem + half * kBoxBytes + r * 128;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint4 gw = *reinterpret_cast<const uint4*>(g + ((i ^ (r & 7)) << 4));
          const uint32_t oe[4] = {ow[i].x, ow[i].y, ow[i].z, ow[i].w}, ge[4] = {gw.x, gw.y, gw.z, gw.w};
          const uint32_t le[4] = {lw[i].x, lw[i].y, lw[i].z, lw[i].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float a, b, c, d, e, f;
            unpack2<T>(oe[k], a, b);
            unpack2<T>(ge[k], c, d);
            unpack2<T>(le[k], e, f);
            delta = fmaf(a + e, c, delta);
            delta = fmaf(b + f, d, delta);
          }
        }
        if (!live) delta = 0.f;  // behind the sequence d_o is its neighbour's
        if (Shape::kHalves == 2) {
          sh->part[half][r] = delta;
          named_bar_sync(1, 256);
          delta = sh->part[0][r] + sh->part[1][r];
        }
      }
      if (live && half == 0) p.delta[at] = delta;
      const float c = p.scale * kLog2e;
      int lift = kRaised<T> ? kFirstLift : 0;
      const uint64_t c2 = pack_f2(c, c), nd2 = pack_f2(-delta, -delta);
      uint64_t l2 = pack_f2(neg_lse + lift, neg_lse + lift);
      const int limit = (p.causal ? min(s.lk, row + off + 1) : s.lk) - half * 64;
      const int open = p.causal ? min(s.lk, r0 + off + 1) : s.lk;
      for (int j = 0; j < n; ++j) {
        ok = ok && warp_wait(&sh->s_full, j & 1, &sh->abort_flag);
        if (!ok) break;
        tc_fence_after();
        float x[64], y[64];
        tmem_load32(tmem + lanes + kS + half * 64, x);
        tmem_load32(tmem + lanes + kS + half * 64 + 32, x + 32);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->s_read);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float a, b;
          unpack_f2(fma_f2(pack_f2(x[2 * i], x[2 * i + 1]), c2, l2), a, b);
          x[2 * i] = exp2_fast(a);
          x[2 * i + 1] = exp2_fast(b);
        }
        ok = warp_wait(&sh->dp_full, j & 1, &sh->abort_flag);
        if (!ok) break;
        tc_fence_after();
        tmem_load32(tmem + lanes + kDp + half * 64, y);
        tmem_load32(tmem + lanes + kDp + half * 64 + 32, y + 32);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->dp_read);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const uint64_t d = mul_f2(pack_f2(x[2 * i], x[2 * i + 1]), add_f2(pack_f2(y[2 * i], y[2 * i + 1]), nd2));
          unpack_f2(d, x[2 * i], x[2 * i + 1]);
        }
        if ((j + 1) * W > open) {
          const int valid = limit - j * W;
#pragma unroll
          for (int i = 0; i < 64; ++i) x[i] = i < valid ? x[i] : 0.f;
        }
        if constexpr (kRaised<T>) {
          const float f = lift_row<Shape::kHalves>(x, lift, live, sh, half, (warp & 3) * 32 + lane, j, ok);
          if (!ok) break;
          if (__any_sync(0xffffffffu, f != 1.f)) {
            l2 = pack_f2(neg_lse + lift, neg_lse + lift);
#pragma unroll
            for (int i = 0; i < 64; ++i) x[i] *= f;
            if (j > 0) {
              ok = warp_wait(&sh->ds_done, (j - 1) & 1, &sh->abort_flag);
              if (!ok) break;
              tc_fence_after();
              scale_sums(tmem + lanes + kDq, half * (DP / Shape::kHalves), (half + 1) * (DP / Shape::kHalves), f);
            }
          }
        }
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) w[i] = pack_half2<T>(x[2 * i], x[2 * i + 1]);
        if (j > 0) {
          ok = warp_wait(&sh->ds_done, (j - 1) & 1, &sh->abort_flag);
          if (!ok) break;
          tc_fence_after();
        }
        tmem_store32(tmem + lanes + kDs + half * 32, w);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->ds_full);
      }
      if (n > 0 && ok) ok = warp_wait(&sh->ds_done, (n - 1) & 1, &sh->abort_flag);
      if (!ok) {
        sh->abort_flag = 1;
        report_status(p.status, GW_ERR_TIMEOUT);
      }
      tc_fence_after();
      store_acc<T>(p.dq, static_cast<T*>(p.dq) + (token * p.H + head) * p.D, tmem + lanes + kDq, half * (DP / Shape::kHalves), (half + 1) * (DP / Shape::kHalves), p.D,
                   exp2f(static_cast<float>(-lift)), p.scale, live, n > 0);
    }
  }
  if (blockIdx.x == 0 && warp == Shape::kLoad) {
    __syncwarp();
    packed_check(p);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == Shape::kIssue) tmem_dealloc(tmem, Shape::kColumns);
}

// The whole cluster meets, and what its blocks wrote before is there behind it.
__device__ __forceinline__ void cluster_meet() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// BLOCKS blocks share the query tiles of one key tile: with two, a cluster, the second adds its sums to the first's at the end
// through the first's shared memory (the first's part, then the second's: a fixed order).
template <typename T, int DP, int BLOCKS>
__global__ void __launch_bounds__(BwdShape<DP>::kThreads, BwdShape<DP>::kBlocks)
packed_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ CUtensorMap tmG, const PackedParams p, const int ab_format) {
  using Shape = BwdShape<DP>;
  constexpr int ST = Shape::kStages, TB = Shape::kOwnBytes, W = Shape::kWalk, WB = Shape::kWalkBytes;
  constexpr uint32_t kS = 0, kDp = W, kDv = 2 * W, kDk = 2 * W + DP;
  // fp16 holds nothing below 2^-24 and few bits below 2^-14, and a P of a long sequence is that small: it is raised by 2^12 (P <= 1)
  // and dv lowered again; bf16 has fp32's range
  constexpr float kLift = kRaised<T> ? 12.f : 0.f;
  constexpr float kLower = kRaised<T> ? 1.f / 4096.f : 1.f;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* k_smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* v_smem = k_smem + TB;
  unsigned char* q_smem = v_smem + TB;
  unsigned char* g_smem = q_smem + ST * WB;
  float* stats = reinterpret_cast<float*>(g_smem + ST * WB);  // [stage][-lse log2 e + lift, -D][W]
  BwdShared* sh = reinterpret_cast<BwdShared*>(stats + ST * 2 * W);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int64_t item = blockIdx.x / BLOCKS;
  const int share = blockIdx.x % BLOCKS, kv = static_cast<int>(item % p.Hk), group = p.H / p.Hk;
  const uint32_t tmem = bwd_setup<DP>(sh, p, true, item / p.Hk, warp, lane);
  if (!sh->found) {
    const int64_t part = (item / p.Hk - sh->tiles) * BLOCKS + share, parts = (gridDim.x / BLOCKS / p.Hk - sh->tiles) * BLOCKS;
    packed_zero_rows<T>(p.dk, nullptr, sh->end, p.total_k, p.Hk, kv, p.D, part, parts, blockDim.x);
    packed_zero_rows<T>(p.dv, nullptr, sh->end, p.total_k, p.Hk, kv, p.D, part, parts, blockDim.x);
  } else {
    const PackedSeq s = {uniform(sh->seq.q0), uniform(sh->seq.lq), uniform(sh->seq.k0), uniform(sh->seq.lk), uniform(sh->seq.tile)};
    const int off = s.lk - s.lq;
    const int c0 = s.tile * kTile;
    const int q_tiles = (s.lq + W - 1) / W;
    const int first = p.causal ? max(0, c0 - off) / W : 0;  // the first query tile that sees one of these keys
    const int per_head = max(0, q_tiles - first);
    const int all = per_head * group;                        // pairs of tiles
    const int begin = share == 0 ? 0 : (all + 1) / BLOCKS;   // this block's: the first half, rounded up, or the rest
    const int n = BLOCKS == 1 ? all : share == 0 ? (all + 1) / 2 : all / 2;
    float dk_lower = 1.f;  // of this thread's row

    if (warp == Shape::kLoad) {
      bool ok = true;
      int i = 0;
      if (lane == 0 && n > 0) {
        mbar_arrive_expect_tx(&sh->own_full, 2 * TB);
        load_rows<DP>(k_smem, &tmK, kv, s.k0 + c0, &sh->own_full);
        load_rows<DP>(v_smem, &tmV, kv, s.k0 + c0, &sh->own_full);
      }
      for (; i < n; ++i) {
        const int st = i % ST, at = begin + i, head = kv * group + at / per_head, r0 = (first + at % per_head) * W;
        ok = warp_wait(&sh->a_empty[st], ((i / ST) & 1u) ^ 1u, &sh->abort_flag);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&sh->a_full[st], WB);
          load_rows<DP, W>(q_smem + st * WB, &tmQ, head, s.q0 + r0, &sh->a_full[st]);
          mbar_arrive_expect_tx(&sh->b_full[st], WB);
          load_rows<DP, W>(g_smem + st * WB, &tmG, head, s.q0 + r0, &sh->b_full[st]);
        }
        float* dst = stats + st * 2 * W;
        const int64_t base = static_cast<int64_t>(head) * p.total_q + s.q0 + r0;
#pragma unroll
        for (int k = 0; k < W / 32; ++k) {
          const int r = lane + 32 * k;
          float l = -INFINITY, d = 0.f;  // rows behind the end: P = 0, dS = 0
          if (r0 + r < s.lq) {
            l = p.lse[base + r];
            l = l == -INFINITY ? -INFINITY : fmaf(-l, kLog2e, kLift);
            d = -p.delta[base + r];
          }
          dst[r] = l;
          dst[W + r] = d;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->st_full[st]);
      }
      if (!ok) sh->abort_flag = 1;
      if (warp_sees(sh->abort_flag) && lane == 0) {  // let the copies in flight land before the shared memory is given up
        if (n > 0) mbar_wait_limit(&sh->own_full, 0, kDrainLimitNs);
        for (int u = max(0, i - ST); u < i; ++u) {
          mbar_wait_limit(&sh->a_full[u % ST], (u / ST) & 1u, kDrainLimitNs);
          mbar_wait_limit(&sh->b_full[u % ST], (u / ST) & 1u, kDrainLimitNs);
        }
        report_status(p.status, GW_ERR_TIMEOUT);
      }
    } else if (warp == Shape::kIssue) {
      const uint32_t idesc_s = make_idesc_mn(ab_format, kTile, W);
      const uint32_t idesc_o = make_idesc_mn(ab_format, kTile, DP) | kBMajorMN;
      const uint64_t kd = make_smem_desc(smem_u32(k_smem)), vd = make_smem_desc(smem_u32(v_smem));
      const uint64_t qd = make_smem_desc(smem_u32(q_smem)), gd = make_smem_desc(smem_u32(g_smem));
      const uint64_t qd_mn = make_smem_desc_mn(smem_u32(q_smem)), gd_mn = make_smem_desc_mn(smem_u32(g_smem));
      bool ok = n == 0 || warp_wait(&sh->own_full, 0, &sh->abort_flag);
      // S^T = K Q^T / dP^T = V d_o^T of query tile i; rows behind the sequence's end become zeros first
      auto product = [&](int i, uint64_t* full, unsigned char* tiles, uint64_t a, uint64_t b, uint32_t d, uint64_t* done) {
        const int st = i % ST, left = s.lq - (first + (begin + i) % per_head) * W;
        ok = warp_wait(&full[st], (i / ST) & 1, &sh->abort_flag);
        if (!ok) return;
        if (left < W) zero_rows_from<DP, W>(tiles + st * WB, left);
        tc_fence_after();
        if (elect_one()) {
          mma_rows<DP>(d, a, b + st * (WB >> 4), idesc_s);
          tc_commit(done);
        }
      };
      // accumulator += (P or dS)^T (d_o or Q): the A operand's two halves of 64 queries are 64 columns apart
      auto accumulate = [&](int i, uint32_t acc, uint32_t a, uint64_t b) {
        const uint64_t at = b + (i % ST) * (WB >> 4);
#pragma unroll
        for (int k = 0; k < W / 16; ++k)
          tc_mma_f16_ts(acc, a + (k >> 2) * 64 + (k & 3) * 8, at + k * (16 * 128 >> 4), idesc_o, (i > 0 || k > 0) ? 1u : 0u);
      };
      if (n > 0 && ok) {
        product(0, sh->a_full, q_smem, kd, qd, tmem + kS, &sh->s_full);
        if (ok) product(0, sh->b_full, g_smem, vd, gd, tmem + kDp, &sh->dp_full);
      }
      for (int i = 0; i < n && ok; ++i) {
        ok = warp_wait(&sh->p_full, i & 1, &sh->abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) accumulate(i, tmem + kDv, tmem + kS, gd_mn);
        if (i + 1 < n) product(i + 1, sh->a_full, q_smem, kd, qd, tmem + kS, &sh->s_full);
        ok = ok && warp_wait(&sh->ds_full, i & 1, &sh->abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          accumulate(i, tmem + kDk, tmem + kDp, qd_mn);
          tc_commit(&sh->a_empty[i % ST]);
        }
        if (i + 1 < n) product(i + 1, sh->b_full, g_smem, vd, gd, tmem + kDp, &sh->dp_full);
      }
      if (n > 0 && elect_one()) tc_commit(&sh->all_done);
      if (!ok) {
        sh->abort_flag = 1;
        if (lane == 0) report_status(p.status, GW_ERR_TIMEOUT);
      }
    } else {
      const int half = warp >> 2;
      const int row = c0 + (warp & 3) * 32 + lane;
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t s_addr = tmem + lanes + kS + half * 64, d_addr = tmem + lanes + kDp + half * 64;
      const float c = p.scale * kLog2e;
      const uint64_t c2 = pack_f2(c, c);
      int lift = kRaised<T> ? kFirstLift : 0;
      float raise = exp2f(lift - kLift);  // from the raised P to the raised dS
      bool ok = true;
      for (int i = 0; i < n; ++i) {
        const int st = i % ST, r0 = (first + (begin + i) % per_head) * W;
        const ulonglong2* l2 = reinterpret_cast<const ulonglong2*>(stats + st * 2 * W + half * 64);
        const ulonglong2* d2 = reinterpret_cast<const ulonglong2*>(stats + st * 2 * W + W + half * 64);
        const bool edge = p.causal && c0 + kTile - 1 > r0 + off;  // some pair of the tiles is masked
        const int from = row - off - r0 - half * 64;              // the first column that sees this key
        ok = warp_wait(&sh->st_full[st], (i / ST) & 1, &sh->abort_flag) && warp_wait(&sh->s_full, i & 1, &sh->abort_flag);
        if (!ok) break;
        tc_fence_after();
        float x[64], y[64];
        uint32_t w[32];
        tmem_load32(s_addr, x);
        tmem_load32(s_addr + 32, x + 32);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const ulonglong2 l = l2[k];
          float a, b, e, f;
          unpack_f2(fma_f2(pack_f2(x[4 * k], x[4 * k + 1]), c2, l.x), a, b);
          unpack_f2(fma_f2(pack_f2(x[4 * k + 2], x[4 * k + 3]), c2, l.y), e, f);
          x[4 * k] = exp2_fast(a);
          x[4 * k + 1] = exp2_fast(b);
          x[4 * k + 2] = exp2_fast(e);
          x[4 * k + 3] = exp2_fast(f);
        }
        if (edge) {
#pragma unroll
          for (int k = 0; k < 64; ++k) x[k] = k >= from ? x[k] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) w[k] = pack_half2<T>(x[2 * k], x[2 * k + 1]);
        tmem_store32(s_addr, w);  // P takes S's place: every thread its own lane, behind its own loads
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full);

        ok = warp_wait(&sh->dp_full, i & 1, &sh->abort_flag);
        if (!ok) break;
        tc_fence_after();
        tmem_load32(d_addr, y);
        tmem_load32(d_addr + 32, y + 32);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const ulonglong2 d = d2[k];
          uint64_t a = mul_f2(pack_f2(x[4 * k], x[4 * k + 1]), add_f2(pack_f2(y[4 * k], y[4 * k + 1]), d.x));
          uint64_t b = mul_f2(pack_f2(x[4 * k + 2], x[4 * k + 3]), add_f2(pack_f2(y[4 * k + 2], y[4 * k + 3]), d.y));
          if (kRaised<T>) {
            a = mul_f2(a, pack_f2(raise, raise));
            b = mul_f2(b, pack_f2(raise, raise));
          }
          unpack_f2(a, y[4 * k], y[4 * k + 1]);
          unpack_f2(b, y[4 * k + 2], y[4 * k + 3]);
        }
        if (edge) {
#pragma unroll
          for (int k = 0; k < 64; ++k) y[k] = k >= from ? y[k] : 0.f;
        }
        if constexpr (kRaised<T>) {
          const float f = lift_row<Shape::kHalves>(y, lift, row < s.lk, sh, half, (warp & 3) * 32 + lane, i, ok);
          if (!ok) break;
          if (__any_sync(0xffffffffu, f != 1.f)) {
            raise = exp2f(lift - kLift);
#pragma unroll
            for (int k = 0; k < 64; ++k) y[k] *= f;
            // dP was asked for behind the last product that adds to dk, so that product is done
            if (i > 0) scale_sums(tmem + lanes + kDk, half * (DP / Shape::kHalves), (half + 1) * (DP / Shape::kHalves), f);
          }
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) w[k] = pack_half2<T>(y[2 * k], y[2 * k + 1]);
        tmem_store32(d_addr, w);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->ds_full);
      }
      if (n > 0 && ok) ok = warp_wait(&sh->all_done, 0, &sh->abort_flag);
      if (!ok) {
        sh->abort_flag = 1;
        report_status(p.status, GW_ERR_TIMEOUT);
      }
      dk_lower = exp2f(static_cast<float>(-lift));
      tc_fence_after();
    }

    // ------------------------------ output: dv by the first four warps, dk by the last four ------------------------------
    const int half = warp >> 2, r = (warp & 3) * 32 + lane, row = c0 + r;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    // the other block's sums, [dv, dk][DP / 4][128 rows], where the operand tiles were
    float4* sums = reinterpret_cast<float4*>(k_smem);
    if (BLOCKS == 2) {
      cluster_meet();  // the first block's tiles have been used
      if (share == 1 && warp < Shape::kLoad && n > 0) {
        uint32_t remote;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(smem_u32(sums)));
        for (int which = 0; which < 2; ++which) {
          if (half != (which == 0 ? 0 : Shape::kHalves - 1)) continue;
#pragma unroll 1
          for (int b = 0; b < DP; b += 32) {
            float o[32];
            tmem_load32(tmem + lanes + (which == 0 ? kDv : kDk) + b, o);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] *= which == 0 ? kLower : dk_lower;
#pragma unroll
            for (int c = 0; c < 8; ++c)
              asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(remote + (((which * (DP / 4) + b / 4 + c) * kTile + r) << 4)),
                           "f"(o[4 * c]), "f"(o[4 * c + 1]), "f"(o[4 * c + 2]), "f"(o[4 * c + 3])
                           : "memory");
          }
        }
      }
      cluster_meet();
    }
    if (share == 0 && warp < Shape::kLoad) {
      const bool live = row < s.lk;
      const int64_t at = (static_cast<int64_t>(s.k0 + row) * p.Hk + kv) * p.D;
      const float4* more = BLOCKS == 2 && all > 1 ? sums + r : nullptr;
      if (half == 0) store_acc<T>(p.dv, static_cast<T*>(p.dv) + at, tmem + lanes + kDv, 0, DP, p.D, kLower, 1.f, live, all > 0, more);
      if (half == Shape::kHalves - 1)
        store_acc<T>(p.dk, static_cast<T*>(p.dk) + at, tmem + lanes + kDk, 0, DP, p.D, dk_lower, p.scale, live, all > 0,
                     more != nullptr ? more + DP / 4 * kTile : nullptr);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == Shape::kIssue) tmem_dealloc(tmem, Shape::kColumns);
}

template <typename T, int DP>
int launch_bwd(const PackedParams& p, int dtype, int dev, int sms, cudaStream_t st) {
  CUtensorMap mq, mk, mv, mg;
  GW_CUDA_TRY(cudaSetDevice(dev));  // a thread that has launched nothing yet has no context to encode tensor maps in
  // each tensor once as the side that a block owns and once as the side that it walks
  int rc = GW_OK;
  auto maps = [&](int q_rows, int k_rows) {
    rc = make_token_map(&mq, p.q, dtype, p.total_q, p.H, p.D, p.qs[0], p.qs[1], q_rows);
    if (rc == GW_OK) rc = make_token_map(&mg, p.d_o, dtype, p.total_q, p.H, p.D, p.dos[0], p.dos[1], q_rows);
    if (rc == GW_OK) rc = make_token_map(&mk, p.k, dtype, p.total_k, p.Hk, p.D, p.ks[0], p.ks[1], k_rows);
    if (rc == GW_OK) rc = make_token_map(&mv, p.v, dtype, p.total_k, p.Hk, p.D, p.vs[0], p.vs[1], k_rows);
    return rc;
  };
  constexpr int W = BwdShape<DP>::kWalk, kThreads = BwdShape<DP>::kThreads;
  maps(kTile, W);
  static OncePerDevice once_q, once_k, once_k2;
  constexpr size_t smem_q = BwdShape<DP>::kSmemQ, smem = BwdShape<DP>::kSmem;
  if (rc == GW_OK) rc = ensure_dynamic_smem(packed_dq_kernel<T, DP>, smem_q, once_q, dev);
  if (rc == GW_OK) rc = ensure_dynamic_smem(packed_dkv_kernel<T, DP, 1>, smem, once_k, dev);
  if (rc == GW_OK) rc = ensure_dynamic_smem(packed_dkv_kernel<T, DP, 2>, smem, once_k2, dev);
  if (rc != GW_OK) return rc;
  const int format = dtype == GW_BF16 ? 1 : 0;
  const int64_t q_items = packed_tile_bound(p.total_q, kTile, p.nseq) * p.H, k_items = packed_tile_bound(p.total_k, kTile, p.nseq) * p.Hk;
  if (q_items > 0x7fffffff || k_items > 0x3fffffff) return GW_ERR_UNSUPPORTED;
  packed_dq_kernel<T, DP><<<static_cast<unsigned>(q_items), kThreads, smem_q, st>>>(mq, mk, mv, mg, p, format);
  GW_LAUNCH_CHECK();
  if (p.dk == nullptr) return GW_OK;  // keys and values without a gradient
  if (W != kTile && maps(W, kTile) != GW_OK) return rc;
  // Few and long blocks -- grouped heads, whose key tiles walk every head of the group -- leave SMs idle at the end: two share a key
  // tile.  Training steps, alone -> shared.  One causal sequence of 4099 tokens, 2 key heads of 64 under 16: 687 -> 447 us, of 128
  // 670 -> 466; ragged prompts, 4 key heads of 128 (1.74 rounds of blocks) 563 -> 518.  Not beyond: 8200 causal tokens (1.76 rounds)
  // 1187 -> 1189, 8 views of 1041 tokens, 4 key heads of 128 (1.78) 446 -> 475.  With 16 pairs of tiles and more for a block: 2 views of 1041
  // tokens, 4 key heads of 128 under 8 (16 pairs) 95 -> 85, 200 queries of 16 heads over 8 (8 pairs) 99 -> 110.  Not for heads of their
  // own: 4099 tokens, 16 heads of 64 451 -> 480, of 128 623 -> 679.
  const int64_t items = (p.total_k + kTile - 1) / kTile * p.Hk, at_once = static_cast<int64_t>(sms) * BwdShape<DP>::kBlocks;
  const bool share = p.H > p.Hk && 4 * items < 7 * at_once && p.total_q * (p.H / p.Hk) >= 16 * static_cast<int64_t>(W) * p.nseq;
  if (!share) {
    packed_dkv_kernel<T, DP, 1><<<static_cast<unsigned>(k_items), kThreads, smem, st>>>(mq, mk, mv, mg, p, format);
    GW_LAUNCH_CHECK();
    return GW_OK;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * k_items));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute cluster = {};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = 2;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cfg.attrs = &cluster;
  cfg.numAttrs = 1;
  GW_CUDA_TRY(cudaLaunchKernelEx(&cfg, packed_dkv_kernel<T, DP, 2>, mq, mk, mv, mg, p, format));
  return GW_OK;
}

}  // namespace

int packed_mma_bwd(const PackedParams& p, int dtype, int dev, int sms, cudaStream_t st) {
  if (dtype == GW_BF16) return p.D <= 64 ? launch_bwd<__nv_bfloat16, 64>(p, dtype, dev, sms, st) : launch_bwd<__nv_bfloat16, 128>(p, dtype, dev, sms, st);
  return p.D <= 64 ? launch_bwd<__half, 64>(p, dtype, dev, sms, st) : launch_bwd<__half, 128>(p, dtype, dev, sms, st);
}

}  // namespace gw
