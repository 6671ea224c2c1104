// Attention over packed sequences on the tcgen05 tensor cores, forward, 16-bit operands, head dim up to 128.
//
// One block owns 256 query rows of one head (two tiles of 128) and walks the keys in tiles of 128.  For each pair of tiles
//   S = Q K^T          both operands in shared memory (TMA, 128-byte swizzle), S in tensor memory, fp32
//   P = 2^(c S - c m)  one thread owns one row: 128 values of its TMEM lane, no shuffles; c = scale log2 e
//   O += P V           P goes back to tensor memory as the 16-bit A operand, O stays in tensor memory
// m is the running maximum, but a lagging one: O and the sum l are rescaled only when a row's maximum has grown by more than
// 2^8 (P then lies within 2^8, where both 16-bit types keep their full precision, and l in fp32), which after the first tiles
// hardly ever happens, so the rescaling pass over O is off the critical path.
//
// Warps 0-3 and 4-7 are the softmax of the two tiles, warp 8 loads, warp 9 issues the products.  The two tiles alternate:
// while one is in its softmax the tensor cores make the other's S and O.
#include "gw_packed_mma.cuh"

namespace gw {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int make_token_map(CUtensorMap* map, const void* base, int dtype, int64_t tokens, int heads, int D, int64_t token_stride, int64_t head_stride) {
  static EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess) return (EncodeTiledFn) nullptr;
    return q == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiledFn>(ptr) : (EncodeTiledFn) nullptr;
  }();
  if (!fn) return GW_ERR_CUDA;
  const cuuint64_t gdim[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens > 0 ? tokens : 1)};
  const cuuint64_t gstride[2] = {static_cast<cuuint64_t>(head_stride) * 2, static_cast<cuuint64_t>(token_stride) * 2};
  const cuuint32_t box[3] = {64, 1, kTile};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(map, dtype == GW_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                        const_cast<void*>(base), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    g_last_cuda_error = static_cast<int>(r);
    return GW_ERR_CUDA;
  }
  return GW_OK;
}

namespace {

constexpr int kFwdThreads = 320;
constexpr float kLag = 8.f;  // a maximum may grow by this much (as a power of two) before O is rescaled

template <int DP>
struct FwdShape {
  static constexpr int kStages = DP == 64 ? 4 : 2;       // K and V rings
  static constexpr int kTileBytes = DP / 64 * kBoxBytes;
  // tensor memory: S of both tiles, then P where it has room of its own (it takes S's place for wide heads), then O
  static constexpr uint32_t kS = 0, kP = DP == 64 ? 256 : 0, kPStride = DP == 64 ? 64 : 128, kO = DP == 64 ? 384 : 256;
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(2 + 2 * kStages) * kTileBytes + 512;
};

template <int STAGES>
struct FwdShared {
  uint64_t q_full[2], s_full[2], p_full[2], o_done[2];
  uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
  PackedSeq seq;
  int64_t tiles, end;
  int found;
  uint32_t tmem_base;
  volatile int abort_flag;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kFwdThreads, 1)
packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const PackedParams p, const int ab_format) {
  using Shape = FwdShape<DP>;
  constexpr int ST = Shape::kStages, TB = Shape::kTileBytes;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* q_smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* k_smem = q_smem + 2 * TB;
  unsigned char* v_smem = k_smem + ST * TB;
  FwdShared<ST>* sh = reinterpret_cast<FwdShared<ST>*>(v_smem + ST * TB);
  static_assert(sizeof(FwdShared<ST>) <= 512, "shared bookkeeping");

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int head = blockIdx.y, kv = head / (p.H / p.Hk);

  if (warp == 8) {
    PackedSeq s{};
    int64_t tiles = 0, end = 0;
    const bool found = packed_find(p, false, 2 * kTile, blockIdx.x, &s, &tiles, &end);
    if (lane == 0) {
      sh->seq = s;
      sh->tiles = tiles;
      sh->end = end;
      sh->found = found;
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sh->q_full[i], 1);
        mbar_init(&sh->s_full[i], 1);
        mbar_init(&sh->p_full[i], 4);
        mbar_init(&sh->o_done[i], 1);
      }
      for (int i = 0; i < ST; ++i) {
        mbar_init(&sh->k_full[i], 1);
        mbar_init(&sh->k_empty[i], 1);
        mbar_init(&sh->v_full[i], 1);
        mbar_init(&sh->v_empty[i], 1);
      }
      sh->abort_flag = 0;
      mbar_fence_init();
      fence_proxy_async_smem();
    }
  }
  if (warp == 9) tmem_alloc(&sh->tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh->tmem_base, 0);
  if (!sh->found) {
    packed_zero_rows<T>(p.o, p.lse, sh->end, p.total_q, p.H, head, p.D, blockIdx.x - sh->tiles, gridDim.x - sh->tiles);
  } else {
    const PackedSeq s = sh->seq;
    const int off = s.lk - s.lq;
    // longest first: under a causal mask the later tiles of a sequence see more keys
    const int tile = p.causal ? (s.lq + 2 * kTile - 1) / (2 * kTile) - 1 - s.tile : s.tile;
    const int r0 = tile * 2 * kTile;
    int keys[2], n[2];  // keys that any row of each tile sees; key tiles
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int last = min(r0 + (t + 1) * kTile, s.lq);
      keys[t] = last <= r0 + t * kTile ? 0 : p.causal ? max(0, min(s.lk, last + off)) : s.lk;
      n[t] = (keys[t] + kTile - 1) / kTile;
    }
    const int most = max(n[0], n[1]);

    if (warp == 8) {
      // ------------------------------ loads ------------------------------
      if (lane == 0) {
        bool ok = true;
        int j = 0;
        for (int t = 0; t < 2; ++t)
          if (n[t] > 0) {
            mbar_arrive_expect_tx(&sh->q_full[t], TB);
            load_rows<DP>(q_smem + t * TB, &tmQ, head, s.q0 + r0 + t * kTile, &sh->q_full[t]);
          }
        for (; j < most; ++j) {
          const int st = j % ST;
          const uint32_t par = ((j / ST) & 1u) ^ 1u;
          ok = mbar_wait_bounded(&sh->k_empty[st], par);
          if (!ok || sh->abort_flag) break;
          mbar_arrive_expect_tx(&sh->k_full[st], TB);
          load_rows<DP>(k_smem + st * TB, &tmK, kv, s.k0 + j * kTile, &sh->k_full[st]);
          ok = mbar_wait_bounded(&sh->v_empty[st], par);
          mbar_arrive_expect_tx(&sh->v_full[st], TB);
          load_rows<DP>(v_smem + st * TB, &tmV, kv, s.k0 + j * kTile, &sh->v_full[st]);
          if (!ok || sh->abort_flag) { ++j; break; }
        }
        if (!ok) sh->abort_flag = 1;
        if (sh->abort_flag) {  // let the copies in flight land before the shared memory is given up
          for (int t = 0; t < 2; ++t)
            if (n[t] > 0) mbar_wait_limit(&sh->q_full[t], 0, kDrainLimitNs);
          for (int u = max(0, j - ST); u < j; ++u) {
            mbar_wait_limit(&sh->k_full[u % ST], (u / ST) & 1u, kDrainLimitNs);
            mbar_wait_limit(&sh->v_full[u % ST], (u / ST) & 1u, kDrainLimitNs);
          }
          report_status(p.status, GW_ERR_TIMEOUT);
        }
      }
    } else if (warp == 9) {
      // ------------------------------ products ------------------------------
      const uint32_t idesc_s = make_idesc_mn(ab_format, kTile, kTile);
      const uint32_t idesc_o = make_idesc_mn(ab_format, kTile, DP) | kBMajorMN;
      const uint64_t qd = make_smem_desc(smem_u32(q_smem)), kd = make_smem_desc(smem_u32(k_smem)), vd = make_smem_desc_mn(smem_u32(v_smem));
      bool ok = true;
      auto scores = [&](int t, int j) {
        if (lane == 0) {
          mma_rows<DP>(tmem + Shape::kS + t * kTile, qd + t * (TB >> 4), kd + (j % ST) * (TB >> 4), idesc_s);
          tc_commit(&sh->s_full[t]);
        }
      };
      if (most > 0) {
        ok = mbar_wait_bounded(&sh->k_full[0], 0);
        for (int t = 0; t < 2 && ok; ++t)
          if (n[t] > 0) {
            ok = mbar_wait_bounded(&sh->q_full[t], 0);
            tc_fence_after();
            if (ok) scores(t, 0);
          }
        if (lane == 0) tc_commit(&sh->k_empty[0]);
      }
      for (int j = 0; j < most && ok && !sh->abort_flag; ++j) {
        const int st = j % ST;
        bool v_here = false, k_next = false;
        for (int t = 0; t < 2; ++t) {
          if (j >= n[t]) continue;
          ok = ok && mbar_wait_bounded(&sh->p_full[t], j & 1);
          if (ok && j + 1 < n[t] && !k_next) {
            ok = mbar_wait_bounded(&sh->k_full[(j + 1) % ST], ((j + 1) / ST) & 1);
            k_next = true;
          }
          if (ok && !v_here) {
            ok = mbar_wait_bounded(&sh->v_full[st], (j / ST) & 1);
            v_here = true;
            if (ok && (j + 1) * kTile > s.lk) zero_rows_from<DP>(v_smem + st * TB, s.lk - j * kTile);
          }
          if (!ok) break;
          tc_fence_after();
          // narrow heads have S free as soon as P is written elsewhere; for wide heads P sits on S
          if (DP == 64 && j + 1 < n[t]) scores(t, j + 1);
          if (lane == 0) {
            const int steps = min(kTile, (keys[t] - j * kTile + 15) & ~15) / 16;
            for (int i = 0; i < steps; ++i)
              tc_mma_f16_ts(tmem + Shape::kO + t * DP, tmem + Shape::kP + t * Shape::kPStride + i * 8,
                            vd + st * (TB >> 4) + i * (16 * 128 >> 4), idesc_o, (j > 0 || i > 0) ? 1u : 0u);
            tc_commit(&sh->o_done[t]);
          }
          if (DP != 64 && j + 1 < n[t]) scores(t, j + 1);
        }
        if (lane == 0 && ok) {
          tc_commit(&sh->v_empty[st]);
          if (k_next) tc_commit(&sh->k_empty[(j + 1) % ST]);
        }
      }
      if (!ok) {
        sh->abort_flag = 1;
        if (lane == 0) report_status(p.status, GW_ERR_TIMEOUT);
      }
    } else {
      // ------------------------------ softmax and output ------------------------------
      const int t = warp >> 2;
      const int row = r0 + t * kTile + (warp & 3) * 32 + lane;
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t s_addr = tmem + lanes + Shape::kS + t * kTile, p_addr = tmem + lanes + Shape::kP + t * Shape::kPStride;
      const uint32_t o_addr = tmem + lanes + Shape::kO + t * DP;
      const float c = p.scale * kLog2e;
      const int limit = p.causal ? min(s.lk, row + off + 1) : s.lk;  // keys this row sees
      const int open = p.causal ? min(s.lk, r0 + t * kTile + off + 1) : s.lk;  // keys that every row of the tile sees
      const int tiles = n[t];
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < tiles; ++j) {
        ok = mbar_wait_bounded(&sh->s_full[t], j & 1);
        if (!ok || sh->abort_flag) break;
        tc_fence_after();
        float x[128];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_load32(s_addr + 32 * i, x + 32 * i);
        tmem_wait_ld();
        if ((j + 1) * kTile > open) {
          const int valid = limit - j * kTile;
#pragma unroll
          for (int i = 0; i < 128; ++i) x[i] = i < valid ? x[i] : -INFINITY;
        }
        float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int i = 4; i < 128; i += 8) {
#pragma unroll
          for (int k = 0; k < 4; ++k) top[k] = fmaxf(top[k], fmaxf(x[i + k], i + 4 + k < 128 ? x[i + 4 + k] : x[i + k]));
        }
        const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        bool o_ready = false;
        if (j == 0) {
          m = mx;
        } else {
          const bool grown = mx > m && !((mx - m) * c <= kLag);  // also from -inf
          if (__any_sync(0xffffffffu, grown)) {
            const float shrink = grown ? exp2_fast((m - mx) * c) : 1.f;
            l *= shrink;
            if (grown) m = mx;
            ok = mbar_wait_bounded(&sh->o_done[t], (j - 1) & 1);
            if (!ok) break;
            o_ready = true;
            tc_fence_after();
#pragma unroll 1
            for (int b = 0; b < DP / 32; ++b) {
              float o[32];
              tmem_load32(o_addr + 32 * b, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= shrink;
              tmem_store32(o_addr + 32 * b, reinterpret_cast<const uint32_t*>(o));
            }
            tmem_wait_st();
          }
        }
        const float base = m == -INFINITY ? 0.f : -m * c;
        const uint64_t c2 = pack_f2(c, c), base2 = pack_f2(base, base);
        uint64_t sum[2] = {0, 0};
        uint32_t pk[64];
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          float a, b;
          unpack_f2(fma_f2(pack_f2(x[2 * i], x[2 * i + 1]), c2, base2), a, b);
          a = exp2_fast(a);
          b = exp2_fast(b);
          sum[i & 1] = add_f2(sum[i & 1], pack_f2(a, b));
          pk[i] = pack_half2<T>(a, b);
        }
        float s0, s1, s2, s3;
        unpack_f2(sum[0], s0, s1);
        unpack_f2(sum[1], s2, s3);
        l += (s0 + s1) + (s2 + s3);
        if (DP == 64 && j > 0 && !o_ready) {  // the previous product still reads P (for wide heads S, and so P, waited for it)
          ok = mbar_wait_bounded(&sh->o_done[t], (j - 1) & 1);
          if (!ok) break;
          tc_fence_after();
        }
        tmem_store32(p_addr, pk);
        tmem_store32(p_addr + 32, pk + 32);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[t]);
      }
      if (tiles > 0 && ok && !sh->abort_flag) ok = mbar_wait_bounded(&sh->o_done[t], (tiles - 1) & 1);
      if (!ok) {
        sh->abort_flag = 1;
        report_status(p.status, GW_ERR_TIMEOUT);
      }
      tc_fence_after();
      const bool live = row < s.lq;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T* dst = static_cast<T*>(p.o) + (static_cast<int64_t>(s.q0 + row) * p.H + head) * p.D;
#pragma unroll 1
      for (int b = 0; b < DP / 32; ++b) {
        if (32 * b >= p.D) break;
        float o[32];
        if (tiles > 0) {
          tmem_load32(o_addr + 32 * b, o);
          tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint4 w;
          uint32_t* e = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            e[k] = l == 0.f ? 0u : pack_half2<T>(o[8 * i + 2 * k] * inv, o[8 * i + 2 * k + 1] * inv);
          if (live && 32 * b + 8 * i < p.D) *reinterpret_cast<uint4*>(dst + 32 * b + 8 * i) = w;
        }
      }
      if (live && p.lse != nullptr)
        p.lse[static_cast<int64_t>(head) * p.total_q + s.q0 + row] = l == 0.f ? -INFINITY : fmaf(m, p.scale, log2f(l) * kLn2);
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

template <typename T, int DP>
int launch_fwd(const PackedParams& p, int dtype, int dev, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  GW_CUDA_TRY(cudaSetDevice(dev));  // a thread that has launched nothing yet has no context to encode tensor maps in
  int rc = make_token_map(&mq, p.q, dtype, p.total_q, p.H, p.D, p.qs[0], p.qs[1]);
  if (rc == GW_OK) rc = make_token_map(&mk, p.k, dtype, p.total_k, p.Hk, p.D, p.ks[0], p.ks[1]);
  if (rc == GW_OK) rc = make_token_map(&mv, p.v, dtype, p.total_k, p.Hk, p.D, p.vs[0], p.vs[1]);
  static OncePerDevice once;
  if (rc == GW_OK) rc = ensure_dynamic_smem(packed_fwd_kernel<T, DP>, FwdShape<DP>::kSmem, once, dev);
  if (rc != GW_OK) return rc;
  const dim3 grid(static_cast<unsigned>(packed_tile_bound(p.total_q, 2 * kTile, p.nseq)), p.H);
  packed_fwd_kernel<T, DP><<<grid, kFwdThreads, FwdShape<DP>::kSmem, st>>>(mq, mk, mv, p, dtype == GW_BF16 ? 1 : 0);
  GW_LAUNCH_CHECK();
  return GW_OK;
}

}  // namespace

int packed_mma_fwd(const PackedParams& p, int dtype, int dev, cudaStream_t st) {
  if (dtype == GW_BF16) return p.D <= 64 ? launch_fwd<__nv_bfloat16, 64>(p, dtype, dev, st) : launch_fwd<__nv_bfloat16, 128>(p, dtype, dev, st);
  return p.D <= 64 ? launch_fwd<__half, 64>(p, dtype, dev, st) : launch_fwd<__half, 128>(p, dtype, dev, st);
}

}  // namespace gw
