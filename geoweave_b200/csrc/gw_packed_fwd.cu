// Attention over packed sequences on the tcgen05 tensor cores, forward, 16-bit operands, head dim up to 128.
//
// One block owns 256 query rows of one head (two tiles of 128; one tile where the rows are few) and walks the keys in tiles of
// 128.  For each pair of tiles
//   S = Q K^T          both operands in shared memory (TMA, 128-byte swizzle), S in tensor memory, fp32
//   P = 2^(c S - c m)  one thread owns one row: 128 values of its TMEM lane, no shuffles; c = scale log2 e
//   O += P V           P goes back to tensor memory as the 16-bit A operand, O stays in tensor memory
// m is the running maximum, but a lagging one: O and the sum l are rescaled only when a row's maximum has grown by more than
// 2^8 (P then lies within 2^8, where both 16-bit types keep their full precision, and l in fp32), which after the first tiles
// hardly ever happens, so the rescaling pass over O is off the critical path.
//
// A persistent block takes its items (the rows of a head) from a list in falling order of work, one in every gridDim: the loads of
// the next item run under the last products and the output of this one.  Warps 0-3 and 4-7 are the softmax of the two tiles,
// warp 8 makes the work list and loads, the rest issue products.  While one tile is in its softmax the tensor cores make the
// other's S and O, and its own next S where P has room beside S (head dims up to 64: one issuing warp for each tile, so
// that neither waits for the other).  For wide heads P sits on S, the tensor cores are busy all the time, and one warp issues
// for both tiles in turn, which keeps them half a period apart; with two issuers their products interleave and the tiles fall into step.
#include "gw_packed_mma.cuh"

namespace gw {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int make_token_map(CUtensorMap* map, const void* base, int dtype, int64_t tokens, int heads, int D, int64_t token_stride, int64_t head_stride,
                   int rows) {
  static EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess) return (EncodeTiledFn) nullptr;
    return q == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiledFn>(ptr) : (EncodeTiledFn) nullptr;
  }();
  if (!fn) return GW_ERR_CUDA;
  const cuuint64_t gdim[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens > 0 ? tokens : 1)};
  const cuuint64_t gstride[2] = {static_cast<cuuint64_t>(head_stride) * 2, static_cast<cuuint64_t>(token_stride) * 2};
  const cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(rows)};
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

constexpr float kLag = 8.f;  // a maximum may grow by this much (as a power of two) before O is rescaled
constexpr int kTiles = 2;    // most query tiles of a block

// TILES: query tiles of a block, two where there are enough of them to occupy the SMs
template <int DP, int TILES>
struct FwdShape {
  static constexpr int kWarps = 4 * TILES, kLoad = kWarps, kIssue = kWarps + 1;  // softmax first, then one that loads, then issuers
  static constexpr int kIssuers = DP == 64 ? TILES : 1;
  static constexpr int kThreads = (kIssue + kIssuers) * 32;
  static constexpr int kStages = DP == 64 ? 3 : 2;  // K and V rings
  static constexpr int kTileBytes = DP / 64 * kBoxBytes;
  // tensor memory: S of both tiles, then P where it has room of its own (it takes S's place for wide heads), then O
  static constexpr uint32_t kS = 0, kP = DP == 64 ? 256 : 0, kPStride = DP == 64 ? 64 : 128, kO = DP == 64 ? 384 : 256;
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(TILES + 2 * kStages) * kTileBytes + 512;
};

enum { kItemRows, kItemTail, kItemEnd };
struct FwdItem {  // the rows of a block, of one head; or some rows behind the last sequence; or the end of the list
  int kind, head, part, q0, lq, k0, lk, off, r0;  // k0, lk: the keys that this item walks; query i sees those up to i + off
  int keys[kTiles], n[kTiles], most;  // keys that any row of each tile sees; key tiles of each, of both
  int64_t slot, slots, end;
};

struct FwdShared {
  uint64_t q_full[kTiles], q_empty[kTiles], s_full[kTiles], s_read[kTiles], p_half[kTiles], p_full[kTiles], o_done[kTiles];
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t item_full[2], item_empty[2];
  FwdItem item[2];
  uint32_t tmem_base;
  volatile int abort_flag;
};
static_assert(sizeof(FwdShared) <= 512, "shared bookkeeping");

// The next item is there when the loads of the one before it have all been issued: for warps whose tile has no rows in that one
// its whole length away, so the limit is long.  After a failure the loading warp ends the list at once.
__device__ __forceinline__ bool wait_item(FwdShared* sh, int i) {
  return warp_wait(&sh->item_full[i & 1], (i >> 1) & 1, &sh->abort_flag, 60 * kWaitLimitNs);
}

// Few rows against many keys: the key tiles of a row tile are divided among `count` items, which leave their unnormalised sums
struct FwdParts {
  int count;   // 1: not divided
  float* o;    // [H, count, total_q, D]
  float2* ml;  // [H, count, total_q]: maximum of scale log2 e S, sum
};

template <typename T, int DP, int TILES>
__global__ void __launch_bounds__(FwdShape<DP, TILES>::kThreads, 1)
packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const PackedParams p, const int64_t slots, const FwdParts fp, const int ab_format) {
  using Shape = FwdShape<DP, TILES>;
  constexpr int ST = Shape::kStages, TB = Shape::kTileBytes, NI = Shape::kIssuers;
  constexpr int kWarps = Shape::kWarps, kLoad = Shape::kLoad, kIssue = Shape::kIssue;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* q_smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* k_smem = q_smem + TILES * TB;
  unsigned char* v_smem = k_smem + ST * TB;
  FwdShared* sh = reinterpret_cast<FwdShared*>(v_smem + ST * TB);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;

  if (warp == kLoad && lane == 0) {
    for (int i = 0; i < TILES; ++i) {
      mbar_init(&sh->q_full[i], 1);
      mbar_init(&sh->q_empty[i], 1);
      mbar_init(&sh->s_full[i], 1);
      mbar_init(&sh->s_read[i], 4);
      mbar_init(&sh->p_half[i], 4);
      mbar_init(&sh->p_full[i], 4);
      mbar_init(&sh->o_done[i], 1);
    }
    for (int i = 0; i < ST; ++i) {
      mbar_init(&sh->k_full[i], 1);
      mbar_init(&sh->k_empty[i], NI);
      mbar_init(&sh->v_full[i], 1);
      mbar_init(&sh->v_empty[i], NI);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh->item_full[i], 1);
      mbar_init(&sh->item_empty[i], kWarps + NI);
    }
    sh->abort_flag = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (warp == kIssue) tmem_alloc(&sh->tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh->tmem_base, 0);
  bool ok = true;

  if (warp == kLoad) {
    // ------------------------------ work list and loads ------------------------------
    uint32_t ring = 0, q_use[kTiles] = {};  // key tiles and query tiles loaded so far
    int i = 0, told = 0;                    // items, and those of them that the others have been told of
    for (int64_t at = blockIdx.x; ok; at += gridDim.x, ++i) {
      FwdItem w{};
      const int parts = TILES == 1 ? fp.count : 1;
      PackedSeq seq{};
      int64_t rank, tiles = 0;
      bool found = false;
      for (;; at += gridDim.x) {  // past the empty slots
        rank = at / parts / p.H;
        if (rank >= slots) break;
        found = packed_find_sorted(p, false, TILES * kTile, rank, &seq, &tiles, &w.end);
        if (found || rank >= tiles) break;
      }
      w.part = static_cast<int>(at % parts);
      w.head = static_cast<int>(at / parts % p.H);
      if (rank >= slots) {
        w.kind = kItemEnd;
      } else if (found) {
        w.kind = kItemRows;
        w.q0 = seq.q0;
        w.lq = seq.lq;
        w.k0 = seq.k0;
        w.lk = seq.lk;
        w.off = seq.lk - seq.lq;
        w.r0 = seq.tile * TILES * kTile;
        if (parts > 1) {  // this part's run of key tiles, out of those that the tile's last row sees
          const int last = min(w.r0 + kTile, w.lq), seen = p.causal ? max(0, min(w.lk, last + w.off)) : w.lk;
          const int each = ((seen + kTile - 1) / kTile + parts - 1) / parts;
          const int from = static_cast<int>(min(static_cast<int64_t>(w.part) * each * kTile, static_cast<int64_t>(seen)));
          w.k0 += from;
          w.lk = static_cast<int>(min(static_cast<int64_t>(each) * kTile, static_cast<int64_t>(seen - from)));
          w.off -= from;
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          const int last = min(w.r0 + (t + 1) * kTile, w.lq);
          w.keys[t] = last <= w.r0 + t * kTile ? 0 : p.causal ? max(0, min(w.lk, last + w.off)) : w.lk;
          w.n[t] = (w.keys[t] + kTile - 1) / kTile;
          w.most = max(w.most, w.n[t]);
        }
      } else {
        w.kind = kItemTail;
        w.slot = (rank - tiles) * parts + w.part;
        w.slots = (slots - tiles) * parts;
      }
      ok = warp_wait(&sh->item_empty[i & 1], ((i >> 1) & 1) ^ 1, &sh->abort_flag);
      if (!ok) break;
      if (lane == 0) {
        sh->item[i & 1] = w;
        mbar_arrive(&sh->item_full[i & 1]);
      }
      ++told;
      if (w.kind == kItemEnd) break;
      if (w.kind == kItemTail) continue;
      const int kv = w.head / (p.H / p.Hk);
      auto load_q = [&](int t) {
        ok = ok && warp_wait(&sh->q_empty[t], (q_use[t] & 1) ^ 1, &sh->abort_flag);
        if (!ok) return;
        if (lane == 0) {
          mbar_arrive_expect_tx(&sh->q_full[t], TB);
          load_rows<DP>(q_smem + t * TB, &tmQ, w.head, w.q0 + w.r0 + t * kTile, &sh->q_full[t]);
        }
        ++q_use[t];
      };
      for (int j = 0; j < w.most && ok; ++j, ++ring) {
        const int st = ring % ST;
        const uint32_t par = ((ring / ST) & 1u) ^ 1u;
        if (j == 0 && w.n[0] > 0) load_q(0);
        ok = ok && warp_wait(&sh->k_empty[st], par, &sh->abort_flag);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&sh->k_full[st], TB);
          load_rows<DP>(k_smem + st * TB, &tmK, kv, w.k0 + j * kTile, &sh->k_full[st]);
        }
        if (TILES == 2 && j == 0 && w.n[1] > 0) load_q(1);
        ok = ok && warp_wait(&sh->v_empty[st], par, &sh->abort_flag);
        if (lane == 0) {  // also after a wait that ran out, so that the drain below finds both copies of the stage
          mbar_arrive_expect_tx(&sh->v_full[st], TB);
          load_rows<DP>(v_smem + st * TB, &tmV, kv, w.k0 + j * kTile, &sh->v_full[st]);
        }
      }
    }
    if (blockIdx.x == 0) packed_check(p);
    if (!ok) sh->abort_flag = 1;
    if (warp_sees(sh->abort_flag) && lane == 0) {
      sh->item[told & 1].kind = kItemEnd;
      mbar_arrive(&sh->item_full[told & 1]);
      // let the copies in flight land before the shared memory is given up
      for (int t = 0; t < TILES; ++t)
        if (q_use[t] > 0) mbar_wait_limit(&sh->q_full[t], (q_use[t] - 1) & 1, kDrainLimitNs);
      for (uint32_t u = ring > ST ? ring - ST : 0u; u <= ring; ++u) {
        mbar_wait_limit(&sh->k_full[u % ST], (u / ST) & 1u, kDrainLimitNs);
        mbar_wait_limit(&sh->v_full[u % ST], (u / ST) & 1u, kDrainLimitNs);
      }
      report_status(p.status, GW_ERR_TIMEOUT);
    }
  } else if (warp >= kIssue) {
    // ------------------------------ products: of one tile, or of both in turn ------------------------------
    const int w0 = warp - kIssue;
    const uint32_t idesc_s = make_idesc_mn(ab_format, kTile, kTile);
    const uint32_t idesc_o = make_idesc_mn(ab_format, kTile, DP) | kBMajorMN;
    const uint64_t qd = make_smem_desc(smem_u32(q_smem)), kd = make_smem_desc(smem_u32(k_smem));
    const uint64_t vd = make_smem_desc_mn(smem_u32(v_smem));
    uint32_t ring = 0, done[kTiles] = {}, q_use[kTiles] = {};  // key tiles in the ring before this item; of each tile; query tiles
    for (int i = 0; ok; ++i) {
      ok = wait_item(sh, i);
      if (!ok) break;
      const FwdItem* item = &sh->item[i & 1];
      const int kind = uniform(item->kind), most = uniform(item->most), lk = uniform(item->lk);
      int n[kTiles], keys[kTiles];
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        n[t] = uniform(item->n[t]);
        keys[t] = uniform(item->keys[t]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->item_empty[i & 1]);
      if (kind == kItemEnd) break;
      if (kind == kItemTail) continue;
      auto scores = [&](int t, int j) {  // S of key tile j; S has been read: for wide heads P, which sits on it, has been used
        const uint32_t at = ring + j, c = done[t] + j;
        if (j == 0) ok = ok && warp_wait(&sh->q_full[t], q_use[t] & 1, &sh->abort_flag);
        if (DP == 64 || j == 0) ok = ok && warp_wait(&sh->k_full[at % ST], (at / ST) & 1, &sh->abort_flag);
        if (DP == 64 && c > 0) ok = ok && warp_wait(&sh->s_read[t], (c - 1) & 1, &sh->abort_flag);
        if (!ok) return;
        tc_fence_after();
        if (elect_one()) {
          mma_rows<DP>(tmem + Shape::kS + t * kTile, qd + t * (TB >> 4), kd + (at % ST) * (TB >> 4), idesc_s);
          tc_commit(&sh->s_full[t]);
          if (j + 1 == n[t]) tc_commit(&sh->q_empty[t]);
        }
      };
      int mine = 0;
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        if (t % NI != w0 || n[t] == 0) continue;
        mine = max(mine, n[t]);
        scores(t, 0);
      }
      // A stage goes back once for each issuer.  One whose tile does not read it still waits until it is full: running ahead
      // of the loads it would count twice in one phase of the barrier.
      auto pass_on = [&](uint64_t* full, uint64_t* empty, uint32_t at) {
        ok = ok && warp_wait(&full[at % ST], (at / ST) & 1, &sh->abort_flag);
        if (ok && lane == 0) mbar_arrive(&empty[at % ST]);
      };
      if (mine > 0) {
        if (elect_one()) tc_commit(&sh->k_empty[ring % ST]);
      } else if (most > 0) {
        pass_on(sh->k_full, sh->k_empty, ring);
      }
      for (int j = 0; j < most && ok; ++j) {
        const uint32_t st = (ring + j) % ST, st_next = (ring + j + 1) % ST;
        bool v_here = false;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          if (t % NI != w0 || j >= n[t]) continue;
          const uint32_t c = done[t] + j;
          if (DP == 64 && j + 1 < n[t]) scores(t, j + 1);  // P has its own place: ahead of this tile's softmax
          if (!v_here) {
            ok = ok && warp_wait(&sh->v_full[st], ((ring + j) / ST) & 1, &sh->abort_flag);
            if (DP != 64 && j + 1 < mine) ok = ok && warp_wait(&sh->k_full[st_next], ((ring + j + 1) / ST) & 1, &sh->abort_flag);
            // With an issuer for each tile both clear these rows, one perhaps while the other's product reads them: zeros over the zeros
            // that it wrote itself and waited for.
            if (ok && (j + 1) * kTile > lk) zero_rows_from<DP>(v_smem + st * TB, lk - j * kTile);
            v_here = true;
          }
          const int steps = min(kTile, (keys[t] - j * kTile + 15) & ~15) / 16;
          const uint32_t oa = tmem + Shape::kO + t * DP, pa = tmem + Shape::kP + t * Shape::kPStride;
          const uint64_t va = vd + st * (TB >> 4);
          // Wide heads: the product over the first half of P runs while the second is being made (a row's O has been rescaled
          // before either half): 16 384 tokens, 16 heads 1811 -> 1782 us, two causal sequences of 3000, 100 rows each 33.5 -> 31.8 us.
          // For narrow heads it is the exponentials that bound the kernel.
          if (DP != 64) {
            ok = ok && warp_wait(&sh->p_half[t], c & 1, &sh->abort_flag);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              if (steps >= 4) {
#pragma unroll
                for (int k = 0; k < 4; ++k) tc_mma_f16_ts(oa, pa + k * 8, va + k * (16 * 128 >> 4), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
              } else {
                for (int k = 0; k < steps; ++k) tc_mma_f16_ts(oa, pa + k * 8, va + k * (16 * 128 >> 4), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
              }
            }
          }
          ok = ok && warp_wait(&sh->p_full[t], c & 1, &sh->abort_flag);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            constexpr int from = DP != 64 ? 4 : 0;
            if (steps == 8) {
#pragma unroll
              for (int k = from; k < 8; ++k) tc_mma_f16_ts(oa, pa + k * 8, va + k * (16 * 128 >> 4), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
            } else {
              for (int k = from; k < steps; ++k) tc_mma_f16_ts(oa, pa + k * 8, va + k * (16 * 128 >> 4), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
            }
            tc_commit(&sh->o_done[t]);
          }
          if (DP != 64 && j + 1 < n[t]) scores(t, j + 1);
        }
        if (j < mine) {
          if (ok && elect_one()) tc_commit(&sh->v_empty[st]);
        } else {
          pass_on(sh->v_full, sh->v_empty, ring + j);
        }
        if (j + 1 < mine) {
          if (ok && elect_one()) tc_commit(&sh->k_empty[st_next]);
        } else if (j + 1 < most) {
          pass_on(sh->k_full, sh->k_empty, ring + j + 1);
        }
      }
      ring += most;
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        done[t] += n[t];
        q_use[t] += n[t] > 0 ? 1 : 0;
      }
    }
    if (!ok) {
      sh->abort_flag = 1;
      if (lane == 0) report_status(p.status, GW_ERR_TIMEOUT);
    }
  } else {
    // ------------------------------ softmax and output ------------------------------
    const int t = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + Shape::kS + t * kTile, p_addr = tmem + lanes + Shape::kP + t * Shape::kPStride;
    const uint32_t o_addr = tmem + lanes + Shape::kO + t * DP;
    const float c = p.scale * kLog2e;
    uint32_t done = 0;  // key tiles of this tile so far
    for (int i = 0; ok; ++i) {
      ok = wait_item(sh, i);
      if (!ok) break;
      const FwdItem* item = &sh->item[i & 1];  // given back behind the output
      const int kind = item->kind;
      if (kind == kItemEnd) break;
      if (kind == kItemTail) {
        packed_zero_rows<T>(p.o, p.lse, item->end, p.total_q, p.H, item->head, p.D, item->slot, item->slots, kWarps * 32);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->item_empty[i & 1]);
        continue;
      }
      const int lk = item->lk, off = item->off, first = item->r0 + t * kTile, row = first + (warp & 3) * 32 + lane;
      const int limit = p.causal ? min(lk, row + off + 1) : lk;   // keys this row sees
      const int open = p.causal ? min(lk, first + off + 1) : lk;  // keys that every row of the tile sees
      const int tiles = item->n[t];
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < tiles; ++j, ++done) {
        ok = warp_wait(&sh->s_full[t], done & 1, &sh->abort_flag);
        if (!ok) break;
        tc_fence_after();
        float x[128];
#pragma unroll
        for (int k = 0; k < 4; ++k) tmem_load32(s_addr + 32 * k, x + 32 * k);
        tmem_wait_ld();
        if (DP == 64) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->s_read[t]);
        }
        if ((j + 1) * kTile > open) {
          const int valid = limit - j * kTile;
#pragma unroll
          for (int k = 0; k < 128; ++k) x[k] = k < valid ? x[k] : -INFINITY;
        }
        float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int k = 4; k < 128; k += 8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], fmaxf(x[k + e], k + 4 + e < 128 ? x[k + 4 + e] : x[k + e]));
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
            ok = warp_wait(&sh->o_done[t], (done - 1) & 1, &sh->abort_flag);
            if (!ok) break;
            o_ready = true;
            tc_fence_after();
#pragma unroll 1
            for (int b = 0; b < DP / 8; ++b) {  // narrow pieces: the row's 128 scores are in registers
              uint32_t o[8];
              tmem_ld_x8(o_addr + 8 * b, o);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * shrink);
              tmem_store8(o_addr + 8 * b, o);
            }
            tmem_wait_st();
          }
        }
        const float base = m == -INFINITY ? 0.f : -m * c;
        const uint64_t c2 = pack_f2(c, c), base2 = pack_f2(base, base);
        uint64_t sum[2] = {0, 0};
        // P as an operand of the second product has the inputs' type, the only one that may stand beside V: off by half a step at most, and
        // o by 0.0010 (37 keys) to 0.0016 of its norm (4000) in bf16, beside the 0.0017 of its own rounding; fp16 an eighth.  P as two
        // operands would keep more and double that product.  l is summed from P before its rounding.
        uint32_t pk[64];
        auto exponentials = [&](int from, int to) {
#pragma unroll
          for (int k = from; k < to; ++k) {
            float a, b;
            unpack_f2(fma_f2(pack_f2(x[2 * k], x[2 * k + 1]), c2, base2), a, b);
            a = exp2_fast(a);
            b = exp2_fast(b);
            sum[k & 1] = add_f2(sum[k & 1], pack_f2(a, b));
            pk[k] = pack_half2<T>(a, b);
          }
        };
        if (DP != 64) {  // wide heads: the tensor cores may begin with the first half of P
          exponentials(0, 32);
          tmem_store32(p_addr, pk);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->p_half[t]);
          exponentials(32, 64);
        } else {
          exponentials(0, 64);
        }
        float s0, s1, s2, s3;
        unpack_f2(sum[0], s0, s1);
        unpack_f2(sum[1], s2, s3);
        l += (s0 + s1) + (s2 + s3);
        if (DP == 64 && j > 0 && !o_ready) {  // the previous product still reads P (for wide heads S, and so P, waited for it)
          ok = warp_wait(&sh->o_done[t], (done - 1) & 1, &sh->abort_flag);
          if (!ok) break;
          tc_fence_after();
        }
        if (DP == 64) tmem_store32(p_addr, pk);
        tmem_store32(p_addr + 32, pk + 32);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[t]);
      }
      if (!ok) break;
      if (tiles > 0) {
        ok = warp_wait(&sh->o_done[t], (done - 1) & 1, &sh->abort_flag);
        if (!ok) break;
        tc_fence_after();
      }
      const bool live = row < item->lq;
      const int64_t token = item->q0 + row;
      const int head = item->head;
      const int64_t part_row = TILES == 1 ? (static_cast<int64_t>(head) * fp.count + item->part) * p.total_q + token : 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->item_empty[i & 1]);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int64_t at = (token * p.H + head) * p.D;
      T *dst = static_cast<T*>(p.o) + at, *low = p.o_low != nullptr ? static_cast<T*>(p.o_low) + at : nullptr;
#pragma unroll 1
      for (int b = 0; b < DP / 32; ++b) {
        if (32 * b >= p.D) break;
        float o[32];
        tmem_load32(o_addr + 32 * b, o);  // without a key: whatever is there, and unused
        tmem_wait_ld();
        if (TILES == 1 && fp.count > 1) {
          if (live) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (32 * b + 4 * k < p.D)
                reinterpret_cast<float4*>(fp.o + part_row * p.D)[8 * b + k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
          continue;
        }
        uint32_t e[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) e[k] = l == 0.f ? 0u : pack_half2<T>(o[2 * k] * inv, o[2 * k + 1] * inv);
        if (live) store_row32(dst + 32 * b, e, p.D - 32 * b, row_sectors(p.o, p.D));
        if (low != nullptr) {
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float u, v;
            unpack2<T>(e[k], u, v);
            e[k] = l == 0.f ? 0u : pack_half2<T>(fmaf(o[2 * k], inv, -u), fmaf(o[2 * k + 1], inv, -v));
          }
          if (live) store_row32(low + 32 * b, e, p.D - 32 * b, row_sectors(p.o_low, p.D));
        }
      }
      tc_fence_before();  // O may be written again once this item's successor has its first P
      if (TILES == 1 && fp.count > 1) {
        if (live) fp.ml[part_row] = make_float2(m * c, l);
        continue;
      }
      if (live && p.lse != nullptr)
        p.lse[head * p.total_q + token] = l == 0.f ? -INFINITY : fmaf(m, p.scale, log2f(l) * kLn2);
    }
    if (!ok) {
      sh->abort_flag = 1;
      report_status(p.status, GW_ERR_TIMEOUT);
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kIssue) tmem_dealloc(tmem, 512);
}

// Joins the parts of a row (a warp a row): o = sum o_i 2^(m_i - m) / sum l_i 2^(m_i - m)
template <typename T>
__global__ void __launch_bounds__(256) packed_join_kernel(const PackedParams p, const FwdParts fp) {
  const int lane = threadIdx.x & 31, col = lane * 4;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5), token = row / p.H;
  const int head = static_cast<int>(row % p.H);
  // rows behind the last sequence are zeros already
  if (token >= p.total_q || p.nseq == 0 || token >= packed_border(p.cu_q, p.nseq, p.total_q)) return;
  const int64_t first = static_cast<int64_t>(head) * fp.count * p.total_q + token;
  const float2 ml = lane < fp.count ? fp.ml[first + lane * p.total_q] : make_float2(-INFINITY, 0.f);
  const float m = [&] {
    float x = ml.y > 0.f || ml.y != ml.y ? ml.x : -INFINITY;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
  }();
  const float weight = ml.y == 0.f ? 0.f : exp2f(ml.x - m);
  float l = ml.y * weight;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < fp.count; ++i) {
    const float f = __shfl_sync(0xffffffffu, weight, i);
    if (f == 0.f || col >= p.D) continue;  // a part without a key left nothing
    const float4 o = *reinterpret_cast<const float4*>(fp.o + (first + i * p.total_q) * p.D + col);
    acc[0] = fmaf(o.x, f, acc[0]);
    acc[1] = fmaf(o.y, f, acc[1]);
    acc[2] = fmaf(o.z, f, acc[2]);
    acc[3] = fmaf(o.w, f, acc[3]);
  }
  const int64_t at = (token * p.H + head) * p.D + col;
  if (col < p.D)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = l == 0.f ? 0.f : acc[i] / l;
      const T rounded = from_float<T>(x);
      static_cast<T*>(p.o)[at + i] = rounded;
      if (p.o_low != nullptr) static_cast<T*>(p.o_low)[at + i] = from_float<T>(x - to_float(rounded));
    }
  if (lane == 0 && p.lse != nullptr) p.lse[head * p.total_q + token] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <typename T, int DP, int TILES>
int launch_fwd(const PackedParams& p, int dtype, int dev, int sms, int parts, void* workspace, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  GW_CUDA_TRY(cudaSetDevice(dev));  // a thread that has launched nothing yet has no context to encode tensor maps in
  int rc = make_token_map(&mq, p.q, dtype, p.total_q, p.H, p.D, p.qs[0], p.qs[1], kTile);
  if (rc == GW_OK) rc = make_token_map(&mk, p.k, dtype, p.total_k, p.Hk, p.D, p.ks[0], p.ks[1], kTile);
  if (rc == GW_OK) rc = make_token_map(&mv, p.v, dtype, p.total_k, p.Hk, p.D, p.vs[0], p.vs[1], kTile);
  using Shape = FwdShape<DP, TILES>;
  static OncePerDevice once;
  if (rc == GW_OK) rc = ensure_dynamic_smem(packed_fwd_kernel<T, DP, TILES>, Shape::kSmem, once, dev);
  if (rc != GW_OK) return rc;
  const int64_t slots = packed_tile_bound(p.total_q, TILES * kTile, p.nseq), items = slots * p.H * parts;
  FwdParts fp{parts, static_cast<float*>(workspace), nullptr};
  fp.ml = reinterpret_cast<float2*>(fp.o + (parts > 1 ? static_cast<int64_t>(p.H) * parts * p.total_q * p.D : 0));
  packed_fwd_kernel<T, DP, TILES><<<static_cast<unsigned>(items < sms ? items : sms), Shape::kThreads, Shape::kSmem, st>>>(
      mq, mk, mv, p, slots, fp, dtype == GW_BF16 ? 1 : 0);
  GW_LAUNCH_CHECK();
  if (parts > 1) {
    packed_join_kernel<T><<<static_cast<unsigned>((p.total_q * p.H + 7) / 8), 256, 0, st>>>(p, fp);
    GW_LAUNCH_CHECK();
  }
  return GW_OK;
}

// Rows for fewer blocks of two tiles than there are SMs: one tile a block, twice the blocks (one view of 1041 tokens, 16 heads: 20.5 us
// against 26.6; 1041 rows against 33 312 keys: 274 against 383).  With three views the two are close, 43 and 45, with 32 two tiles
// win, 290 us against 357, since both share every key tile.  (Each alone, with cold caches.)
bool few_rows(const PackedParams& p, int sms) { return (p.total_q + 2 * kTile - 1) / (2 * kTile) * p.H < sms; }

// Fewer row tiles than half the SMs, and keys enough for at least six key tiles a part: the keys are divided too (300 rows, 8 heads
// against 8328 keys: 29 us against 76; 1041 rows, 4 heads against 33 312: 87 against 274).  With nine key tiles in two parts
// the second kernel costs what they bring (23.6 against 20.5).
int key_parts(const PackedParams& p, int sms) {
  int64_t tiles = (p.total_q + kTile - 1) / kTile;
  if (tiles < p.nseq) tiles = p.nseq;  // each sequence has a tile of its own
  if (p.nseq == 0 || tiles * p.H * 2 > sms) return 1;
  int64_t parts = sms / (tiles * p.H);
  const int64_t run = p.total_k / p.nseq / (6 * kTile);
  if (parts > run) parts = run;
  return static_cast<int>(parts < 2 ? 1 : parts > 16 ? 16 : parts);
}

template <typename T>
int choose_fwd(const PackedParams& p, int dtype, int dev, int sms, void* workspace, cudaStream_t st) {
  const bool few = few_rows(p, sms);
  const int parts = few ? key_parts(p, sms) : 1;
  if (p.D <= 64)
    return few ? launch_fwd<T, 64, 1>(p, dtype, dev, sms, parts, workspace, st) : launch_fwd<T, 64, 2>(p, dtype, dev, sms, 1, nullptr, st);
  return few ? launch_fwd<T, 128, 1>(p, dtype, dev, sms, parts, workspace, st) : launch_fwd<T, 128, 2>(p, dtype, dev, sms, 1, nullptr, st);
}

}  // namespace

size_t packed_mma_fwd_bytes(const PackedParams& p, int sms) {
  const int parts = few_rows(p, sms) ? key_parts(p, sms) : 1;
  return parts > 1 ? static_cast<size_t>(p.H) * parts * p.total_q * (p.D + 2) * 4 : 0;
}

int packed_mma_fwd(const PackedParams& p, int dtype, int dev, int sms, void* workspace, cudaStream_t st) {
  return dtype == GW_BF16 ? choose_fwd<__nv_bfloat16>(p, dtype, dev, sms, workspace, st) : choose_fwd<__half>(p, dtype, dev, sms, workspace, st);
}

}  // namespace gw
