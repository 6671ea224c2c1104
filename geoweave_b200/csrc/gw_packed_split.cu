// Attention over packed sequences for a few query rows per key head (single new tokens): the work is divided along the keys.
//
// At most 16 rows (query rows x heads of a group) share a key head, so the pass is bound by reading k and v once.  A block takes
// one chunk of one sequence's keys for one key head and keeps a running maximum, sum and output per row; a second kernel joins
// the chunks: with (m_i, l_i, o_i) of each, m = max m_i, l = sum l_i 2^(m_i - m), o = sum o_i 2^(m_i - m) / l.
//
// 16-bit operands: each warp walks its share of the keys in steps of 32 (16 for wide heads) with m16n8k16 products; K and V come by
// TMA into a ring of its own, three steps deep (192 KB in flight an SM), so the warps never wait for one another.  The tensor cores
// are idle most of the time (16 rows against 128 lanes would leave tcgen05 nothing to win).
#include "gw_packed_mma.cuh"

namespace gw {
namespace {

constexpr int kRows = 16;        // rows of one key head
constexpr int kSplitThreads = 128;

// A warp's step: 32 keys (16 for wide heads) of K and V, 8 KB; each of the four warps has a ring of three
template <int DP>
struct SplitShape {
  static constexpr int NT = DP == 64 ? 4 : 2;      // n8 tiles of keys a step
  static constexpr int kKeys = 8 * NT;
  static constexpr int kBoxes = DP / 64;           // boxes of 64 columns
  static constexpr int kBox = kKeys * 128;         // bytes
  static constexpr int kStep = 2 * kBoxes * kBox;  // K and V
  static constexpr int kStages = 3;
  static constexpr size_t kSmem = 1024 + static_cast<size_t>(kSplitThreads / 32) * kStages * kStep;
};

// four 8 x 8 matrices of 16-bit values from shared memory, one row address a lane; `trans`: transposed on the way
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_matrices_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

struct SplitParams {
  PackedParams p;
  int chunk;       // keys per block
  int rows;        // rows of a key head that the caller promises: queries x heads of a group
  int64_t slots;   // chunk slots in the workspace
  float* part_o;   // [slots, Hk, rows, D]
  float* part_ml;  // [slots, Hk, rows, 2]: maximum of scale log2 e S, sum
};

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Keys that row r (query r / group of the sequence) may see, counted from the sequence's first key
__device__ __forceinline__ int row_limit(const PackedParams& p, const PackedSeq& s, int r, int group, int rows) {
  if (r >= rows) return 0;
  return p.causal ? min(s.lk, r / group + s.lk - s.lq + 1) : s.lk;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kSplitThreads, 2)
split_mma_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const SplitParams sp) {
  using Shape = SplitShape<DP>;
  constexpr int NT = Shape::NT, NB = Shape::kBoxes, ST = Shape::kStages, STEP = Shape::kKeys, STRIDE = STEP * (kSplitThreads / 32);
  const PackedParams& p = sp.p;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ float red_ml[kSplitThreads / 32][kRows][2];
  __shared__ uint64_t full[kSplitThreads / 32][ST];
  float(*red_o)[kRows][DP] = reinterpret_cast<float(*)[kRows][DP]>(smem);  // behind the last step
  static_assert(sizeof(float) * (kSplitThreads / 32) * kRows * DP <= Shape::kSmem - 1024, "the join fits the rings");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, quad = lane & 3;
  // the key heads of one chunk side by side: a token's heads are neighbours in memory, and are read at about the same time
  const int kv = blockIdx.x % p.Hk, group = p.H / p.Hk;
  const int64_t slot = blockIdx.x / p.Hk;
  let_dependents_launch();
  if (lane == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&full[warp][i], 1);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  __syncwarp();
  PackedSeq s;
  int64_t tiles, end;
  if (!packed_find(p, true, sp.chunk, slot, &s, &tiles, &end)) return;
  const int rows = min(sp.rows, s.lq * group);
  if (rows == 0) return;
  const int k_chunk = s.tile * sp.chunk, k_to = k_chunk + min(sp.chunk, s.lk - k_chunk), k_from = k_chunk + warp * STEP;
  unsigned char* ring = smem + warp * ST * Shape::kStep;
  const int steps = k_from < k_to ? (k_to - k_from + STRIDE - 1) / STRIDE : 0;
  auto fetch = [&](int i) {  // step i of this warp
    if (i < steps && elect_one()) {
      unsigned char* at = ring + i % ST * Shape::kStep;
      mbar_arrive_expect_tx(&full[warp][i % ST], Shape::kStep);
      load_rows<DP, STEP>(at, &tmK, kv, s.k0 + k_from + i * STRIDE, &full[warp][i % ST]);
      load_rows<DP, STEP>(at + NB * Shape::kBox, &tmV, kv, s.k0 + k_from + i * STRIDE, &full[warp][i % ST]);
    }
  };
#pragma unroll
  for (int i = 0; i < ST; ++i) fetch(i);

  // Q fragments: rows g and g + 8, columns 16 i + 2 quad, + 1 and + 8, + 9
  uint32_t qa[DP / 16][4];
#pragma unroll
  for (int i = 0; i < DP / 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = g + 8 * (e & 1), col = 16 * i + 8 * (e >> 1) + 2 * quad;
      qa[i][e] = 0;
      if (r < rows && col < p.D)
        qa[i][e] = *reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.q) + (s.q0 + r / group) * p.qs[0] +
                                                      (kv * group + r % group) * p.qs[1] + col);
    }
  const int lim0 = row_limit(p, s, g, group, rows), lim1 = row_limit(p, s, g + 8, group, rows);
  float o[DP / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  const float c = p.scale * kLog2e;
  bool ok = true;

  int it = 0;
  for (; it < steps; ++it) {
    const int k0 = k_from + it * STRIDE;
    unsigned char* at = ring + it % ST * Shape::kStep;
    const uint32_t kt = smem_u32(at), vt = kt + NB * Shape::kBox;
    ok = warp_wait(&full[warp][it % ST], (it / ST) & 1, nullptr);
    if (!ok) break;
    if (k0 + STEP > k_to) {  // the last step: V rows behind the chunk may hold anything, and meet weights of zero
#pragma unroll 1
      for (int b = 0; b < NB; ++b)
        for (int i = (k_to - k0) * 8 + lane; i < STEP * 8; i += 32) *reinterpret_cast<uint4*>(at + (NB + b) * Shape::kBox + i * 16) = make_uint4(0, 0, 0, 0);
      __syncwarp();
    }
    float sc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
      const int row = 8 * t + (lane & 7);
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {  // 32 columns: the four matrices are their 8-column chunks
        uint32_t kf[4];
        const int chunk = (i & 1) * 4 + (lane >> 3);
        load_matrices(kf, kt + (i >> 1) * Shape::kBox + row * 128 + ((chunk ^ (row & 7)) << 4));
        mma_16816(sc[t], qa[2 * i], kf[0], kf[1], T{});
        mma_16816(sc[t], qa[2 * i + 1], kf[2], kf[3], T{});
      }
    }
    float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int key = k0 + 8 * t + 2 * quad + e;
        sc[t][e] = (key < lim0 && key < k_to) ? sc[t][e] * c : -INFINITY;
        sc[t][2 + e] = (key < lim1 && key < k_to) ? sc[t][2 + e] * c : -INFINITY;
        t0 = fmaxf(t0, sc[t][e]);
        t1 = fmaxf(t1, sc[t][2 + e]);
      }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, d));
      t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, d));
    }
    t0 = fmaxf(m0, t0);
    t1 = fmaxf(m1, t1);
    const float b0 = t0 == -INFINITY ? 0.f : t0, b1 = t1 == -INFINITY ? 0.f : t1;
    const float f0 = exp2_fast(m0 - b0), f1 = exp2_fast(m1 - b1);
    m0 = t0;
    m1 = t1;
    l0 *= f0;
    l1 *= f1;
    uint32_t pa[NT][2];  // P in the inputs' type, as the product with V needs it; l is summed before that rounding
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float a = exp2_fast(sc[t][0] - b0), b = exp2_fast(sc[t][1] - b0), d = exp2_fast(sc[t][2] - b1), e = exp2_fast(sc[t][3] - b1);
      l0 += a + b;
      l1 += d + e;
      pa[t][0] = pack_half2<T>(a, b);
      pa[t][1] = pack_half2<T>(d, e);
    }
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) {
      o[i][0] *= f0;
      o[i][1] *= f0;
      o[i][2] *= f1;
      o[i][3] *= f1;
    }
#pragma unroll
    for (int t = 0; t < NT; t += 2) {
      const uint32_t a[4] = {pa[t][0], pa[t][1], pa[t + 1][0], pa[t + 1][1]};
      const int row = 8 * t + (lane & 15);  // matrices: keys 0-7 and 8-15 of this pair of tiles, two 8-column chunks
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        uint32_t vf[4];
        const int chunk = (i & 3) * 2 + (lane >> 4);
        load_matrices_trans(vf, vt + (i >> 2) * Shape::kBox + row * 128 + ((chunk ^ (row & 7)) << 4));
        mma_16816(o[2 * i], a, vf[0], vf[1], T{});
        mma_16816(o[2 * i + 1], a, vf[2], vf[3], T{});
      }
    }
    __syncwarp();  // every lane has read the step
    fetch(it + ST);
  }
  if (!ok) {  // let the copies in flight land before the shared memory is given up
    if (lane == 0) {
      for (int i = it; i < steps && i < it + ST; ++i) mbar_wait_limit(&full[warp][i % ST], (i / ST) & 1, kDrainLimitNs);
      report_status(p.status, GW_ERR_TIMEOUT);
    }
  }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, d);
    l1 += __shfl_xor_sync(0xffffffffu, l1, d);
  }
  __syncthreads();  // the rings are free
  // join the four warps: lane (g, quad) holds rows g and g + 8 of columns 8 i + 2 quad and + 1
  if (quad == 0) {
    red_ml[warp][g][0] = m0;
    red_ml[warp][g][1] = l0;
    red_ml[warp][g + 8][0] = m1;
    red_ml[warp][g + 8][1] = l1;
  }
#pragma unroll
  for (int i = 0; i < DP / 8; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      red_o[warp][g][8 * i + 2 * quad + e] = o[i][e];
      red_o[warp][g + 8][8 * i + 2 * quad + e] = o[i][2 + e];
    }
  __syncthreads();
  const int64_t at = (slot * p.Hk + kv) * sp.rows;
  for (int i = threadIdx.x; i < rows * p.D; i += kSplitThreads) {
    const int r = i / p.D, col = i % p.D;
    float m = red_ml[0][r][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = fmaxf(m, red_ml[w][r][0]);
    const float base = m == -INFINITY ? 0.f : m;
    float acc = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2f(red_ml[w][r][0] - base);
      acc = fmaf(red_o[w][r][col], f, acc);
      l = fmaf(red_ml[w][r][1], f, l);
    }
    sp.part_o[(at + r) * p.D + col] = acc;
    if (col == 0) {
      sp.part_ml[(at + r) * 2] = m;
      sp.part_ml[(at + r) * 2 + 1] = l;
    }
  }
}

// A block joins the chunks of one row (blockIdx.z) of one sequence and key head (blocks x < nseq): its threads share the chunks in
// groups of D / 4, each thread four columns.  Blocks x = nseq clear the rows behind the last sequence.  Sequences with more rows
// than the caller promised are reported.
template <typename T>
__global__ void __launch_bounds__(kSplitThreads) split_join_kernel(const SplitParams sp, const int max_q) {
  const PackedParams& p = sp.p;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kv = blockIdx.y, group = p.H / p.Hk, b = blockIdx.x, r = blockIdx.z;
  if (b == p.nseq) {
    wait_for_predecessor();  // every block: the kernel must not end before the chunks do
    if (r > 0) return;
    if (kv == 0 && warp == 0) packed_check(p);
    const int64_t end = p.nseq > 0 ? packed_border(p.cu_q, p.nseq, p.total_q) : 0;
    for (int h = kv * group; h < (kv + 1) * group; ++h) packed_zero_rows<T>(p.o, p.lse, end, p.total_q, p.H, h, p.D, 0, 1, blockDim.x);
    return;
  }
  __shared__ float red[kSplitThreads / 32];
  __shared__ float4 acc_s[kSplitThreads];
  __shared__ float l_s[kSplitThreads];
  const int q0 = packed_border(p.cu_q, b, p.total_q), q1 = packed_border(p.cu_q, b + 1, p.total_q);
  const int k0 = packed_border(p.cu_k, b, p.total_k), k1 = packed_border(p.cu_k, b + 1, p.total_k);
  const int lq = max(0, q1 - q0), lk = max(0, k1 - k0);
  if (lq > max_q && threadIdx.x == 0) report_status(p.status, GW_ERR_INVALID_ARG);
  if (r >= min(lq, max_q) * group) {
    wait_for_predecessor();
    return;
  }
  const int64_t before = packed_slot(p, true, sp.chunk, b);  // the sequence's first chunk
  wait_for_predecessor();
  const int64_t left = sp.slots - before;
  const int chunks = static_cast<int>(min((static_cast<int64_t>(lk) + sp.chunk - 1) / sp.chunk, left < 0 ? 0 : left));
  const int64_t row0 = (before * p.Hk + kv) * sp.rows + r, step = static_cast<int64_t>(p.Hk) * sp.rows;  // partial rows of the chunks

  float m = -INFINITY;
  for (int n = threadIdx.x; n < chunks; n += kSplitThreads) m = fmaxf(m, sp.part_ml[(row0 + n * step) * 2]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (lane == 0) red[warp] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float base = m == -INFINITY ? 0.f : m;

  const int cols = p.D / 4, groups = kSplitThreads / cols, mine = threadIdx.x / cols, col = threadIdx.x % cols;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  if (mine < groups) {
#pragma unroll 4
    for (int n = mine; n < chunks; n += groups) {
      const int64_t at = row0 + n * step;
      const float2 ml = *reinterpret_cast<const float2*>(sp.part_ml + at * 2);
      const float4 o = *reinterpret_cast<const float4*>(sp.part_o + at * p.D + 4 * col);
      const float f = exp2f(ml.x - base);
      l = fmaf(ml.y, f, l);
      acc.x = fmaf(o.x, f, acc.x);
      acc.y = fmaf(o.y, f, acc.y);
      acc.z = fmaf(o.z, f, acc.z);
      acc.w = fmaf(o.w, f, acc.w);
    }
  }
  acc_s[threadIdx.x] = acc;
  l_s[threadIdx.x] = l;
  __syncthreads();
  if (mine > 0) return;
  for (int i = 1; i < groups; ++i) {  // in a fixed order
    const float4 o = acc_s[threadIdx.x + i * cols];
    acc.x += o.x;
    acc.y += o.y;
    acc.z += o.z;
    acc.w += o.w;
    l += l_s[threadIdx.x + i * cols];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t token = q0 + r / group;
  const int head = kv * group + r % group;
  const int64_t at = (token * p.H + head) * p.D + 4 * col;
  const float v[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = l == 0.f ? 0.f : v[i];
    const T rounded = from_float<T>(x);
    static_cast<T*>(p.o)[at + i] = rounded;
    if (p.o_low != nullptr) static_cast<T*>(p.o_low)[at + i] = from_float<T>(x - to_float(rounded));
  }
  if (col == 0 && p.lse != nullptr) p.lse[head * p.total_q + token] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <typename T, int DP>
int launch_split_mma(const SplitParams& sp, int dtype, dim3 grid, int dev, cudaStream_t st) {
  const PackedParams& p = sp.p;
  CUtensorMap mk, mv;
  GW_CUDA_TRY(cudaSetDevice(dev));  // a thread that has launched nothing yet has no context to encode tensor maps in
  int rc = make_token_map(&mk, p.k, dtype, p.total_k, p.Hk, p.D, p.ks[0], p.ks[1], SplitShape<DP>::kKeys);
  if (rc == GW_OK) rc = make_token_map(&mv, p.v, dtype, p.total_k, p.Hk, p.D, p.vs[0], p.vs[1], SplitShape<DP>::kKeys);
  static OncePerDevice once;
  if (rc == GW_OK) rc = ensure_dynamic_smem(split_mma_kernel<T, DP>, SplitShape<DP>::kSmem, once, dev);
  if (rc != GW_OK) return rc;
  split_mma_kernel<T, DP><<<grid, kSplitThreads, SplitShape<DP>::kSmem, st>>>(mk, mv, sp);
  return GW_OK;
}

template <typename T>
int launch_split(const SplitParams& sp, int max_q, int dtype, int dev, cudaStream_t st) {
  if (sp.slots * sp.p.Hk > 0x7fffffff) return GW_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(sp.slots * sp.p.Hk));
  int rc;
  if constexpr (sizeof(T) == 2)
    rc = sp.p.D <= 64 ? launch_split_mma<T, 64>(sp, dtype, grid, dev, st) : launch_split_mma<T, 128>(sp, dtype, grid, dev, st);
  else
    rc = packed_plain_split(sp.p, sp.chunk, sp.rows, sp.slots, sp.part_o, sp.part_ml, st);
  if (rc != GW_OK) return rc;
  GW_LAUNCH_CHECK();
  // the join may be launched while the last chunks still run: it reads the borders, then waits for them
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sp.p.nseq + 1, sp.p.Hk, sp.rows);
  cfg.blockDim = dim3(kSplitThreads);
  cfg.stream = st;
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  GW_CUDA_TRY(cudaLaunchKernelEx(&cfg, split_join_kernel<T>, sp, max_q));
  GW_LAUNCH_CHECK();
  return GW_OK;
}

// Chunks of a size that gives every SM about four blocks, two at a time: with eight the fixed cost of a block shows (24 caches of 129 to
// 33 312 keys, 4 key heads: 49 us against 45; one cache of 33 312 keys, 16 key heads: 47 against 41), with two the uneven ends of ragged
// caches do (16 key heads: 131 against 121).  No shorter than two steps of a block's warps.
int chunk_keys(int64_t total_k, int Hk, int sms) {
  const int64_t want = total_k * Hk / (4 * static_cast<int64_t>(sms));
  const int64_t c = (want + 127) / 128 * 128;
  return static_cast<int>(c < 256 ? 256 : c > (1 << 20) ? (1 << 20) : c);
}

int64_t split_slots(const PackedParams& p, int chunk) { return p.total_k / chunk + p.nseq + 1; }

}  // namespace

bool packed_split_fits(const PackedParams& p, int64_t max_q) {
  return max_q > 0 && max_q <= kRows / (p.H / p.Hk) && p.Hk <= 65535;  // no product: the bound may be any 64-bit number
}

size_t packed_split_bytes(const PackedParams& p, int64_t max_q, int sms) {
  return static_cast<size_t>(split_slots(p, chunk_keys(p.total_k, p.Hk, sms))) * p.H * max_q * (p.D + 2) * 4;
}

int packed_split_fwd(const PackedParams& p, int dtype, int64_t max_q, int dev, int sms, void* workspace, cudaStream_t st) {
  SplitParams sp;
  sp.p = p;
  sp.chunk = chunk_keys(p.total_k, p.Hk, sms);
  sp.rows = static_cast<int>(max_q) * (p.H / p.Hk);
  sp.slots = split_slots(p, sp.chunk);
  sp.part_o = static_cast<float*>(workspace);
  sp.part_ml = sp.part_o + sp.slots * p.Hk * sp.rows * p.D;
  const int most = static_cast<int>(max_q);
  if (dtype == GW_F32) return launch_split<float>(sp, most, dtype, dev, st);
  if (dtype == GW_BF16) return launch_split<__nv_bfloat16>(sp, most, dtype, dev, st);
  return launch_split<__half>(sp, most, dtype, dev, st);
}

}  // namespace gw
