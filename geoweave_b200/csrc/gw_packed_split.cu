// Attention over packed sequences for a few query rows per key head (single new tokens): the work is divided along the keys.
//
// At most 16 rows (query rows x heads of a group) share a key head, so the pass is bound by reading k and v once.  A block takes
// one chunk of one sequence's keys for one key head and keeps a running maximum, sum and output per row; a second kernel joins
// the chunks: with (m_i, l_i, o_i) of each, m = max m_i, l = sum l_i 2^(m_i - m), o = sum o_i 2^(m_i - m) / l.
//
// 16-bit operands: each warp walks the keys in steps of 32 (16 for wide heads) with m16n8k16 products.  Every lane copies the 16-byte
// pieces that its own fragments need into a ring of its own in shared memory, three steps deep (about 190 KB in flight an
// SM), and nothing is synchronised or exchanged: a contraction may run over the columns in any order as
// long as both operands agree, so a lane's piece of a K row is its B fragment as it stands, and Q is gathered to match; for P V
// a lane reads the same eight columns of two neighbouring keys and interleaves them.  The tensor cores are idle most of
// the time here (16 rows against 128 lanes would leave tcgen05 waiting for a layout it needs in shared memory).
#include "gw_packed_mma.cuh"

namespace gw {
namespace {

constexpr int kRows = 16;        // rows of one key head
constexpr int kSplitThreads = 128;

// 16 bytes global -> shared, asynchronously; zeros where there is nothing to read
__device__ __forceinline__ void copy16(uint4* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {  // all but the last N groups of this thread have arrived
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A warp's step: 32 keys (16 for wide heads), K and V pieces of every lane, 8 KB; a ring of three for each of four warps
template <int DP>
struct SplitShape {
  static constexpr int NT = DP == 64 ? 4 : 2;  // n8 tiles of keys a step
  static constexpr int KP = DP / 32;           // 16-byte pieces of a K row in one lane
  static constexpr int CG = DP / 64;           // 16-byte pieces of a V row in one lane
  static constexpr int kPieces = NT * KP + NT * 2 * CG;
  static constexpr int kStages = 3;
  static constexpr size_t kRing = static_cast<size_t>(kSplitThreads) * kPieces * kStages * 16;
};

struct SplitParams {
  PackedParams p;
  int chunk;       // keys per block
  int64_t slots;   // chunk slots in the workspace
  float* part_o;   // [slots, Hk, 16, D]
  float* part_ml;  // [slots, Hk, 16, 2]: maximum of scale log2 e S, sum
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
__global__ void __launch_bounds__(kSplitThreads, 2) split_mma_kernel(const SplitParams sp) {
  using Shape = SplitShape<DP>;
  constexpr int NT = Shape::NT, KP = Shape::KP, CG = Shape::CG, ST = Shape::kStages;
  const PackedParams& p = sp.p;
  extern __shared__ uint4 ring[];  // [stage][piece][thread]; every lane reads what it copied itself, so nothing is synchronised
  __shared__ float red_ml[kSplitThreads / 32][kRows][2];
  float(*red_o)[kRows][DP] = reinterpret_cast<float(*)[kRows][DP]>(ring);  // behind the last step
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, quad = lane & 3;
  // the key heads of one chunk side by side: a token's heads are neighbours in memory, and are read at about the same time
  const int kv = blockIdx.x % p.Hk, group = p.H / p.Hk;
  const int64_t slot = blockIdx.x / p.Hk;
  PackedSeq s;
  int64_t tiles, end;
  if (!packed_find(p, true, sp.chunk, slot, &s, &tiles, &end)) return;
  const int rows = min(kRows, s.lq * group);
  if (rows == 0) return;
  const int k_from = s.tile * sp.chunk, k_to = min(s.lk, k_from + sp.chunk);

  // Q fragments; lane (g, quad) holds columns 32 i + 8 quad .. + 7 of rows g and g + 8
  uint32_t qa[KP][2][4];
#pragma unroll
  for (int i = 0; i < KP; ++i) {
    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
    const int col = 32 * i + 8 * quad;
    if (col < p.D) {
      if (g < rows)
        lo = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (s.q0 + g / group) * p.qs[0] + (kv * group + g % group) * p.qs[1] + col);
      if (g + 8 < rows)
        hi = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (s.q0 + (g + 8) / group) * p.qs[0] +
                                             (kv * group + (g + 8) % group) * p.qs[1] + col);
    }
    qa[i][0][0] = lo.x; qa[i][0][1] = hi.x; qa[i][0][2] = lo.y; qa[i][0][3] = hi.y;
    qa[i][1][0] = lo.z; qa[i][1][1] = hi.z; qa[i][1][2] = lo.w; qa[i][1][3] = hi.w;
  }
  const int lim0 = row_limit(p, s, g, group, rows), lim1 = row_limit(p, s, g + 8, group, rows);
  const T* kb = static_cast<const T*>(p.k) + static_cast<int64_t>(s.k0) * p.ks[0] + kv * p.ks[1];
  const T* vb = static_cast<const T*>(p.v) + static_cast<int64_t>(s.k0) * p.vs[0] + kv * p.vs[1];

  float o[CG * 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
  for (int i = 0; i < CG * 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  const float c = p.scale * kLog2e;
  constexpr int STEP = 8 * NT, STRIDE = STEP * (kSplitThreads / 32);

  auto fetch = [&](int k0, int stage) {
    uint4* at = ring + stage * Shape::kPieces * kSplitThreads + threadIdx.x;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const int key = k0 + 8 * t + g, col = 32 * i + 8 * quad;
        const bool there = key < k_to && col < p.D;
        copy16(at + (t * KP + i) * kSplitThreads, there ? kb + key * p.ks[0] + col : kb, there);
      }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < CG; ++i) {
          const int key = k0 + 8 * t + 2 * quad + e, col = 64 * i + 8 * g;
          const bool there = key < k_to && col < p.D;
          copy16(at + (NT * KP + (t * 2 + e) * CG + i) * kSplitThreads, there ? vb + key * p.vs[0] + col : vb, there);
        }
  };
  int ahead = k_from + warp * STEP, stage = 0;
#pragma unroll
  for (int i = 0; i < ST - 1; ++i, ahead += STRIDE) {
    if (ahead < k_to) fetch(ahead, i);
    copies_commit();
  }
  for (int k0 = k_from + warp * STEP; k0 < k_to; k0 += STRIDE, ahead += STRIDE) {
    copies_wait<ST - 2>();
    uint4 kf[NT][KP], vf[NT][2][CG];
    {
      const uint4* at = ring + stage * Shape::kPieces * kSplitThreads + threadIdx.x;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int i = 0; i < KP; ++i) kf[t][i] = at[(t * KP + i) * kSplitThreads];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < CG; ++i) vf[t][e][i] = at[(NT * KP + (t * 2 + e) * CG + i) * kSplitThreads];
      }
    }
    // the stage that the step before this one has used
    if (ahead < k_to) fetch(ahead, stage == 0 ? ST - 1 : stage - 1);
    copies_commit();
    stage = stage == ST - 1 ? 0 : stage + 1;
    float sc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        mma_16816(sc[t], qa[i][0], kf[t][i].x, kf[t][i].y, T{});
        mma_16816(sc[t], qa[i][1], kf[t][i].z, kf[t][i].w, T{});
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
    uint32_t pa[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float a = exp2_fast(sc[t][0] - b0), b = exp2_fast(sc[t][1] - b0), d = exp2_fast(sc[t][2] - b1), e = exp2_fast(sc[t][3] - b1);
      l0 += a + b;
      l1 += d + e;
      pa[t][0] = pack_half2<T>(a, b);
      pa[t][1] = pack_half2<T>(d, e);
    }
#pragma unroll
    for (int i = 0; i < CG * 8; ++i) {
      o[i][0] *= f0;
      o[i][1] *= f0;
      o[i][2] *= f1;
      o[i][3] *= f1;
    }
#pragma unroll
    for (int t = 0; t < NT; t += 2) {
      const uint32_t a[4] = {pa[t][0], pa[t][1], pa[t + 1][0], pa[t + 1][1]};
#pragma unroll
      for (int i = 0; i < CG; ++i) {
        const uint32_t x[2][4] = {{vf[t][0][i].x, vf[t][0][i].y, vf[t][0][i].z, vf[t][0][i].w}, {vf[t][1][i].x, vf[t][1][i].y, vf[t][1][i].z, vf[t][1][i].w}};
        const uint32_t y[2][4] = {{vf[t + 1][0][i].x, vf[t + 1][0][i].y, vf[t + 1][0][i].z, vf[t + 1][0][i].w},
                                  {vf[t + 1][1][i].x, vf[t + 1][1][i].y, vf[t + 1][1][i].z, vf[t + 1][1][i].w}};
#pragma unroll
        for (int w = 0; w < 4; ++w) {  // columns 64 i + 8 g + 2 w and + 1: n8 tiles 8 i + 2 w and + 1
          mma_16816(o[8 * i + 2 * w], a, __byte_perm(x[0][w], x[1][w], 0x5410), __byte_perm(y[0][w], y[1][w], 0x5410), T{});
          mma_16816(o[8 * i + 2 * w + 1], a, __byte_perm(x[0][w], x[1][w], 0x7632), __byte_perm(y[0][w], y[1][w], 0x7632), T{});
        }
      }
    }
  }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, d);
    l1 += __shfl_xor_sync(0xffffffffu, l1, d);
  }
  copies_wait<0>();
  __syncthreads();  // the ring is free
  // join the four warps.  The accumulator of n8 tile 8 i + j holds, in lane (g, quad), rows g and g + 8 of the tile's columns
  // 2 quad and 2 quad + 1, and the tile's column n stands for column 64 i + 8 n + j of the head
  if (quad == 0) {
    red_ml[warp][g][0] = m0;
    red_ml[warp][g][1] = l0;
    red_ml[warp][g + 8][0] = m1;
    red_ml[warp][g + 8][1] = l1;
  }
#pragma unroll
  for (int i = 0; i < CG; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        red_o[warp][g][64 * i + 8 * (2 * quad + e) + j] = o[8 * i + j][e];
        red_o[warp][g + 8][64 * i + 8 * (2 * quad + e) + j] = o[8 * i + j][2 + e];
      }
  __syncthreads();
  const int64_t at = (slot * p.Hk + kv) * kRows;
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
    if (r > 0) return;
    PackedSeq s;
    int64_t tiles, end;
    packed_find(p, false, 1, static_cast<int64_t>(0x7fffffffffffffff), &s, &tiles, &end);
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
  if (r >= min(lq, max_q) * group) return;
  int64_t before = 0;  // chunks in front of this sequence
  for (int i = lane; i < b; i += 32) {
    const int c0 = packed_border(p.cu_k, i, p.total_k), c1 = packed_border(p.cu_k, i + 1, p.total_k);
    before += (max(0, c1 - c0) + sp.chunk - 1) / sp.chunk;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) before += __shfl_xor_sync(0xffffffffu, before, d);
  const int64_t left = sp.slots - before;
  const int chunks = static_cast<int>(min(static_cast<int64_t>((lk + sp.chunk - 1) / sp.chunk), left < 0 ? 0 : left));
  const int64_t row0 = (before * p.Hk + kv) * kRows + r, step = static_cast<int64_t>(p.Hk) * kRows;  // partial rows of the chunks

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
  T* dst = static_cast<T*>(p.o) + (token * p.H + head) * p.D + 4 * col;
  const float v[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
  for (int i = 0; i < 4; ++i) dst[i] = from_float<T>(l == 0.f ? 0.f : v[i]);
  if (col == 0 && p.lse != nullptr) p.lse[head * p.total_q + token] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <typename T, int DP>
int launch_split_mma(const SplitParams& sp, dim3 grid, int dev, cudaStream_t st) {
  static OncePerDevice once;
  const int rc = ensure_dynamic_smem(split_mma_kernel<T, DP>, SplitShape<DP>::kRing, once, dev);
  if (rc != GW_OK) return rc;
  split_mma_kernel<T, DP><<<grid, kSplitThreads, SplitShape<DP>::kRing, st>>>(sp);
  return GW_OK;
}

template <typename T>
int launch_split(const SplitParams& sp, int max_q, int dev, cudaStream_t st) {
  if (sp.slots * sp.p.Hk > 0x7fffffff) return GW_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(sp.slots * sp.p.Hk));
  int rc;
  if constexpr (sizeof(T) == 2)
    rc = sp.p.D <= 64 ? launch_split_mma<T, 64>(sp, grid, dev, st) : launch_split_mma<T, 128>(sp, grid, dev, st);
  else
    rc = packed_plain_split(sp.p, sp.chunk, sp.slots, sp.part_o, sp.part_ml, st);
  if (rc != GW_OK) return rc;
  GW_LAUNCH_CHECK();
  split_join_kernel<T><<<dim3(sp.p.nseq + 1, sp.p.Hk, max_q * (sp.p.H / sp.p.Hk)), kSplitThreads, 0, st>>>(sp, max_q);
  GW_LAUNCH_CHECK();
  return GW_OK;
}

// Chunks of a size that gives every SM about eight blocks, but no shorter than four steps of a block's warps: below that
// the fixed cost of a block and of the join outweighs what more blocks bring.
int chunk_keys(int64_t total_k, int Hk, int sms) {
  const int64_t want = total_k * Hk / (8 * static_cast<int64_t>(sms));
  const int64_t c = (want + 127) / 128 * 128;
  return static_cast<int>(c < 256 ? 256 : c > (1 << 20) ? (1 << 20) : c);
}

int64_t split_slots(const PackedParams& p, int chunk) { return p.total_k / chunk + p.nseq + 1; }

}  // namespace

bool packed_split_fits(const PackedParams& p, int64_t max_q) {
  return max_q > 0 && max_q * (p.H / p.Hk) <= kRows && p.Hk <= 65535;
}

size_t packed_split_bytes(const PackedParams& p, int sms) {
  return static_cast<size_t>(split_slots(p, chunk_keys(p.total_k, p.Hk, sms))) * p.Hk * kRows * (p.D + 2) * 4;
}

int packed_split_fwd(const PackedParams& p, int dtype, int64_t max_q, int dev, int sms, void* workspace, cudaStream_t st) {
  SplitParams sp;
  sp.p = p;
  sp.chunk = chunk_keys(p.total_k, p.Hk, sms);
  sp.slots = split_slots(p, sp.chunk);
  sp.part_o = static_cast<float*>(workspace);
  sp.part_ml = sp.part_o + sp.slots * p.Hk * kRows * p.D;
  const int most = static_cast<int>(max_q);
  if (dtype == GW_F32) return launch_split<float>(sp, most, dev, st);
  if (dtype == GW_BF16) return launch_split<__nv_bfloat16>(sp, most, dev, st);
  return launch_split<__half>(sp, most, dev, st);
}

}  // namespace gw
