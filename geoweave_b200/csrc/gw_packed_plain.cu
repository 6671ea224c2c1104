// Attention over packed sequences on the plain arithmetic units, forward and backward, any head dim up to 128.
//
//   S = scale * q k^T over the allowed pairs,  P = softmax(S),  o = P v,  lse = log sum exp S
//   D = rowsum(d_o * o),  dP = d_o v^T,  dS = P * (dP - D) * scale,  dq = dS k,  dk = sum_heads dS^T q,  dv = sum_heads P^T d_o
//
// fp32 end to end: every product is an fp32 FMA, so this is the path of fp32 tensors, whose 24-bit operands the tensor cores
// would round.  A block of 256 threads owns 64 rows and walks the other side in tiles of 64; a thread holds a 4 x 4 piece of
// each 64 x 64 product and 4 rows x DP/16 columns of each accumulator.  The backward pass is two kernels (one owns query rows
// and makes dq and D, one owns key rows and makes dk and dv), so no sum needs atomics and results do not depend on timing.
#include "gw_packed_mma.cuh"

namespace gw {
namespace {

constexpr int BT = 64;        // rows and columns of a tile
constexpr int NT = 256;       // threads: 16 x 16
constexpr int WP = BT + 4;    // padded row of a 64 x 64 tile in shared memory

// [64 rows][DP + 4] fp32 tile of rows row0.. (rows at or beyond `rows`, columns beyond D: zero), by asynchronous 16-byte copies:
// complete behind tiles_here() and a barrier
template <int DP>
__device__ __forceinline__ void load_tile(float* dst, const void* base, int64_t token0, int rows, int64_t ts, int64_t hs, int head, int D) {
  const float* src = static_cast<const float*>(base) + head * hs + token0 * ts;
#pragma unroll 4
  for (int i = threadIdx.x; i < BT * DP / 4; i += NT) {
    const int r = i / (DP / 4), c = i % (DP / 4) * 4;
    const bool there = r < rows && c < D;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + r * (DP + 4) + c)), "l"(there ? src + r * ts + c : src),
                 "r"(there ? 16 : 0)
                 : "memory");
  }
}
__device__ __forceinline__ void tiles_here() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// acc[i][j] = <a row ty*R+i, b row tx+16*j>: two partial sums each, over the even and the odd columns, so that one packed
// instruction makes both
template <int DP, int R>
__device__ __forceinline__ void dot_tile(float (&acc)[R][4], const float* a, const float* b, int ty, int tx) {
  uint64_t sum[R][4];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = 0;
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    ulonglong2 av[R], bv[4];
#pragma unroll
    for (int i = 0; i < R; ++i) av[i] = *reinterpret_cast<const ulonglong2*>(a + (ty * R + i) * (DP + 4) + d);
#pragma unroll
    for (int j = 0; j < 4; ++j) bv[j] = *reinterpret_cast<const ulonglong2*>(b + (tx + 16 * j) * (DP + 4) + d);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sum[i][j] = fma_f2(av[i].x, bv[j].x, sum[i][j]);
        sum[i][j] = fma_f2(av[i].y, bv[j].y, sum[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float even, odd;
      unpack_f2(sum[i][j], even, odd);
      acc[i][j] = even + odd;
    }
}

// acc[i][c] += sum_k w[ty*R+i][k] * m[k][column c of this thread]; columns tx*4 + 64*(c/4) + c%4, two to a packed value.  The tile's
// 64 products are summed by themselves first: a sum of n products in one go is off by about 2^-24 sqrt(n / 6) of its size, this one by
// sqrt(64 / 6) and sqrt(n / 384) (gradients of a key head under eight over 1348 causal tokens: 1.7e-6 -> 5e-7 of their norm).  A single
// row unrolls all steps: 24 single tokens of 16 heads over 4 against 129 to 33 312 keys 242 us, 255 with four steps at a time.
template <int DP, int R>
__device__ __forceinline__ void accumulate(uint64_t (&acc)[R][DP / 32], const float* w, const float* m, int ty, int tx) {
  uint64_t part[R][DP / 32];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) part[i][c] = 0;
#pragma unroll (R == 1 ? BT / 4 : 4)
  for (int k = 0; k < BT; k += 4) {
    float4 wv[R];
#pragma unroll
    for (int i = 0; i < R; ++i) wv[i] = *reinterpret_cast<const float4*>(w + (ty * R + i) * WP + k);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int c = 0; c < DP / 32; c += 2) {
        const ulonglong2 mv = *reinterpret_cast<const ulonglong2*>(m + (k + kk) * (DP + 4) + tx * 4 + 32 * c);
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const float x = kk == 0 ? wv[i].x : kk == 1 ? wv[i].y : kk == 2 ? wv[i].z : wv[i].w;
          part[i][c] = fma_f2(pack_f2(x, x), mv.x, part[i][c]);
          part[i][c + 1] = fma_f2(pack_f2(x, x), mv.y, part[i][c + 1]);
        }
      }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) acc[i][c] = add_f2(acc[i][c], part[i][c]);
}

template <int DP>
__device__ __forceinline__ void store_rows(void* out, const uint64_t (&acc)[4][DP / 32], const float (&mul)[4], int64_t token0, int rows, int heads,
                                           int head, int D, int ty, int tx) {
  float* dst = static_cast<float*>(out);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty * 4 + i;
    if (r >= rows) continue;
#pragma unroll
    for (int c = 0; c < DP / 32; c += 2) {
      float v[4];
      unpack_f2(acc[i][c], v[0], v[1]);
      unpack_f2(acc[i][c + 1], v[2], v[3]);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = mul[i] == 0.f ? 0.f : v[e] * mul[i];
      const int col = tx * 4 + 32 * c;
      if (col < D) *reinterpret_cast<float4*>(dst + ((token0 + r) * heads + head) * D + col) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
}

__device__ __forceinline__ float reduce16_max(float x) {
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
  return x;
}
__device__ __forceinline__ float reduce16_sum(float x) {
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}

// The block's work; false when it has none (then the rows behind the last sequence have been dealt with).
__device__ __forceinline__ bool block_tile(const PackedParams& p, bool key_side, int head, PackedSeq* s, void* out, void* out2, float* lse) {
  int64_t tiles, end;
  if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0 && threadIdx.x < 32) packed_check(p);
  if (packed_find(p, key_side, BT, blockIdx.x, s, &tiles, &end)) return true;
  const int64_t total = key_side ? p.total_k : p.total_q, parts = gridDim.x - tiles, part = blockIdx.x - tiles;
  const int heads = key_side ? p.Hk : p.H;
  packed_zero_rows<float>(out, lse, end, total, heads, head, p.D, part, parts, blockDim.x);
  if (out2 != nullptr) packed_zero_rows<float>(out2, nullptr, end, total, heads, head, p.D, part, parts, blockDim.x);
  return false;
}

template <int DP>
__global__ void __launch_bounds__(NT) plain_fwd_kernel(const PackedParams p) {
  extern __shared__ float smem[];
  float *qt = smem, *kt = qt + BT * (DP + 4), *vt = kt + BT * (DP + 4), *w = vt + BT * (DP + 4);
  const int head = blockIdx.y, kv = head / (p.H / p.Hk), ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  PackedSeq s;
  if (!block_tile(p, false, head, &s, p.o, nullptr, p.lse)) return;
  const int r0 = s.tile * BT, rows = min(BT, s.lq - r0), off = s.lk - s.lq;
  const int keys = p.causal ? max(0, min(s.lk, r0 + rows + off)) : s.lk;  // keys that the tile's last row sees
  load_tile<DP>(qt, p.q, s.q0 + r0, rows, p.qs[0], p.qs[1], head, p.D);
  float m[4], l[4];
  uint64_t acc[4][DP / 32];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) acc[i][c] = 0;
  }
  const float c2 = p.scale * kLog2e;
  for (int k0 = 0; k0 < keys; k0 += BT) {
    __syncthreads();
    load_tile<DP>(kt, p.k, s.k0 + k0, s.lk - k0, p.ks[0], p.ks[1], kv, p.D);
    load_tile<DP>(vt, p.v, s.k0 + k0, s.lk - k0, p.vs[0], p.vs[1], kv, p.D);
    tiles_here();
    __syncthreads();
    float sc[4][4];
    dot_tile<DP, 4>(sc, qt, kt, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = r0 + ty * 4 + i;
      const int limit = (p.causal ? min(s.lk, row + off + 1) : s.lk) - k0;
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sc[i][j] = (tx + 16 * j < limit) ? sc[i][j] * c2 : -INFINITY;
        top = fmaxf(top, sc[i][j]);
      }
      top = fmaxf(m[i], reduce16_max(top));
      const float base = top == -INFINITY ? 0.f : top;
      const float shrink = exp2f(m[i] - base);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = exp2f(sc[i][j] - base);
        w[(ty * 4 + i) * WP + tx + 16 * j] = e;
        sum += e;
      }
      l[i] = l[i] * shrink + reduce16_sum(sum);
      m[i] = top;
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) acc[i][c] = mul_f2(acc[i][c], pack_f2(shrink, shrink));
    }
    __syncwarp();  // a row's weights are written and read by one warp
    accumulate<DP, 4>(acc, w, vt, ty, tx);
  }
  float mul[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    mul[i] = l[i] == 0.f ? 0.f : 1.f / l[i];
    const int r = ty * 4 + i;
    if (p.lse != nullptr && tx == 0 && r < rows)
      p.lse[head * p.total_q + s.q0 + r0 + r] = l[i] == 0.f ? -INFINITY : (m[i] + log2f(l[i])) * kLn2;
  }
  store_rows<DP>(p.o, acc, mul, s.q0 + r0, rows, p.H, head, p.D, ty, tx);
}

// P of a 4 x 4 piece; rows of the piece are query rows (this kernel's lse per row) or key rows (lse per column)
__device__ __forceinline__ float prob(float s, float c2, float lse) {
  return lse == -INFINITY ? 0.f : exp2f(fmaf(s, c2, -lse * kLog2e));
}

template <int DP>
__global__ void __launch_bounds__(NT, DP == 64 ? 2 : 1) plain_dq_kernel(const PackedParams p) {
  extern __shared__ float smem[];
  float *qt = smem, *dt = qt + BT * (DP + 4), *kt = dt + BT * (DP + 4), *vt = kt + BT * (DP + 4), *w = vt + BT * (DP + 4);
  const int head = blockIdx.y, kv = head / (p.H / p.Hk), ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  PackedSeq s;
  if (!block_tile(p, false, head, &s, p.dq, nullptr, nullptr)) return;
  const int r0 = s.tile * BT, rows = min(BT, s.lq - r0), off = s.lk - s.lq;
  const int keys = p.causal ? max(0, min(s.lk, r0 + rows + off)) : s.lk;
  load_tile<DP>(qt, p.o, s.q0 + r0, rows, static_cast<int64_t>(p.H) * p.D, p.D, head, p.D);
  load_tile<DP>(dt, p.d_o, s.q0 + r0, rows, p.dos[0], p.dos[1], head, p.D);
  tiles_here();
  __syncthreads();
  float lse[4], delta[4];
  uint64_t acc[4][DP / 32];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty * 4 + i;
    float sum = 0.f;
    for (int c = tx; c < DP; c += 16) sum = fmaf(qt[r * (DP + 4) + c], dt[r * (DP + 4) + c], sum);
    delta[i] = reduce16_sum(sum);
    lse[i] = r < rows ? p.lse[head * p.total_q + s.q0 + r0 + r] : -INFINITY;
    if (r < rows && tx == 0) p.delta[head * p.total_q + s.q0 + r0 + r] = delta[i];
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) acc[i][c] = 0;
  }
  __syncthreads();
  load_tile<DP>(qt, p.q, s.q0 + r0, rows, p.qs[0], p.qs[1], head, p.D);
  const float c2 = p.scale * kLog2e;
  for (int k0 = 0; k0 < keys; k0 += BT) {
    __syncthreads();
    load_tile<DP>(kt, p.k, s.k0 + k0, s.lk - k0, p.ks[0], p.ks[1], kv, p.D);
    load_tile<DP>(vt, p.v, s.k0 + k0, s.lk - k0, p.vs[0], p.vs[1], kv, p.D);
    tiles_here();
    __syncthreads();
    float sc[4][4], dp[4][4];
    dot_tile<DP, 4>(sc, qt, kt, ty, tx);
    dot_tile<DP, 4>(dp, dt, vt, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = r0 + ty * 4 + i;
      const int limit = (p.causal ? min(s.lk, row + off + 1) : s.lk) - k0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[(ty * 4 + i) * WP + tx + 16 * j] = (tx + 16 * j < limit) ? prob(sc[i][j], c2, lse[i]) * (dp[i][j] - delta[i]) : 0.f;
    }
    __syncwarp();
    accumulate<DP, 4>(acc, w, kt, ty, tx);
  }
  const float mul[4] = {p.scale, p.scale, p.scale, p.scale};
  store_rows<DP>(p.dq, acc, mul, s.q0 + r0, rows, p.H, head, p.D, ty, tx);
}

template <int DP>
__global__ void __launch_bounds__(NT) plain_dkv_kernel(const PackedParams p) {
  extern __shared__ float smem[];
  float *kt = smem, *vt = kt + BT * (DP + 4), *qt = vt + BT * (DP + 4), *dt = qt + BT * (DP + 4), *w = dt + BT * (DP + 4);
  float* st = w + BT * WP;  // lse, delta of the tile's 64 queries
  const int kv = blockIdx.y, group = p.H / p.Hk, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  PackedSeq s;
  if (!block_tile(p, true, kv, &s, p.dk, p.dv, nullptr)) return;
  const int c0 = s.tile * BT, rows = min(BT, s.lk - c0), off = s.lk - s.lq;
  const int first = p.causal ? max(0, c0 - off) / BT * BT : 0;  // the first query tile that sees one of these keys
  load_tile<DP>(kt, p.k, s.k0 + c0, rows, p.ks[0], p.ks[1], kv, p.D);
  load_tile<DP>(vt, p.v, s.k0 + c0, rows, p.vs[0], p.vs[1], kv, p.D);
  uint64_t ak[4][DP / 32], av[4][DP / 32];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) ak[i][c] = av[i][c] = 0;
  const float c2 = p.scale * kLog2e;
  for (int head = kv * group; head < (kv + 1) * group; ++head)
    for (int r0 = first; r0 < s.lq; r0 += BT) {
      __syncthreads();
      load_tile<DP>(qt, p.q, s.q0 + r0, s.lq - r0, p.qs[0], p.qs[1], head, p.D);
      load_tile<DP>(dt, p.d_o, s.q0 + r0, s.lq - r0, p.dos[0], p.dos[1], head, p.D);
      if (threadIdx.x < 2 * BT) {
        const int r = threadIdx.x & (BT - 1);
        const bool live = r0 + r < s.lq;
        const int64_t at = head * p.total_q + s.q0 + r0 + r;
        st[threadIdx.x] = threadIdx.x < BT ? (live ? p.lse[at] : -INFINITY) : (live ? p.delta[at] : 0.f);
      }
      tiles_here();
      __syncthreads();
      float sc[4][4], dp[4][4];
      dot_tile<DP, 4>(sc, kt, qt, ty, tx);
      dot_tile<DP, 4>(dp, vt, dt, ty, tx);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = c0 + ty * 4 + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = tx + 16 * j;
          const bool seen = !p.causal || key <= r0 + r + off;
          sc[i][j] = seen ? prob(sc[i][j], c2, st[r]) : 0.f;
          dp[i][j] = seen ? sc[i][j] * (dp[i][j] - st[BT + r]) : 0.f;
          w[(ty * 4 + i) * WP + r] = sc[i][j];
        }
      }
      __syncwarp();  // a row's weights are written and read by one warp
      accumulate<DP, 4>(av, w, dt, ty, tx);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) w[(ty * 4 + i) * WP + tx + 16 * j] = dp[i][j];
      __syncwarp();
      accumulate<DP, 4>(ak, w, qt, ty, tx);
    }
  const float mul[4] = {p.scale, p.scale, p.scale, p.scale}, one[4] = {1.f, 1.f, 1.f, 1.f};
  store_rows<DP>(p.dk, ak, mul, s.k0 + c0, rows, p.Hk, kv, p.D, ty, tx);
  store_rows<DP>(p.dv, av, one, s.k0 + c0, rows, p.Hk, kv, p.D, ty, tx);
}

// The forward for at most 16 rows of one key head and one chunk of keys (see gw_packed_split.cu): a thread holds one row.
// The rows come first in the tile's 64 x (DP + 4) place; partial results are joined by the caller.
template <int DP>
__global__ void __launch_bounds__(NT) plain_split_kernel(const PackedParams p, const int chunk, const int max_rows, float* part_o, float* part_ml) {
  extern __shared__ float smem[];
  float *qt = smem, *kt = qt + 16 * (DP + 4), *vt = kt + BT * (DP + 4), *w = vt + BT * (DP + 4);
  const int kv = blockIdx.x % p.Hk, group = p.H / p.Hk, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const int64_t slot = blockIdx.x / p.Hk;
  PackedSeq s;
  int64_t tiles, end;
  if (!packed_find(p, true, chunk, slot, &s, &tiles, &end)) return;
  const int rows = min(max_rows, s.lq * group);
  if (rows == 0) return;
  const int from = s.tile * chunk, to = from + min(chunk, s.lk - from);
  for (int i = threadIdx.x; i < 16 * DP; i += NT) {
    const int r = i / DP, c = i % DP;
    qt[r * (DP + 4) + c] =
        r < rows && c < p.D ? static_cast<const float*>(p.q)[(s.q0 + r / group) * p.qs[0] + (kv * group + r % group) * p.qs[1] + c] : 0.f;
  }
  let_dependents_launch();
  const int limit = ty < rows ? (p.causal ? min(to, ty / group + s.lk - s.lq + 1) : to) : 0;  // keys this row sees
  const float c2 = p.scale * kLog2e;
  float m = -INFINITY, l = 0.f;
  uint64_t acc[1][DP / 32];
#pragma unroll
  for (int c = 0; c < DP / 32; ++c) acc[0][c] = 0;
  for (int k0 = from; k0 < to; k0 += BT) {
    __syncthreads();
    load_tile<DP>(kt, p.k, s.k0 + k0, to - k0, p.ks[0], p.ks[1], kv, p.D);
    load_tile<DP>(vt, p.v, s.k0 + k0, to - k0, p.vs[0], p.vs[1], kv, p.D);
    tiles_here();
    __syncthreads();
    float sc[1][4];
    dot_tile<DP, 1>(sc, qt, kt, ty, tx);
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      sc[0][j] = k0 + tx + 16 * j < limit ? sc[0][j] * c2 : -INFINITY;
      top = fmaxf(top, sc[0][j]);
    }
    top = fmaxf(m, reduce16_max(top));
    const float base = top == -INFINITY ? 0.f : top, shrink = exp2f(m - base);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float e = exp2f(sc[0][j] - base);
      w[ty * WP + tx + 16 * j] = e;
      sum += e;
    }
    l = l * shrink + reduce16_sum(sum);
    m = top;
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) acc[0][c] = mul_f2(acc[0][c], pack_f2(shrink, shrink));
    __syncwarp();  // a row's weights are written and read by one warp
    accumulate<DP, 1>(acc, w, vt, ty, tx);
  }
  if (ty >= rows) return;
  const int64_t at = (slot * p.Hk + kv) * max_rows + ty;
#pragma unroll
  for (int c = 0; c < DP / 32; c += 2) {
    const int col = tx * 4 + 32 * c;
    if (col < p.D) *reinterpret_cast<ulonglong2*>(part_o + at * p.D + col) = make_ulonglong2(acc[0][c], acc[0][c + 1]);
  }
  if (tx == 0) {
    part_ml[at * 2] = m;
    part_ml[at * 2 + 1] = l;
  }
}

template <int DP>
constexpr size_t tiles_bytes(int tiles) { return static_cast<size_t>(tiles) * BT * (DP + 4) * 4 + BT * WP * 4 + 2 * BT * 4; }

template <int DP>
int launch_fwd(const PackedParams& p, cudaStream_t st) {
  int dev = 0;
  GW_CUDA_TRY(cudaGetDevice(&dev));
  static OncePerDevice once;
  const int rc = ensure_dynamic_smem(plain_fwd_kernel<DP>, tiles_bytes<DP>(3), once, dev);
  if (rc != GW_OK) return rc;
  plain_fwd_kernel<DP><<<dim3(static_cast<unsigned>(packed_tile_bound(p.total_q, BT, p.nseq)), p.H), NT, tiles_bytes<DP>(3), st>>>(p);
  GW_LAUNCH_CHECK();
  return GW_OK;
}

template <int DP>
int launch_bwd(const PackedParams& p, cudaStream_t st) {
  int dev = 0;
  GW_CUDA_TRY(cudaGetDevice(&dev));
  static OncePerDevice once_q, once_k;
  int rc = ensure_dynamic_smem(plain_dq_kernel<DP>, tiles_bytes<DP>(4), once_q, dev);
  if (rc != GW_OK) return rc;
  rc = ensure_dynamic_smem(plain_dkv_kernel<DP>, tiles_bytes<DP>(4), once_k, dev);
  if (rc != GW_OK) return rc;
  plain_dq_kernel<DP><<<dim3(static_cast<unsigned>(packed_tile_bound(p.total_q, BT, p.nseq)), p.H), NT, tiles_bytes<DP>(4), st>>>(p);
  GW_LAUNCH_CHECK();
  if (p.dk == nullptr) return GW_OK;  // keys and values without a gradient
  plain_dkv_kernel<DP><<<dim3(static_cast<unsigned>(packed_tile_bound(p.total_k, BT, p.nseq)), p.Hk), NT, tiles_bytes<DP>(4), st>>>(p);
  GW_LAUNCH_CHECK();
  return GW_OK;
}

template <int DP>
int launch_split(const PackedParams& p, int chunk, int max_rows, int64_t slots, float* part_o, float* part_ml, cudaStream_t st) {
  int dev = 0;
  GW_CUDA_TRY(cudaGetDevice(&dev));
  static OncePerDevice once;
  const int rc = ensure_dynamic_smem(plain_split_kernel<DP>, tiles_bytes<DP>(3), once, dev);
  if (rc != GW_OK) return rc;
  plain_split_kernel<DP><<<static_cast<unsigned>(slots * p.Hk), NT, tiles_bytes<DP>(3), st>>>(p, chunk, max_rows, part_o, part_ml);
  GW_LAUNCH_CHECK();
  return GW_OK;
}

}  // namespace

int packed_plain_fwd(const PackedParams& p, cudaStream_t st) { return p.D <= 64 ? launch_fwd<64>(p, st) : launch_fwd<128>(p, st); }
int packed_plain_bwd(const PackedParams& p, cudaStream_t st) { return p.D <= 64 ? launch_bwd<64>(p, st) : launch_bwd<128>(p, st); }
int packed_plain_split(const PackedParams& p, int chunk, int max_rows, int64_t slots, float* part_o, float* part_ml, cudaStream_t st) {
  return p.D <= 64 ? launch_split<64>(p, chunk, max_rows, slots, part_o, part_ml, st) : launch_split<128>(p, chunk, max_rows, slots, part_o, part_ml, st);
}

}  // namespace gw
