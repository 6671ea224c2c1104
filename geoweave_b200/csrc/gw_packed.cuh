// Attention over packed sequences: the problem description shared by its kernels, and how a block finds its work.
//
// Sequences lie back to back along the token axis; cu_q / cu_k (int32 [nseq + 1], on the device) hold their borders.  The
// host never reads them: a grid is launched for the largest number of tiles that the totals allow,
// floor(total / tile) + nseq, plus one, and each block finds its sequence by a warp-wide search over the borders.
// Blocks behind the last tile (one at least) share the rows behind the last sequence, which get zeros.
#pragma once

#include "gw_common.cuh"

namespace gw {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct PackedParams {
  const void *q, *k, *v;
  const int32_t *cu_q, *cu_k;
  int nseq;
  int64_t total_q, total_k;
  int H, Hk, D;
  int64_t qs[2], ks[2], vs[2];  // element strides {token, head}
  float scale;
  int causal;
  void* o;        // [total_q, H, D] contiguous
  void* o_low;    // like o: what rounding o to 16 bits took off, for the backward pass; nullable
  float* lse;     // [H, total_q] natural logarithm, nullable in the forward pass
  // backward
  const void* d_o;
  int64_t dos[2];
  float* delta;   // [H, total_q]: rowsum(d_o * (o + o_low))
  void *dq, *dk, *dv;  // contiguous
  int* status;
};

// One sequence as its tiles see it; every field is in bounds whatever the border arrays hold.
struct PackedSeq {
  int q0, lq, k0, lk;  // first row and length on both sides
  int tile;            // tile number within the sequence
};

__device__ __forceinline__ int packed_border(const int32_t* cu, int i, int64_t total) {
  const int c = cu[i];
  return c < 0 ? 0 : (c > total ? static_cast<int>(total) : c);
}

// Warp-wide: reports border arrays that do not start at zero, decrease or pass the totals.  One warp of a call does it, behind
// its other work.
__device__ __forceinline__ void packed_check(const PackedParams& p) {
  bool bad = false;
  for (int b = threadIdx.x & 31; b < p.nseq; b += 32) {
    const int q0 = p.cu_q[b], q1 = p.cu_q[b + 1], k0 = p.cu_k[b], k1 = p.cu_k[b + 1];
    bad |= q0 < 0 || q1 < q0 || q1 > p.total_q || k0 < 0 || k1 < k0 || k1 > p.total_k || (b == 0 && (q0 != 0 || k0 != 0));
  }
  if (__any_sync(0xffffffffu, bad) && (threadIdx.x & 31) == 0) report_status(p.status, GW_ERR_INVALID_ARG);
}

// The first slot of sequence b's tiles (b = nseq: the first slot behind all of them).  Sequence b has slots for one tile more than fit in front
// of it: floor(border / R) + b rises by at least ceil(length / R) from b to b + 1, so every tile has a slot of its own, some slots stay
// empty, and a slot's sequence is found by a search over the borders instead of a sum over all lengths.
__device__ __forceinline__ int64_t packed_slot(const PackedParams& p, bool key_side, int tile_rows, int b) {
  return packed_border(key_side ? p.cu_k : p.cu_q, b, key_side ? p.total_k : p.total_q) / tile_rows + static_cast<int64_t>(b);
}

// Warp-wide: the tile in `slot` of all sequences' tiles (tile_rows rows each, along the q or the k side).  True when there is one.
// Otherwise *tiles is the first slot behind the last sequence (`slot` may lie in front of it, and be an empty one) and *end
// the row there.  All lanes get the same answers.  32 borders are looked at in a step, so the steps are the logarithm of the number of
// sequences to the base of 32: two for a thousand.
__device__ __forceinline__ bool packed_find(const PackedParams& p, bool key_side, int tile_rows, int64_t slot, PackedSeq* out,
                                            int64_t* tiles, int64_t* end) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.nseq;  // the sequence is one of these
  while (hi - lo > 32) {
    const int step = (hi - lo + 31) / 32, b = lo + lane * step;
    const unsigned here = __ballot_sync(0xffffffffu, lane == 0 || (b < hi && packed_slot(p, key_side, tile_rows, b) <= slot));
    lo += (31 - __clz(here)) * step;
    hi = min(hi, lo + step);
  }
  const int b = lo + lane;
  int q0 = 0, q1 = 0, k0 = 0, k1 = 0;
  if (b < hi) {
    q0 = packed_border(p.cu_q, b, p.total_q);
    q1 = packed_border(p.cu_q, b + 1, p.total_q);
    k0 = packed_border(p.cu_k, b, p.total_k);
    k1 = packed_border(p.cu_k, b + 1, p.total_k);
    q1 = max(q0, q1);
    k1 = max(k0, k1);
  }
  const int64_t at = slot - ((key_side ? k0 : q0) / tile_rows + static_cast<int64_t>(b));
  const unsigned here = __ballot_sync(0xffffffffu, b < hi && at >= 0);
  if (here != 0) {
    const int src = 31 - __clz(here);
    out->q0 = __shfl_sync(0xffffffffu, q0, src);
    out->lq = __shfl_sync(0xffffffffu, q1, src) - out->q0;
    out->k0 = __shfl_sync(0xffffffffu, k0, src);
    out->lk = __shfl_sync(0xffffffffu, k1, src) - out->k0;
    const int64_t tile = __shfl_sync(0xffffffffu, at, src);
    out->tile = static_cast<int>(tile);
    if (tile < (static_cast<int64_t>(key_side ? out->lk : out->lq) + tile_rows - 1) / tile_rows) return true;
  }
  *tiles = p.nseq > 0 ? packed_slot(p, key_side, tile_rows, p.nseq) : 0;
  *end = p.nseq > 0 ? packed_border(key_side ? p.cu_k : p.cu_q, p.nseq, key_side ? p.total_k : p.total_q) : 0;
  return false;
}

// Tiles of a sequence whose work is at least x (in tiles of the other side); the work of a tile is the number of keys (key side:
// queries) that its rows see.  Under a causal mask work grows towards the last query tile and falls from the first key tile.
__device__ __forceinline__ int packed_at_least(const PackedParams& p, bool key_side, int R, int lq, int lk, int x) {
  const int n = ((key_side ? lk : lq) + R - 1) / R, other = key_side ? lq : lk;
  if (x <= 0) return n;
  const int64_t below = static_cast<int64_t>(x - 1) * R;  // work of x tiles: more than this
  if (!p.causal) return other > below ? n : 0;
  if (key_side) {
    if (lq <= below || lk <= below) return 0;
    return min(n, static_cast<int>((lk - below + R - 1) / R));
  }
  if (lk <= below) return 0;
  const int64_t y = below - (lk - lq);  // the tile's last query must lie behind this
  return y < 0 ? n : n - static_cast<int>(y / R);
}

// As packed_find, but tile `rank` in falling order of work, so that blocks which start late have little left to do.  For up to
// kSortedSeqs sequences; with more of them each is a small part of the whole and the order of the arrays serves as well.
constexpr int kSortedSeqs = 64;
__device__ __forceinline__ bool packed_find_sorted(const PackedParams& p, bool key_side, int R, int64_t rank, PackedSeq* out, int64_t* tiles,
                                                   int64_t* end) {
  if (p.nseq > kSortedSeqs) {
    if (!packed_find(p, key_side, R, rank, out, tiles, end)) return false;
    if (p.causal && !key_side) out->tile = (out->lq + R - 1) / R - 1 - out->tile;
    return true;
  }
  const int lane = threadIdx.x & 31;
  constexpr int SETS = kSortedSeqs / 32;
  int q0[SETS], lq[SETS], k0[SETS], lk[SETS], top = 0;
#pragma unroll
  for (int i = 0; i < SETS; ++i) {
    const int b = i * 32 + lane;
    q0[i] = lq[i] = k0[i] = lk[i] = 0;
    if (b < p.nseq) {
      q0[i] = packed_border(p.cu_q, b, p.total_q);
      k0[i] = packed_border(p.cu_k, b, p.total_k);
      lq[i] = max(0, packed_border(p.cu_q, b + 1, p.total_q) - q0[i]);
      lk[i] = max(0, packed_border(p.cu_k, b + 1, p.total_k) - k0[i]);
    }
    top = max(top, ((key_side ? lq[i] : lk[i]) + R - 1) / R);
  }
  top = static_cast<int>(__reduce_max_sync(0xffffffffu, static_cast<unsigned>(top)));
  auto count = [&](int x) {  // totals fit 32 bits: fewer than 2^31 tokens, and each tile holds one at least
    int n = 0;
#pragma unroll
    for (int i = 0; i < SETS; ++i) n += packed_at_least(p, key_side, R, lq[i], lk[i], x);
    return static_cast<int64_t>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(n)));
  };
  const int64_t all = count(0);
  if (rank >= all) {
    *tiles = all;
    *end = p.nseq > 0 ? packed_border(key_side ? p.cu_k : p.cu_q, p.nseq, key_side ? p.total_k : p.total_q) : 0;
    return false;
  }
  int lo = 0, hi = top;  // the largest x with more than `rank` tiles of that much work
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (count(mid) > rank)
      lo = mid;
    else
      hi = mid - 1;
  }
  int64_t left = rank - count(lo + 1);
#pragma unroll
  for (int i = 0; i < SETS; ++i) {
    const int ge = packed_at_least(p, key_side, R, lq[i], lk[i], lo), more = packed_at_least(p, key_side, R, lq[i], lk[i], lo + 1);
    int incl = ge - more;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += up;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    if (left < total) {
      const int src = __ffs(__ballot_sync(0xffffffffu, left < incl)) - 1;
      const int at = static_cast<int>(left) - (incl - (ge - more));
      const int n = ((key_side ? lk[i] : lq[i]) + R - 1) / R;
      out->q0 = __shfl_sync(0xffffffffu, q0[i], src);
      out->lq = __shfl_sync(0xffffffffu, lq[i], src);
      out->k0 = __shfl_sync(0xffffffffu, k0[i], src);
      out->lk = __shfl_sync(0xffffffffu, lk[i], src);
      out->tile = __shfl_sync(0xffffffffu, key_side ? more + at : n - ge + at, src);
      return true;
    }
    left -= total;
  }
  return false;  // not reached: the counts above say that the tile exists
}

// The rows of one head behind the last sequence, shared by the blocks `part` of `parts`, each with its first `threads` threads.  Nothing
// for the blocks of empty slots, whose part is negative.
template <typename T>
__device__ __forceinline__ void packed_zero_rows(void* out, float* lse, int64_t from, int64_t to, int heads, int head, int D, int64_t part,
                                                 int64_t parts, int threads) {
  if (part < 0) return;
  T* dst = static_cast<T*>(out);
  const int64_t n = (to - from) * D;
  for (int64_t i = part * threads + threadIdx.x; i < n; i += parts * threads)
    dst[((from + i / D) * heads + head) * D + i % D] = from_float<T>(0.f);
  if (lse != nullptr)
    for (int64_t i = from + part * threads + threadIdx.x; i < to; i += parts * threads)
      lse[static_cast<int64_t>(head) * to + i] = -INFINITY;
}

// Programmatic launch: the kernel behind this one in the stream may start early / everything in front of this kernel is complete.
__device__ __forceinline__ void let_dependents_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

inline int64_t packed_tile_bound(int64_t total, int tile_rows, int nseq) { return total / tile_rows + nseq + 1; }

// fp32 tensors (gw_packed_plain.cu)
int packed_plain_fwd(const PackedParams& p, cudaStream_t st);
int packed_plain_bwd(const PackedParams& p, cudaStream_t st);
int packed_plain_split(const PackedParams& p, int chunk, int max_rows, int64_t slots, float* part_o, float* part_ml, cudaStream_t st);
// 16-bit tensors (gw_packed_fwd.cu, gw_packed_bwd.cu)
size_t packed_mma_fwd_bytes(const PackedParams& p, int sms);
int packed_mma_fwd(const PackedParams& p, int dtype, int dev, int sms, void* workspace, cudaStream_t st);
int packed_mma_bwd(const PackedParams& p, int dtype, int dev, int sms, cudaStream_t st);
// few query rows, divided along the keys (gw_packed_split.cu)
bool packed_split_fits(const PackedParams& p, int64_t max_q);
size_t packed_split_bytes(const PackedParams& p, int64_t max_q, int sms);
int packed_split_fwd(const PackedParams& p, int dtype, int64_t max_q, int dev, int sms, void* workspace, cudaStream_t st);

}  // namespace gw
