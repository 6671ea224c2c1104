// Rotary positions with several axes (time, height, width): a head's columns are divided among the axes, axis a owning
// width_a of them side by side; inside an axis column j pairs with column j + width_a / 2 and the pair turns by
// pos[t, a] * f^(-2j / width_a), read from tables of cosines and sines:
//
//   y[j] = x[j] c - x[j + h] s,   y[j + h] = x[j + h] c + x[j] s,   h = width_a / 2
//
// Columns behind the last axis are copied.  A rotation's transpose is the rotation by the opposite angle, so the backward
// pass is the same kernel with s negated.  The reference's two-axis embedding is widths (D/2, D/2)
// (easyvolcap/official_vggt/layers/rope.py:134-188).
//
// Bound by memory: q and k are read once and written once.  A thread owns one piece of the columns (V pairs, or V copied
// columns) of one token and walks the heads, so cosines and sines are loaded once for all heads; V is the widest piece of at
// most 16 bytes that the widths, strides and pointers allow.  Blocks stay and take tokens gridDim apart: 33 312 tokens of 16 + 16
// heads of 64 in bf16, sliced from a projection's output, 58 us a pass among others = 4.7 TB/s (64 with a block for every four tokens; a
// copy of as many contiguous bytes takes 45 us), 61 us alone with cold caches; fp32 5.4 TB/s.  Looked at and dropped: whole
// 16-byte pieces a lane with the partners found through shared memory (104 us: the registers for two angles a column halve
// the occupancy), loads ahead of the position (96 us, the same), other block sizes.  Without the position and angle loads it
// takes 56 us, so they are not the bound.
#include "gw_common.cuh"

namespace gw {
namespace {

constexpr int kAxes = 4;
constexpr int kThreads = 256;
// Blocks an SM, and so registers a thread (33 312 tokens, alone with cold caches): with whole 16-byte pieces the compiler needs more
// (fp32: 93 us with four against 102 with six; bf16, two axes: 53 against 60), with 8-byte ones more threads are better (bf16,
// three axes, 12-column halves: 61 with six against 69 with four).
template <typename T, int V>
constexpr int kBlocksPerSm = sizeof(T) * V >= 16 ? 4 : 6;

struct RotaryParams {
  const void *q, *k;
  void *q_out, *k_out;
  int64_t tokens, per_batch;
  int H, Hk, D, axes;
  int half[kAxes];
  int turned;  // columns that turn
  int64_t qs[3], ks[3];  // element strides {batch, token, head}
  const void* pos;
  int pos64;
  const float *cos_tab, *sin_tab;  // [table_rows, turned / 2]
  int table_rows;
  float sign;
  int head_lanes, tokens_per_block;
  int* status;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Piece {
  T e[V];
};

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, (kBlocksPerSm<T, V>)) rotary_axes_kernel(const RotaryParams p) {
  const int pairs = p.turned / 2 / V, units = pairs + (p.D - p.turned + V - 1) / V;
  const int per_token = units * p.head_lanes;
  const int slot = threadIdx.x / per_token;
  if (slot >= p.tokens_per_block) return;
  const int unit = (threadIdx.x % per_token) % units, lane = (threadIdx.x % per_token) / units;
  using P = Piece<T, V>;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * p.tokens_per_block;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * p.tokens_per_block + slot; t < p.tokens; t += stride) {
    const int64_t b = t / p.per_batch, n = t % p.per_batch;
    const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + n * p.qs[1];
    const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + n * p.ks[1];
    T* qo = static_cast<T*>(p.q_out) + t * p.H * p.D;
    T* ko = static_cast<T*>(p.k_out) + t * p.Hk * p.D;

    if (unit >= pairs) {  // a piece behind the axes
      const int c = p.turned + (unit - pairs) * V;
#pragma unroll 4
      for (int h = lane; h < p.H + p.Hk; h += p.head_lanes) {
        const bool is_q = h < p.H;
        const T* src = is_q ? q + h * p.qs[2] : k + (h - p.H) * p.ks[2];
        T* dst = is_q ? qo + h * p.D : ko + (h - p.H) * p.D;
        *reinterpret_cast<P*>(dst + c) = *reinterpret_cast<const P*>(src + c);
      }
      continue;
    }

    int a = 0, before = 0;  // the axis of this piece, and the angles of the axes in front of it
    while (unit * V >= before + p.half[a]) before += p.half[a++];
    const int lo = unit * V + before, hi = lo + p.half[a];
    const int64_t at = t * p.axes + a;
    int64_t pos = p.pos64 ? static_cast<const int64_t*>(p.pos)[at] : static_cast<const int32_t*>(p.pos)[at];
    if (pos < 0 || pos >= p.table_rows) {  // outside the tables: say so and carry on
      report_status(p.status, GW_ERR_INVALID_ARG);
      pos = 0;
    }
    const Piece<float, V> c = *reinterpret_cast<const Piece<float, V>*>(p.cos_tab + pos * (p.turned / 2) + unit * V);
    Piece<float, V> s = *reinterpret_cast<const Piece<float, V>*>(p.sin_tab + pos * (p.turned / 2) + unit * V);
#pragma unroll
    for (int i = 0; i < V; ++i) s.e[i] *= p.sign;
#pragma unroll 4
    for (int h = lane; h < p.H + p.Hk; h += p.head_lanes) {
      const bool is_q = h < p.H;
      const T* src = is_q ? q + h * p.qs[2] : k + (h - p.H) * p.ks[2];
      T* dst = is_q ? qo + h * p.D : ko + (h - p.H) * p.D;
      P x = *reinterpret_cast<const P*>(src + lo), y = *reinterpret_cast<const P*>(src + hi);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float u = to_float(x.e[i]), w = to_float(y.e[i]);
        x.e[i] = from_float<T>(fmaf(u, c.e[i], -w * s.e[i]));
        y.e[i] = from_float<T>(fmaf(w, c.e[i], u * s.e[i]));
      }
      *reinterpret_cast<P*>(dst + lo) = x;
      *reinterpret_cast<P*>(dst + hi) = y;
    }
  }
}

template <typename T, int V>
int launch(RotaryParams p, int sms, cudaStream_t st) {
  const int units = p.turned / 2 / V + (p.D - p.turned + V - 1) / V;
  const int heads = p.H + p.Hk;
  p.head_lanes = (heads + 3) / 4;  // four heads a thread keep eight loads in flight
  if (p.head_lanes * units > kThreads) p.head_lanes = kThreads / units;
  p.tokens_per_block = kThreads / (units * p.head_lanes);
  const int64_t need = (p.tokens + p.tokens_per_block - 1) / p.tokens_per_block, most = static_cast<int64_t>(sms) * kBlocksPerSm<T, V>;
  const int64_t grid = need < most ? need : most;
  rotary_axes_kernel<T, V><<<static_cast<unsigned>(grid), kThreads, 0, st>>>(p);
  GW_LAUNCH_CHECK();
  return GW_OK;
}

template <typename T>
int dispatch(const RotaryParams& p, int v, int sms, cudaStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (v == 8) return launch<T, 8>(p, sms, st);
  if (v >= 4) return launch<T, 4>(p, sms, st);
  if (v == 2) return launch<T, 2>(p, sms, st);
  return launch<T, 1>(p, sms, st);
}

}  // namespace
}  // namespace gw

using namespace gw;

extern "C" int gw_rotary_axes(const void* q, const void* k, int dtype, int B, int64_t N, int H, int Hk, int D, const int64_t* q_strides,
                              const int64_t* k_strides, const void* pos, int pos_is_64, int axes, const int* widths, const float* cos_tab,
                              const float* sin_tab, int table_rows, int inverse, void* q_out, void* k_out, int* status_dev,
                              gw_stream_t stream) {
  if (!q || !q_strides || !pos || !widths || !cos_tab || !sin_tab || !q_out || (Hk > 0 && (!k || !k_strides || !k_out)))
    return GW_ERR_INVALID_ARG;
  if (B < 0 || N < 0 || H <= 0 || Hk < 0 || D <= 0 || axes <= 0 || table_rows <= 0) return GW_ERR_INVALID_ARG;
  if (axes > kAxes || D > 256) return GW_ERR_UNSUPPORTED;
  if (dtype != GW_F32 && dtype != GW_BF16 && dtype != GW_F16) return GW_ERR_UNSUPPORTED;
  RotaryParams p{};
  int64_t all = 0;  // OR of everything the piece width has to divide, in elements
  for (int a = 0; a < axes; ++a) {
    if (widths[a] <= 0 || widths[a] % 2 != 0) return GW_ERR_INVALID_ARG;
    p.half[a] = widths[a] / 2;
    p.turned += widths[a];
    all |= p.half[a];
  }
  if (p.turned > D) return GW_ERR_INVALID_ARG;
  const size_t es = dtype_size(dtype);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(q_out) |
       reinterpret_cast<uintptr_t>(k_out)) % es != 0 ||
      (reinterpret_cast<uintptr_t>(cos_tab) | reinterpret_cast<uintptr_t>(sin_tab)) % 4 != 0 ||
      reinterpret_cast<uintptr_t>(pos) % (pos_is_64 ? 8 : 4) != 0)
    return GW_ERR_INVALID_ARG;
  if (B == 0 || N == 0) return GW_OK;
  if (static_cast<int64_t>(B) > 0x7fffffffffffll / N) return GW_ERR_UNSUPPORTED;
  p.q = q; p.k = k; p.q_out = q_out; p.k_out = k_out;
  p.tokens = B * N; p.per_batch = N; p.H = H; p.Hk = Hk; p.D = D; p.axes = axes;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = q_strides[i];
    p.ks[i] = Hk > 0 ? k_strides[i] : 0;
    all |= p.qs[i] | p.ks[i];
  }
  p.pos = pos; p.pos64 = pos_is_64; p.cos_tab = cos_tab; p.sin_tab = sin_tab; p.table_rows = table_rows;
  p.sign = inverse ? -1.f : 1.f;
  p.status = status_dev;
  all |= D | (D - p.turned);
  int v = es == 2 ? 8 : 4;
  const uintptr_t data = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) |
                         (Hk > 0 ? reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out) : 0);
  const uintptr_t tabs = reinterpret_cast<uintptr_t>(cos_tab) | reinterpret_cast<uintptr_t>(sin_tab);
  while (v > 1 && (all % v != 0 || data % (v * es) != 0 || tabs % (v * 4) != 0)) v /= 2;  // pieces of the tables: v floats
  int dev = 0;
  DeviceFacts facts;
  const int rc = device_facts(&dev, &facts);
  if (rc != GW_OK) return rc;
  if (facts.cc_major != 10) return GW_ERR_NO_SM100;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == GW_F32) return dispatch<float>(p, v, facts.sms, st);
  if (dtype == GW_BF16) return dispatch<__nv_bfloat16>(p, v, facts.sms, st);
  return dispatch<__half>(p, v, facts.sms, st);
}
