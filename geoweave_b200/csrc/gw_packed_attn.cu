// C entry points of the attention over packed sequences: argument checks and the choice of kernel.
#include "gw_packed.cuh"

using namespace gw;

namespace {

int check_packed(const PackedParams& p, int dtype, int* dev, DeviceFacts* facts) {
  if (!p.q || !p.k || !p.v || !p.cu_q || !p.cu_k || p.nseq < 0 || p.total_q < 0 || p.total_k < 0) return GW_ERR_INVALID_ARG;
  if (p.H <= 0 || p.Hk <= 0 || p.H % p.Hk != 0 || p.D <= 0) return GW_ERR_INVALID_ARG;
  if (!(p.scale > 0.f) || !(p.scale * kLog2e <= 3.4028234e38f)) return GW_ERR_INVALID_ARG;  // the kernels multiply with scale log2 e
  if (dtype != GW_F32 && dtype != GW_BF16 && dtype != GW_F16) return GW_ERR_UNSUPPORTED;
  if (p.D > 128 || p.D % 8 != 0 || p.H > 65535 || p.total_q > 0x7fffff00 || p.total_k > 0x7fffff00 || p.nseq > 0xffffff)
    return GW_ERR_UNSUPPORTED;
  const int64_t es = static_cast<int64_t>(dtype_size(dtype));
  for (const void* t : {p.q, p.k, p.v, static_cast<const void*>(p.o), static_cast<const void*>(p.o_low)})
    if (!aligned16(t)) return GW_ERR_INVALID_ARG;
  for (const void* t : {static_cast<const void*>(p.cu_q), static_cast<const void*>(p.cu_k), static_cast<const void*>(p.lse),
                        static_cast<const void*>(p.delta), static_cast<const void*>(p.status)})
    if (reinterpret_cast<uintptr_t>(t) % 4 != 0) return GW_ERR_INVALID_ARG;
  for (const int64_t s : {p.qs[0], p.qs[1], p.ks[0], p.ks[1], p.vs[0], p.vs[1]})
    if (s <= 0 || s * es % 16 != 0) return GW_ERR_INVALID_ARG;
  const int rc = device_facts(dev, facts);
  if (rc != GW_OK) return rc;
  return facts->cc_major == 10 ? GW_OK : GW_ERR_NO_SM100;
}

PackedParams make_params(const void* q, const void* k, const void* v, const int32_t* cu_q, const int32_t* cu_k, int nseq, int64_t total_q,
                         int64_t total_k, int H, int Hk, int D, const int64_t* qs, const int64_t* ks, const int64_t* vs, float scale,
                         int causal, int* status) {
  PackedParams p{};
  p.q = q; p.k = k; p.v = v; p.cu_q = cu_q; p.cu_k = cu_k; p.nseq = nseq; p.total_q = total_q; p.total_k = total_k;
  p.H = H; p.Hk = Hk; p.D = D; p.scale = scale; p.causal = causal ? 1 : 0; p.status = status;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = qs ? qs[i] : 0;
    p.ks[i] = ks ? ks[i] : 0;
    p.vs[i] = vs ? vs[i] : 0;
  }
  return p;
}

}  // namespace

namespace {

// Up to 16 rows (query rows x heads of a group) of a key head: the kernel for single tokens.  16-bit tensors of few rows: the keys
// divided among blocks.  Both leave partial results (fp32) in the workspace.
size_t fwd_bytes(const PackedParams& p, int dtype, int64_t max_q, int sms) {
  if (packed_split_fits(p, max_q)) return packed_split_bytes(p, max_q, sms);
  return dtype == GW_F32 ? 0 : packed_mma_fwd_bytes(p, sms);
}

}  // namespace

extern "C" size_t gw_packed_attn_fwd_workspace_bytes(int dtype, int nseq, int64_t total_q, int64_t total_k, int H, int Hk, int D,
                                                     int64_t max_q) {
  if (nseq < 0 || total_q <= 0 || total_k < 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || D <= 0 || D > 128) return 0;
  PackedParams p{};
  p.nseq = nseq; p.total_q = total_q; p.total_k = total_k; p.H = H; p.Hk = Hk; p.D = D;
  int dev = 0;
  DeviceFacts facts;
  return device_facts(&dev, &facts) == GW_OK ? fwd_bytes(p, dtype, max_q, facts.sms) : 0;
}

extern "C" int gw_packed_attn_fwd(const void* q, const void* k, const void* v, int dtype, const int32_t* cu_q, const int32_t* cu_k, int nseq,
                                  int64_t total_q, int64_t total_k, int H, int Hk, int D, const int64_t* q_strides,
                                  const int64_t* k_strides, const int64_t* v_strides, float scale, int causal, int64_t max_q, void* out,
                                  void* out_low, float* lse, void* workspace, size_t workspace_bytes, int* status_dev, gw_stream_t stream) {
  PackedParams p = make_params(q, k, v, cu_q, cu_k, nseq, total_q, total_k, H, Hk, D, q_strides, k_strides, v_strides, scale, causal, status_dev);
  p.o = out;
  p.o_low = dtype == GW_F32 ? nullptr : out_low;
  p.lse = lse;
  if (!out || max_q < 0) return GW_ERR_INVALID_ARG;
  int dev = 0;
  DeviceFacts facts;
  const int rc = check_packed(p, dtype, &dev, &facts);
  if (rc != GW_OK) return rc;
  if (total_q == 0) return GW_OK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const size_t need = fwd_bytes(p, dtype, max_q, facts.sms);
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return GW_ERR_WORKSPACE;
  if (packed_split_fits(p, max_q)) return packed_split_fwd(p, dtype, max_q, dev, facts.sms, workspace, st);
  return dtype == GW_F32 ? packed_plain_fwd(p, st) : packed_mma_fwd(p, dtype, dev, facts.sms, workspace, st);
}

extern "C" size_t gw_packed_attn_bwd_workspace_bytes(int64_t total_q, int H) {
  return total_q > 0 && H > 0 ? static_cast<size_t>(total_q) * H * 4 : 0;
}

extern "C" int gw_packed_attn_bwd(const void* q, const void* k, const void* v, const void* out, const void* out_low, const float* lse, const void* d_out,
                                  int dtype,
                                  const int32_t* cu_q, const int32_t* cu_k, int nseq, int64_t total_q, int64_t total_k, int H, int Hk,
                                  int D, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                  const int64_t* d_out_strides, float scale, int causal, void* dq, void* dk, void* dv, void* workspace,
                                  size_t workspace_bytes, int* status_dev, gw_stream_t stream) {
  PackedParams p = make_params(q, k, v, cu_q, cu_k, nseq, total_q, total_k, H, Hk, D, q_strides, k_strides, v_strides, scale, causal, status_dev);
  if (!out || !lse || !d_out || !d_out_strides || !dq || !dk != !dv) return GW_ERR_INVALID_ARG;
  p.o = const_cast<void*>(out);
  p.o_low = dtype == GW_F32 ? nullptr : const_cast<void*>(out_low);
  p.lse = const_cast<float*>(lse);
  p.d_o = d_out;
  p.delta = static_cast<float*>(workspace);
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.dos[0] = d_out_strides[0];
  p.dos[1] = d_out_strides[1];
  int dev = 0;
  DeviceFacts facts;
  const int rc = check_packed(p, dtype, &dev, &facts);
  if (rc != GW_OK) return rc;
  for (const void* t : {d_out, static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv)})
    if (!aligned16(t)) return GW_ERR_INVALID_ARG;
  for (const int64_t s : {p.dos[0], p.dos[1]})
    if (s <= 0 || s * static_cast<int64_t>(dtype_size(dtype)) % 16 != 0) return GW_ERR_INVALID_ARG;
  if (total_q > 0 && (!workspace || workspace_bytes < gw_packed_attn_bwd_workspace_bytes(total_q, H))) return GW_ERR_WORKSPACE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == GW_F32 ? packed_plain_bwd(p, st) : packed_mma_bwd(p, dtype, dev, facts.sms, st);
}
