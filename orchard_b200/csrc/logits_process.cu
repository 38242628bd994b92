// Penalties for repeated tokens, sparse biases and grammar masks on a batch of logits rows, in
// one pass over the logits.
//
// For the token with global id v = base + i of row m (fp32 arithmetic, one rounding on store):
//   seen(v): v occurs in history[m][0 .. hist_len);  c(v): its count in [gen_start, hist_len)
//   l = seen ? (l > 0 ? l / repetition : l * repetition) : l
//   l -= frequency * c + (c > 0 ? presence : 0)
//   l += the row's bias for v (the last one listed)
//   l = -inf where the row's mask has bit v clear
//
// Bound by memory: every logit is read and written once. A CTA takes a slice of one row's
// vocabulary; it counts the row's history into a table of the slice in shared memory (integer
// atomics: the result has no order) and streams the slice past it.
#include <algorithm>

#include "orch_common.cuh"

namespace orch {

namespace {

constexpr int kLpThreads = 256;
constexpr int kLpMaxSlice = 8192;
constexpr uint32_t kLpSeen = 0x80000000u;  // top bit of a table word: seen; below it the count

struct LpArgs {
  const void* in;
  void* out;
  int M, V, ld, base;
  const int* hist;
  int hist_ld;
  const int* hist_len;
  const int* gen_start;
  const float* pen;
  const int* bias_ids;
  const float* bias_vals;
  const int* bias_off;
  int num_bias;
  const uint32_t* masks;
  int mask_words, num_masks;
  const int* mask_rows;
  int slice;
  uint32_t* check;
};

template <typename T>
__global__ void __launch_bounds__(kLpThreads) logits_process_kernel(const LpArgs a) {
  extern __shared__ uint32_t lp_tab[];  // [slice] seen and counts, then [slice] bias entries
  pdl_trigger();
  pdl_wait();
  const int m = blockIdx.y, i0 = blockIdx.x * a.slice, n = min(a.slice, a.V - i0), tid = threadIdx.x;
  const int hlen = a.hist ? a.hist_len[m] : 0, g0 = a.hist && a.gen_start ? a.gen_start[m] : 0;
  const int b0 = a.bias_ids ? a.bias_off[m] : 0, b1 = a.bias_ids ? a.bias_off[m + 1] : 0;
  const int mr = a.masks ? a.mask_rows[m] : -1;
  if (hlen < 0 || hlen > a.hist_ld || b0 < 0 || b1 < b0 || b1 > a.num_bias || mr >= a.num_masks) {
    if (tid == 0) atomicOr(a.check, 16u);
    return;
  }
  const bool pen = a.pen != nullptr && hlen > 0, bias = b1 > b0;
  uint32_t* btab = lp_tab + a.slice;
  if (pen || bias) {
    for (int i = tid; i < n; i += kLpThreads) {
      lp_tab[i] = 0u;
      if (bias) btab[i] = 0u;
    }
    __syncthreads();
    const int lo = a.base + i0;
    if (pen) {
      const int* h = a.hist + (size_t)m * a.hist_ld;
      for (int j = tid; j < hlen; j += kLpThreads) {
        const int v = h[j];
        if (v >= lo && v - lo < n) {
          atomicOr(&lp_tab[v - lo], kLpSeen);
          if (j >= g0) atomicAdd(&lp_tab[v - lo], 1u);
        }
      }
    }
    for (int j = b0 + tid; j < b1; j += kLpThreads) {
      const int v = a.bias_ids[j];
      if (v >= lo && v - lo < n) atomicMax(&btab[v - lo], (uint32_t)(j - b0 + 1));
    }
    __syncthreads();
  }
  const float rep = pen ? a.pen[3 * m] : 1.f, pres = pen ? a.pen[3 * m + 1] : 0.f, freq = pen ? a.pen[3 * m + 2] : 0.f;
  const uint32_t* mask = mr >= 0 ? a.masks + (size_t)mr * a.mask_words : nullptr;
  const T* in = static_cast<const T*>(a.in) + (size_t)m * a.ld + i0;
  T* out = static_cast<T*>(a.out) + (size_t)m * a.ld + i0;
  for (int i = tid; i < n; i += kLpThreads) {
    float l = to_f32(in[i]);
    if (pen) {
      const uint32_t t = lp_tab[i];
      if (t != 0u) {
        l = l > 0.f ? l / rep : l * rep;
        const uint32_t c = t & ~kLpSeen;
        if (c != 0u) l -= fmaf(freq, (float)c, pres);
      }
    }
    if (bias) {
      const uint32_t t = btab[i];
      if (t != 0u) l += a.bias_vals[b0 + t - 1];
    }
    if (mask != nullptr) {
      const uint32_t v = (uint32_t)(a.base + i0 + i);
      const uint32_t w = v >> 5;
      if (!((w < (uint32_t)a.mask_words ? mask[w] : 0u) >> (v & 31u) & 1u)) l = -INFINITY;
    }
    out[i] = from_f32<T>(l);
  }
}

}  // namespace

}  // namespace orch

using namespace orch;

// The reference samples from the logits as they are (orchard/model.py:244-252).
extern "C" int orch_logits_process(const void* logits, void* out, int dt, uint32_t M, uint32_t V, uint32_t ld,
                                   uint32_t base, const int32_t* history, uint32_t history_ld, const int32_t* hist_len,
                                   const int32_t* gen_start, const float* penalties, const int32_t* bias_ids,
                                   const float* bias_vals, const int32_t* bias_off, uint32_t num_bias,
                                   const uint32_t* masks, uint32_t mask_words, uint32_t num_masks,
                                   const int32_t* mask_rows, void* stream) {
  if (M == 0) return ORCH_OK;
  ORCH_REQUIRE(logits && out && V > 0, "logits_process: null pointer or empty vocabulary");
  ORCH_REQUIRE(dt == ORCH_F32 || dt == ORCH_F16, "logits_process: bad dtype");
  ORCH_REQUIRE(ld >= V && (uint64_t)base + V <= 0x7fffffffu, "logits_process: row stride below V, or ids out of range");
  ORCH_REQUIRE((history == nullptr) == (penalties == nullptr) && (!history || (hist_len && history_ld <= 0x7fffffffu)),
               "logits_process: penalties need history and hist_len (and history penalties)");
  ORCH_REQUIRE(!bias_ids || (bias_vals && bias_off && num_bias <= 0x7fffffffu),
               "logits_process: bias_ids need bias_vals and bias_off");
  ORCH_REQUIRE(!masks || (mask_rows && mask_words > 0 && mask_words <= 0x4000000u && num_masks <= 0x7fffffffu),
               "logits_process: masks need mask_rows and mask_words");
  ORCH_REQUIRE(M <= 65535, "logits_process: at most 65,535 rows");
  LpArgs a;
  a.in = logits;
  a.out = out;
  a.M = (int)M;
  a.V = (int)V;
  a.ld = (int)ld;
  a.base = (int)base;
  a.hist = history;
  a.hist_ld = (int)history_ld;
  a.hist_len = hist_len;
  a.gen_start = gen_start;
  a.pen = penalties;
  a.bias_ids = bias_ids;
  a.bias_vals = bias_vals;
  a.bias_off = bias_off;
  a.num_bias = bias_ids ? (int)num_bias : 0;
  a.masks = masks;
  a.mask_words = (int)mask_words;
  a.num_masks = (int)num_masks;
  a.mask_rows = mask_rows;
  // slices of whole mask words, enough of them for two CTAs per SM
  const uint64_t per = ((uint64_t)M * V + 2 * num_sms() - 1) / (2 * num_sms());
  a.slice = (int)(std::min<uint64_t>(std::max<uint64_t>(per, 512), kLpMaxSlice) + 31) / 32 * 32;
  ORCH_CHECK_WORD(a.check);
  const dim3 grid((V + a.slice - 1) / a.slice, M), none(0, 0, 0);
  const size_t smem = (size_t)a.slice * 4 * (bias_ids ? 2 : history ? 1 : 0);
  static bool attr_done[64] = {};
  const int dev = device_index();
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    ORCH_CUDA(cudaFuncSetAttribute(logits_process_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kLpMaxSlice * 4));
    ORCH_CUDA(cudaFuncSetAttribute(logits_process_kernel<__half>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kLpMaxSlice * 4));
    attr_done[dev] = true;
  }
  if (dt == ORCH_F32)
    ORCH_CUDA(launch_k(logits_process_kernel<float>, grid, dim3(kLpThreads), smem, as_stream(stream), none, a));
  else
    ORCH_CUDA(launch_k(logits_process_kernel<__half>, grid, dim3(kLpThreads), smem, as_stream(stream), none, a));
  return check_launch("logits_process");
}
