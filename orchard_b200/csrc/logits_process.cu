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
// vocabulary, requests it (16 logits per thread; in wide batches the first half of it) before
// anything else, and while those loads are in flight counts the row's history into a table of the
// slice in shared memory (integer atomics: the result has no order). A slice is as small as keeps
// the grid within one round of CTAs, so that few rows still use many SMs; wide batches take the
// largest slice, two rounds of loads, where the history is read least often (128 rows x 131,072
// with 4,095 ids of history: 37 us, 42 us with slices of one round, 24 us with no control at all;
// sharing the history over a cluster's tables took 93 us, its distributed-shared-memory atomics
// being slow).
#include <algorithm>

#include "orch_common.cuh"

namespace orch {

namespace {

constexpr int kLpThreads = 512;
constexpr int kLpEach = 16;  // logits per thread at most
constexpr int kLpRounds = 2;  // of wide batches: a slice twice as large reads the history half as often
constexpr int kLpMaxSlice = kLpThreads * kLpEach * kLpRounds;
// A table word of the slice. Packed: occurrences that count (15 bits), seen before them (bit 15),
// bias entry + 1 (16 bits). Histories or bias lists too long for that take two words:
// occurrences and seen, and the bias entry.
constexpr int kLpPackedHist = 32767, kLpPackedBias = 65534;
// Ids of a list at most: the loops over it count up to 4 x kLpThreads past its end.
constexpr uint32_t kLpMaxList = 0x7fff0000u;

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
  int slice, pieces;
  uint32_t* check;
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) LpVec {
  T v[VEC];
};

// VEC: logits per load (16 bytes, or one where in and out lie differently). WIDE: two-word table.
template <typename T, int VEC, bool WIDE>
__global__ void __launch_bounds__(kLpThreads, 3) logits_process_kernel(const LpArgs a) {
  constexpr int P = kLpEach / VEC;
  constexpr uint32_t kSeen = WIDE ? 0x80000000u : 0x8000u, kCount = kSeen - 1u;
  extern __shared__ __align__(16) uint32_t lp_tab[];
  pdl_trigger();
  pdl_wait();
  // Slices are cut where 16-byte pieces begin: a row whose first logit lies k elements past such a
  // place is taken as if k elements (never touched) came before it. This CTA has elements [beg, n)
  // from `first` on. (128 rows x 131,071: 37.0 us, 50.6 us with single loads; 64 x 32,000, which
  // has no such row, 7.5 us with the additional indexing and 7.2 us without.)
  const int m = blockIdx.y, tid = threadIdx.x, i0 = blockIdx.x * a.slice;
  const T* row = static_cast<const T*>(a.in) + (size_t)m * a.ld;
  const int k = VEC > 1 ? (int)(((uintptr_t)row & 15) / sizeof(T)) : 0;
  const int beg = max(0, k - i0), n = min(a.slice, a.V + k - i0), first = i0 - k;
  if (n <= 0) return;
  const int hlen = a.hist ? a.hist_len[m] : 0, g0 = a.hist && a.gen_start ? a.gen_start[m] : 0;
  const int b0 = a.bias_ids ? a.bias_off[m] : 0, b1 = a.bias_ids ? a.bias_off[m + 1] : 0;
  const int mr = a.masks ? a.mask_rows[m] : -1;
  const T* in = row + first;
  LpVec<T, VEC> x[P];
  auto load = [&](int r0) {  // this thread's logits of the round that begins at r0
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int i = r0 + (p * kLpThreads + tid) * VEC;
      if (p < a.pieces) {
        if (VEC == 1 || (i >= beg && i + VEC <= n)) {
          if (i < n) x[p] = *reinterpret_cast<const LpVec<T, VEC>*>(in + i);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (i + e >= beg && i + e < n) x[p].v[e] = in[i + e];
        }
      }
    }
  };
  load(0);
  if (hlen < 0 || hlen > a.hist_ld || b0 < 0 || b1 < b0 || b1 > a.num_bias || mr >= a.num_masks) {
    if (tid == 0) atomicOr(a.check, 16u);
    return;
  }
  const bool pen = a.pen != nullptr && hlen > 0, bias = b1 > b0;
  uint32_t* btab = WIDE ? lp_tab + a.slice : lp_tab;
  if (pen || bias) {
    for (int i = tid * 4; i < a.slice * (WIDE ? 2 : 1); i += kLpThreads * 4)
      *reinterpret_cast<uint4*>(lp_tab + i) = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    // ids as unsigned distances from the slice's first: one comparison, none below it passes
    const uint32_t lo = (uint32_t)(a.base + first + beg), un = (uint32_t)(n - beg);
    uint32_t* tab = lp_tab + beg;
    if (bias) {
      for (int j = b0 + tid; j < b1; j += kLpThreads) {
        const uint32_t v = (uint32_t)a.bias_ids[j] - lo;
        if (v < un) atomicMax(&btab[beg + v], (uint32_t)(j - b0 + 1) << (WIDE ? 0 : 16));
      }
      if (!WIDE) __syncthreads();  // the maximum is over words without counts
    }
    if (pen) {
      const int* h = a.hist + (size_t)m * a.hist_ld;
      for (int j0 = tid; j0 < hlen; j0 += 4 * kLpThreads) {
        uint32_t v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = j0 + u * kLpThreads < hlen ? (uint32_t)h[j0 + u * kLpThreads] - lo : un;
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (v[u] < un) {
            if (j0 + u * kLpThreads >= g0)
              atomicAdd(&tab[v[u]], 1u);
            else
              atomicOr(&tab[v[u]], kSeen);
          }
      }
    }
    __syncthreads();
  }
  const float rep = pen ? a.pen[3 * m] : 1.f, pres = pen ? a.pen[3 * m + 1] : 0.f, freq = pen ? a.pen[3 * m + 2] : 0.f;
  const uint32_t* mask = mr >= 0 ? a.masks + (size_t)mr * a.mask_words : nullptr;
  T* out = static_cast<T*>(a.out) + (size_t)m * a.ld + first;
  // one logit whose table words are not all zero
  auto touch = [&](T v, uint32_t t, uint32_t b) {
    float l = to_f32(v);
    const uint32_t c = t & kCount;
    if (t & (kSeen | kCount)) l = l > 0.f ? l / rep : l * rep;
    if (c != 0u) l -= fmaf(freq, (float)c, pres);
    if (b != 0u) l += a.bias_vals[b0 + (int)b - 1];
    return from_f32<T>(l);
  };
  const int span = kLpThreads * VEC * a.pieces;  // logits of a round
#pragma unroll 1
  for (int r0 = 0; r0 < n; r0 += span) {
    if (r0 > 0) load(r0);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int i = r0 + (p * kLpThreads + tid) * VEC;
      if (p >= a.pieces || i >= n) continue;
      if (pen || bias) {
        // most groups of VEC are untouched: their words are looked at together (the table ends
        // on a multiple of VEC, its words past n are zero)
        uint32_t t[VEC], any = 0u;
        if (VEC >= 4) {
#pragma unroll
          for (int e = 0; e < VEC; e += 4) {
            const uint4 w = *reinterpret_cast<const uint4*>(lp_tab + i + e);
            t[e] = w.x, t[(e + 1) % VEC] = w.y, t[(e + 2) % VEC] = w.z, t[(e + 3) % VEC] = w.w;
          }
        } else {
          t[0] = lp_tab[i];
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) any |= t[e] | (WIDE ? btab[i + e] : 0u);
        if (any != 0u) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const uint32_t b = WIDE ? btab[i + e] : t[e] >> 16;
            if ((t[e] | b) != 0u) x[p].v[e] = touch(x[p].v[e], t[e], b);
          }
        }
      }
      if (mask != nullptr) {
        // the mask bits of VEC ids from v0 on: a word, and the next one where they straddle (v0 may
        // lie before id 0: word -1 then has no bits that count)
        const int v0 = a.base + first + i, w = v0 >> 5, s = v0 & 31, nw = a.mask_words;
        const uint32_t lo_w = w >= 0 && w < nw ? mask[w] : 0u, hi_w = s + VEC > 32 && w + 1 < nw ? mask[w + 1] : 0u;
        const uint32_t ok = __funnelshift_r(lo_w, hi_w, s);
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (!(ok >> e & 1u)) x[p].v[e] = from_f32<T>(-INFINITY);
      }
      if (VEC == 1 || (i >= beg && i + VEC <= n)) {
        *reinterpret_cast<LpVec<T, VEC>*>(out + i) = x[p];
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (i + e >= beg && i + e < n) out[i + e] = x[p].v[e];
      }
    }
  }
}

template <typename T, int VEC, bool WIDE>
int lp_launch(LpArgs a, cudaStream_t st) {
  static bool attr_done[64] = {};
  const int dev = device_index();
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    ORCH_CUDA(cudaFuncSetAttribute(logits_process_kernel<T, VEC, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   kLpMaxSlice * 4 * (WIDE ? 2 : 1)));
    attr_done[dev] = true;
  }
  const uint64_t round = 3 * (uint64_t)num_sms(), unit = kLpThreads * VEC;
  const uint64_t span = (uint64_t)a.V + VEC - 1;  // with the elements before a row's first piece
  a.pieces = 1;
  while (a.pieces < kLpEach / VEC && (span + unit * a.pieces - 1) / (unit * a.pieces) * a.M > round) ++a.pieces;
  a.slice = (int)unit * a.pieces * (a.pieces == kLpEach / VEC ? kLpRounds : 1);
  const dim3 grid((unsigned)((span + a.slice - 1) / a.slice), a.M), none(0, 0, 0);
  const size_t smem = a.hist || a.bias_ids ? (size_t)a.slice * 4 * (WIDE ? 2 : 1) : 0;
  ORCH_CUDA(launch_k(logits_process_kernel<T, VEC, WIDE>, grid, dim3(kLpThreads), smem, st, none, a));
  return check_launch("logits_process");
}

template <typename T>
int lp_dispatch(const LpArgs& a, cudaStream_t st) {
  constexpr int V16 = 16 / sizeof(T);
  const bool wide = a.hist_ld > kLpPackedHist || a.num_bias > kLpPackedBias;
  // rows need not begin on 16 bytes, as long as in and out lie alike
  const bool vec = (((uintptr_t)a.in ^ (uintptr_t)a.out) & 15) == 0;
  if (vec) return wide ? lp_launch<T, V16, true>(a, st) : lp_launch<T, V16, false>(a, st);
  return wide ? lp_launch<T, 1, true>(a, st) : lp_launch<T, 1, false>(a, st);
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
  ORCH_REQUIRE(ld >= V && ld <= 0x7fffffffu && (uint64_t)base + V <= 0x7fff0000u,
               "logits_process: row stride below V or too large, or ids out of range");
  ORCH_REQUIRE((history == nullptr) == (penalties == nullptr) && (!history || (hist_len && history_ld <= kLpMaxList)),
               "logits_process: penalties need history and hist_len (and history penalties), or history_ld is too large");
  ORCH_REQUIRE(!bias_ids || (bias_vals && bias_off && num_bias <= kLpMaxList),
               "logits_process: bias_ids need bias_vals and bias_off, or num_bias is too large");
  ORCH_REQUIRE(!masks || (mask_rows && mask_words > 0 && mask_words <= 0x4000000u && num_masks <= 0x7fffffffu),
               "logits_process: masks need mask_rows and mask_words");
  ORCH_REQUIRE(M <= 65535, "logits_process: at most 65,535 rows");
  ORCH_REQUIRE((((uintptr_t)logits | (uintptr_t)out) & (dt == ORCH_F32 ? 3 : 1)) == 0 &&
                   (((uintptr_t)history | (uintptr_t)hist_len | (uintptr_t)gen_start | (uintptr_t)penalties |
                     (uintptr_t)bias_ids | (uintptr_t)bias_vals | (uintptr_t)bias_off | (uintptr_t)masks |
                     (uintptr_t)mask_rows) & 3) == 0,
               "logits_process: buffers must be aligned for their elements");
  LpArgs a;
  a.in = logits;
  a.out = out;
  a.M = (int)M;
  a.V = (int)V;
  a.ld = (int)ld;
  a.base = (int)base;
  a.hist = history;
  a.hist_ld = history ? (int)history_ld : 0;
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
  ORCH_CHECK_WORD(a.check);
  return dt == ORCH_F32 ? lp_dispatch<float>(a, as_stream(stream)) : lp_dispatch<__half>(a, as_stream(stream));
}
