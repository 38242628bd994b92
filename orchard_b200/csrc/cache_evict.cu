// Eviction from the KV cache by accumulated attention weight.
//
// Each (row, K/V head) keeps n = min(len, budget) of its len entries: first the protected ones
// (position > newest position - recent), then by mass, equal masses by the lower index. Attention
// does not depend on the order of the entries (the keys carry their rotation), so the survivors
// are not shifted: those below n stay where they are, and the j-th hole below n takes the j-th
// survivor at or above n. An eviction of a few entries then moves a few rows of K and V instead
// of the whole cache, and no move reads what another writes.
//
// One CTA per (row, K/V head). Masses become unsigned keys in the order of the floats; the
// n-th largest key is found by a radix select, eight bits a pass, over a histogram in shared
// memory; ranks among equal keys and the holes' and survivors' numbers come from counts per
// warp segment and ballots, so the result does not depend on the order of atomics.
#include <algorithm>

#include "orch_common.cuh"

namespace orch {

namespace {

constexpr int kEvThreads = 512;
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kEvMoves = 2048;  // moves listed at a time
constexpr int kEvStaged = 160 * 1024;        // shared memory for bits and keys: 39,000 entries
constexpr uint32_t kEvMaxLen = 1000000;      // a bit per entry still fits

struct EvArgs {
  __half* kc;
  __half* vc;
  const float* mass;
  const int* pos;
  const int* lens;
  const int* slots;
  float* mass_out;
  int* pos_out;
  int* lens_out;
  int M, nkv, hd, max_seq, num_slots, budget;
  uint32_t recent;
  uint32_t* check;
};

// Unsigned keys in the order of the floats: -0 counts as 0, a NaN (1) is below every number.
// Two values stand for entries outside the set that the cut falls into: kEvDrop and kEvKeep.
constexpr uint32_t kEvDrop = 0u, kEvKeep = 0xffffffffu;
__device__ __forceinline__ uint32_t ev_key(float v) {
  if (v != v) return 1u;
  const uint32_t u = __float_as_uint(v + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum of one value per warp over the CTA's earlier warps, and the total. Every thread calls.
__device__ __forceinline__ int ev_before(int v, int* sh, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  if (lane == 0) sh[warp] = v;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kEvWarps; ++w) {
    if (w < warp) before += sh[w];
    total += sh[w];
  }
  return before;
}

// STAGED: the keys stay in shared memory; caches too long for that read mass and position
// again in every pass.
template <bool STAGED>
__global__ void __launch_bounds__(kEvThreads) cache_evict_kernel(const EvArgs a) {
  extern __shared__ uint32_t ev_smem[];  // survivors, a bit per entry; then the keys
  __shared__ int hist[256];
  __shared__ int sh[kEvWarps];
  __shared__ int pick[2];
  __shared__ int hole[kEvMoves], from[kEvMoves];
  pdl_trigger();
  pdl_wait();
  const int kv = blockIdx.x % a.nkv, m = blockIdx.x / a.nkv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = a.slots ? a.slots[m] : m, len = a.lens[m];
  if (slot < 0 || slot >= a.num_slots || len < 0 || len > a.max_seq) {
    if (tid == 0) atomicOr(a.check, slot < 0 || slot >= a.num_slots ? 8u : 2u);
    return;
  }
  int twice = 0;  // an earlier row with this slot takes it; two must not move the same entries
  if (a.slots)
    for (int r = tid; r < m; r += kEvThreads) twice |= a.slots[r] == slot;
  if (__syncthreads_or(twice)) {
    if (tid == 0) atomicOr(a.check, 8u);
    return;
  }
  const int n = min(len, a.budget);
  const size_t base = ((size_t)slot * a.nkv + kv) * a.max_seq;
  const float* mass = a.mass + base;
  const int* pos = a.pos + base;
  float* mass_out = a.mass_out + base;
  int* pos_out = a.pos_out + base;
  if (kv == 0 && tid == 0) a.lens_out[m] = n;
  if (n == len || n == 0) {
    if (mass_out != mass)
      for (int e = tid; e < n; e += kEvThreads) mass_out[e] = mass[e];
    if (pos_out != pos)
      for (int e = tid; e < n; e += kEvThreads) pos_out[e] = pos[e];
    return;
  }

  // protected entries: newer than newest - recent
  int newest = -0x7fffffff - 1;
  for (int e = tid; e < len; e += kEvThreads) newest = max(newest, pos[e]);
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (lane == 0) sh[warp] = newest;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kEvWarps; ++w) newest = max(newest, sh[w]);
  const long long guard = (long long)newest - a.recent;
  int cnt = 0;
  for (int e = tid; e < len; e += kEvThreads) cnt += pos[e] > guard;
  cnt = __reduce_add_sync(0xffffffffu, cnt);
  int guarded;
  ev_before(cnt, sh, guarded);
  // the set that the cut falls into (the protected ones when they alone fill n), and how many
  // of it stay (at least one)
  const bool inner = guarded >= n;
  int want = inner ? n : n - guarded;
  uint32_t* bits = ev_smem;
  const int words = (len + 31) / 32;
  uint32_t* keys = ev_smem + (a.max_seq + 31) / 32;
  auto make = [&](int e) {
    const bool p = pos[e] > guard;
    return p == inner ? ev_key(mass[e]) : p ? kEvKeep : kEvDrop;
  };
  auto key = [&](int e) { return STAGED ? keys[e] : make(e); };
  if (STAGED)
    for (int e = tid; e < len; e += kEvThreads) keys[e] = make(e);

  // radix select: `cut`, the want-th largest key of the set, and how many of its equals stay
  uint32_t cut = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kEvThreads) hist[i] = 0;
    __syncthreads();
    for (int e = tid; e < len; e += kEvThreads) {
      const uint32_t k = key(e);
      if (k == kEvDrop || k == kEvKeep) continue;
      if (shift == 24 || (k >> (shift + 8)) == (cut >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255u], 1);
    }
    __syncthreads();
    if (warp == 0) {  // lane l: bins 255 - 8l .. 248 - 8l, largest first
      int s[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += s[i] = hist[255 - 8 * lane - i];
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      int before = incl - sum;
      if (before < want && want <= incl) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (before < want && want <= before + s[i]) {
            pick[0] = 255 - 8 * lane - i;
            pick[1] = want - before;
          }
          before += s[i];
        }
      }
    }
    __syncthreads();
    cut |= (uint32_t)pick[0] << shift;
    want = pick[1];  // of the keys with this prefix
    __syncthreads();
  }

  // Survivors: keys above the cut, and the first `want` equal to it. Each warp takes a
  // contiguous run of words; ranks are the run's start plus a count of bits.
  const int run = (words + kEvWarps - 1) / kEvWarps;
  const int w0 = min(words, warp * run), w1 = min(words, w0 + run);
  int ties = 0;
  for (int w = w0; w < w1; ++w) {
    const int e = w * 32 + lane;
    ties += __popc(__ballot_sync(0xffffffffu, e < len && key(e) == cut));
  }
  int total;
  int tie = ev_before(ties, sh, total);
  int holes = 0, tails = 0;
  for (int w = w0; w < w1; ++w) {
    const int e = w * 32 + lane;
    const uint32_t k = e < len ? key(e) : kEvDrop;
    const uint32_t eq = __ballot_sync(0xffffffffu, k == cut);
    const bool stay = k > cut || (k == cut && tie + __popc(eq & ((1u << lane) - 1u)) < want);
    tie += __popc(eq);
    const uint32_t b = __ballot_sync(0xffffffffu, stay);
    if (lane == 0) bits[w] = b;
    const uint32_t low = w * 32 + 32 <= n ? 0xffffffffu : w * 32 >= n ? 0u : (1u << (n - w * 32)) - 1u;
    holes += __popc(~b & low);
    tails += __popc(b & ~low);
  }
  int moves;
  const int hole0 = ev_before(holes, sh, total);
  const int tail0 = ev_before(tails, sh, moves);  // as many holes as survivors past n

  const bool apart = mass_out != mass || pos_out != pos;
  if (apart) {  // the survivors that stay in place, before the moved ones
    for (int e = tid; e < n; e += kEvThreads)
      if (bits[e >> 5] >> (e & 31) & 1u) {
        mass_out[e] = mass[e];
        pos_out[e] = pos[e];
      }
  }
  const int pieces = a.hd / 8;  // 16-byte pieces of a K or V row
  uint4* kr = reinterpret_cast<uint4*>(a.kc + base * a.hd);
  uint4* vr = reinterpret_cast<uint4*>(a.vc + base * a.hd);
  for (int at = 0; at < moves; at += kEvMoves) {
    const int count = min(kEvMoves, moves - at);
    __syncthreads();  // bits complete; the lists of the round before are done with
    int h = hole0 - at, t = tail0 - at;
    for (int w = w0; w < w1; ++w) {
      const uint32_t b = bits[w], low = w * 32 + 32 <= n ? 0xffffffffu : w * 32 >= n ? 0u : (1u << (n - w * 32)) - 1u;
      const uint32_t bh = ~b & low, bt = b & ~low, below = (1u << lane) - 1u;
      const int rh = h + __popc(bh & below), rt = t + __popc(bt & below);
      if ((bh >> lane & 1u) && rh >= 0 && rh < count) hole[rh] = w * 32 + lane;
      if ((bt >> lane & 1u) && rt >= 0 && rt < count) from[rt] = w * 32 + lane;
      h += __popc(bh);
      t += __popc(bt);
    }
    __syncthreads();
    for (int i = tid; i < count * pieces; i += kEvThreads) {
      const int j = i / pieces, c = i - j * pieces;
      const size_t s = (size_t)from[j] * pieces + c, d = (size_t)hole[j] * pieces + c;
      const uint4 k4 = kr[s], v4 = vr[s];
      kr[d] = k4;
      vr[d] = v4;
    }
    for (int j = tid; j < count; j += kEvThreads) {
      mass_out[hole[j]] = mass[from[j]];
      pos_out[hole[j]] = pos[from[j]];
    }
  }
}

}  // namespace

}  // namespace orch

using namespace orch;

// No counterpart in the reference, whose host cache keeps every position
// (orchard/model.py:112-124).
extern "C" int orch_cache_evict(void* k_cache, void* v_cache, const float* mass, const int32_t* positions,
                                const int32_t* lens, const int32_t* slots, float* mass_out, int32_t* positions_out,
                                int32_t* lens_out, uint32_t M, uint32_t num_kv_heads, uint32_t head_dim,
                                uint32_t max_seq, uint32_t num_slots, uint32_t budget, uint32_t recent, void* stream) {
  if (M == 0) return ORCH_OK;
  ORCH_REQUIRE(k_cache && v_cache && mass && positions && lens && mass_out && positions_out && lens_out,
               "cache_evict: null pointer");
  ORCH_REQUIRE(num_kv_heads > 0 && max_seq > 0 && num_slots > 0 && num_slots <= 0x7fffffffu, "cache_evict: empty shape");
  ORCH_REQUIRE(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 1024, "cache_evict: head_dim must be a multiple of 8, at most 1024");
  ORCH_REQUIRE((((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0, "cache_evict: caches must be 16-byte aligned");
  ORCH_REQUIRE(lens_out != lens, "cache_evict: lens_out must not be lens (heads read it while others finish)");
  ORCH_REQUIRE((mass_out == mass) == (positions_out == positions),
               "cache_evict: mass and positions are both updated in place, or neither");
  if (max_seq > kEvMaxLen) return fail(ORCH_ERR_UNSUPPORTED, "cache_evict: max_seq above 1,000,000");
  if ((uint64_t)M * num_kv_heads > 0x7fffffffu) return fail(ORCH_ERR_UNSUPPORTED, "cache_evict: too many rows and heads");
  EvArgs a;
  a.kc = static_cast<__half*>(k_cache);
  a.vc = static_cast<__half*>(v_cache);
  a.mass = mass;
  a.pos = positions;
  a.lens = lens;
  a.slots = slots;
  a.mass_out = mass_out;
  a.pos_out = positions_out;
  a.lens_out = lens_out;
  a.M = (int)M;
  a.nkv = (int)num_kv_heads;
  a.hd = (int)head_dim;
  a.max_seq = (int)max_seq;
  a.num_slots = (int)num_slots;
  a.budget = (int)std::min<uint32_t>(budget, max_seq);
  a.recent = recent;
  ORCH_CHECK_WORD(a.check);
  static bool attr_done[64] = {};
  const int dev = device_index();
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    ORCH_CUDA(cudaFuncSetAttribute(cache_evict_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvStaged));
    ORCH_CUDA(cudaFuncSetAttribute(cache_evict_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvStaged));
    attr_done[dev] = true;
  }
  const size_t bits = ((size_t)max_seq + 31) / 32 * 4, staged = bits + (size_t)max_seq * 4;
  const dim3 grid((unsigned)(M * num_kv_heads)), none(0, 0, 0);
  if (staged <= (size_t)kEvStaged)
    ORCH_CUDA(launch_k(cache_evict_kernel<true>, grid, dim3(kEvThreads), staged, as_stream(stream), none, a));
  else
    ORCH_CUDA(launch_k(cache_evict_kernel<false>, grid, dim3(kEvThreads), bits, as_stream(stream), none, a));
  return check_launch("cache_evict");
}
