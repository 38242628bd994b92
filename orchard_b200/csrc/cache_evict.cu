// Eviction from the KV cache by accumulated attention weight.
//
// Each (row, K/V head) keeps n = min(len, budget) of its len entries: first the protected ones
// (position > newest position - recent), then by mass, equal masses by the lower index. Attention
// does not depend on the order of the entries (the keys carry their rotation), so the survivors
// are not shifted: those below n stay where they are, and the j-th hole below n takes the j-th
// survivor at or above n. An eviction of a few entries then moves a few rows of K and V instead
// of the whole cache, and no move reads what another writes.
//
// A cluster of CTAs takes one (row, K/V head). Every CTA of it makes the same selection (reading
// 8 bytes per entry, mostly from L2) and moves its share of the rows, so no list crosses CTAs; the
// cluster meets once, before masses and positions are written in place. Masses become unsigned
// keys in the order of the floats; the n-th largest is found by a radix select of 11, 11 and 10
// bits over histograms in shared memory, which ends early when a bucket stays whole. (Eight bits
// would put the masses of one binade or two into one bin and serialise its atomics.) Ranks among
// equal keys and the numbers of holes and survivors come from ballots and bit counts, so the
// result does not depend on the order of atomics.
//
// Bound by memory where many rows move (each is read and written once); a step that drops an
// entry or two is bound by the chain of barriers of the selection.
#include <algorithm>

#include "orch_common.cuh"

namespace orch {

namespace {

constexpr int kEvThreads = 512;
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kEvMoves = 2048;  // moves listed at a time
constexpr int kEvBins = 2048;
constexpr int kEvHeld = 4;  // positions per thread that stay in registers
constexpr int kEvStaged = 192 * 1024;    // shared memory for bits and keys: 46,000 entries
constexpr uint32_t kEvMaxLen = 1000000;  // a bit per entry still fits

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
  int cluster;  // CTAs per (row, K/V head)
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

__device__ __forceinline__ void ev_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void ev_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// STAGED: the keys stay in shared memory; caches too long for that read mass and position
// again in every pass.
template <bool STAGED>
__global__ void __launch_bounds__(kEvThreads, 2) cache_evict_kernel(const EvArgs a) {
  extern __shared__ uint32_t ev_smem[];  // survivors, a bit per entry; then the keys
  __shared__ union {
    __align__(16) int hist[3][kEvBins];
    struct {
      int hole[kEvMoves], from[kEvMoves];
    } list;
  } u;
  __shared__ int sh[2][kEvWarps];
  __shared__ int pick[3];
  pdl_trigger();
  pdl_wait();
  const int part = blockIdx.x % a.cluster, rh = blockIdx.x / a.cluster;
  const int kv = rh % a.nkv, m = rh / a.nkv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slot = a.slots ? a.slots[m] : m, len = a.lens[m];
  if (slot < 0 || slot >= a.num_slots || len < 0 || len > a.max_seq) {  // the whole cluster leaves
    if (tid == 0) atomicOr(a.check, slot < 0 || slot >= a.num_slots ? 8u : 2u);
    return;
  }
  int twice = 0;  // an earlier row with this slot takes it; two must not move the same entries
  if (a.slots)
    for (int r = tid; r < m; r += kEvThreads) twice |= a.slots[r] == slot;
  const int n = min(len, a.budget);
  const size_t base = ((size_t)slot * a.nkv + kv) * a.max_seq;
  const float* mass = a.mass + base;
  const int* pos = a.pos + base;
  float* mass_out = a.mass_out + base;
  int* pos_out = a.pos_out + base;
  uint32_t* bits = ev_smem;
  uint32_t* keys = ev_smem + (a.max_seq + 31) / 32;

  // newest position; the keys of all masses, if they fit
  int held[kEvHeld], newest = -0x7fffffff - 1;
  float mh[kEvHeld];
#pragma unroll
  for (int i = 0; i < kEvHeld; ++i) {
    const int e = tid + i * kEvThreads;
    held[i] = e < len ? pos[e] : newest;
    mh[i] = STAGED && e < len ? mass[e] : 0.f;
  }
  for (int i = tid * 4; i < 3 * kEvBins; i += kEvThreads * 4)
    *reinterpret_cast<int4*>(&u.hist[0][0] + i) = make_int4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < kEvHeld; ++i) {
    const int e = tid + i * kEvThreads;
    newest = max(newest, held[i]);
    if (STAGED && e < len) keys[e] = ev_key(mh[i]);
  }
#pragma unroll 4
  for (int e = tid + kEvHeld * kEvThreads; e < len; e += kEvThreads) {
    newest = max(newest, pos[e]);
    if (STAGED) keys[e] = ev_key(mass[e]);
  }
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (lane == 0) sh[0][warp] = newest;
  if (__syncthreads_or(twice)) {
    if (tid == 0) atomicOr(a.check, 8u);
    return;
  }
  if (kv == 0 && part == 0 && tid == 0) a.lens_out[m] = n;
  if (n == len || n == 0) {
    if (part == 0 && mass_out != mass)
      for (int e = tid; e < n; e += kEvThreads) {
        mass_out[e] = mass[e];
        pos_out[e] = pos[e];
      }
    return;
  }
#pragma unroll
  for (int w = 0; w < kEvWarps; ++w) newest = max(newest, sh[0][w]);
  const long long guard = (long long)newest - a.recent;  // protected: positions above it

  // The set that the cut falls into is the unprotected entries (inner: the protected ones, when
  // they alone fill n). Keys outside it become kEvKeep or kEvDrop; the set's first digits are
  // counted on the way, as if it were the unprotected ones.
  bool inner = false;
  auto make = [&](uint32_t k, bool p) { return p == inner ? k : p ? kEvKeep : kEvDrop; };
  auto key = [&](int e) { return STAGED ? keys[e] : make(ev_key(mass[e]), pos[e] > guard); };
  auto tally = [&](int* hist, uint32_t k, uint32_t bin, bool in) {
    if (in && k != kEvDrop && k != kEvKeep) atomicAdd(&hist[bin], 1);
  };
  int cnt = 0;
  auto first = [&](int e, int p) {
    const bool g = p > guard;
    const uint32_t k = make(STAGED ? keys[e] : ev_key(mass[e]), g);
    if (STAGED && g) keys[e] = k;
    cnt += g;
    tally(u.hist[0], k, k >> 21, true);
  };
#pragma unroll
  for (int i = 0; i < kEvHeld; ++i)
    if (tid + i * kEvThreads < len) first(tid + i * kEvThreads, held[i]);
#pragma unroll 4
  for (int e = tid + kEvHeld * kEvThreads; e < len; e += kEvThreads) first(e, pos[e]);
  cnt = __reduce_add_sync(0xffffffffu, cnt);
  if (lane == 0) sh[1][warp] = cnt;
  __syncthreads();
  int guarded = 0;
#pragma unroll
  for (int w = 0; w < kEvWarps; ++w) guarded += sh[1][w];
  int want = n - guarded;  // of the set
  if (guarded >= n) {      // uniform: the protected entries compete among themselves
    inner = true;
    want = n;
    for (int i = tid; i < kEvBins; i += kEvThreads) u.hist[0][i] = 0;
    __syncthreads();
    for (int e = tid; e < len; e += kEvThreads) {
      const uint32_t k = make(ev_key(mass[e]), pos[e] > guard);
      if (STAGED) keys[e] = k;
      tally(u.hist[0], k, k >> 21, true);
    }
    __syncthreads();
  }

  // radix select: entries whose key >> shift is above cut stay, and the first `want` equal to it
  uint32_t cut = 0;
  int shift = 21, equal = 0;
#pragma unroll 1
  for (int d = 0;; ++d) {
    const int* hist = u.hist[d];
    const int4 h4 = *reinterpret_cast<const int4*>(hist + kEvBins - 4 - 4 * tid);  // from the largest down
    const int s[4] = {h4.w, h4.z, h4.y, h4.x};
    const int sum = s[0] + s[1] + s[2] + s[3];
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sh[d & 1][warp] = incl;
    __syncthreads();
    int before = incl - sum;
#pragma unroll
    for (int w = 0; w < kEvWarps; ++w)
      if (w < warp) before += sh[d & 1][w];
    if (before < want && want <= before + sum) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (before < want && want <= before + s[i]) {
          pick[0] = kEvBins - 1 - 4 * tid - i;
          pick[1] = want - before;
          pick[2] = s[i];
        }
        before += s[i];
      }
    }
    __syncthreads();
    const int width = d == 2 ? 10 : 11;
    cut = d == 0 ? (uint32_t)pick[0] : (cut << width) | (uint32_t)pick[0];
    want = pick[1];
    equal = pick[2];
    if (d == 2 || want == equal) break;  // every bit used, or the whole bucket stays
    const int next = d == 0 ? 10 : 0;
    for (int e = tid; e < len; e += kEvThreads) {
      const uint32_t k = key(e);
      tally(u.hist[d + 1], k, (k >> next) & (d == 0 ? 2047u : 1023u), (k >> shift) == cut);
    }
    shift = next;
    __syncthreads();
  }

  // Survivors. Each warp takes a contiguous run of 32-entry words; ranks are the run's start
  // plus a count of bits.
  const int words = (len + 31) / 32, run = (words + kEvWarps - 1) / kEvWarps;
  const int w0 = min(words, warp * run), w1 = min(words, w0 + run);
  int tie = 0;
  if (want < equal) {
    int ties = 0;
    for (int w = w0; w < w1; ++w) {
      const int e = w * 32 + lane;
      const uint32_t k = e < len ? key(e) : kEvKeep;
      ties += __popc(__ballot_sync(0xffffffffu, k != kEvKeep && k != kEvDrop && (k >> shift) == cut));
    }
    __syncthreads();
    if (lane == 0) sh[0][warp] = ties;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kEvWarps; ++w)
      if (w < warp) tie += sh[0][w];
  }
  auto below_n = [&](int w) { return w * 32 + 32 <= n ? 0xffffffffu : w * 32 >= n ? 0u : (1u << (n - w * 32)) - 1u; };
  int holes = 0, tails = 0;
  for (int w = w0; w < w1; ++w) {
    const int e = w * 32 + lane;
    const uint32_t k = e < len ? key(e) : kEvDrop, kk = k >> shift;
    const bool in = k != kEvDrop && k != kEvKeep;
    const uint32_t eq = __ballot_sync(0xffffffffu, in && kk == cut);
    const bool stay = k == kEvKeep || (in && (kk > cut || (kk == cut && tie + __popc(eq & ((1u << lane) - 1u)) < want)));
    tie += want < equal ? __popc(eq) : -32;  // the whole bucket stays: no rank reaches want
    const uint32_t b = __ballot_sync(0xffffffffu, stay), low = below_n(w);
    if (lane == 0) bits[w] = b;
    holes += __popc(~b & low);
    tails += __popc(b & ~low);
  }
  __syncthreads();
  if (lane == 0) {
    sh[0][warp] = holes;
    sh[1][warp] = tails;
  }
  __syncthreads();
  if (a.cluster > 1) ev_cluster_arrive();  // mass and positions have been read
  int hole0 = 0, tail0 = 0, moves = 0;  // as many holes as survivors past n
#pragma unroll
  for (int w = 0; w < kEvWarps; ++w) {
    if (w < warp) hole0 += sh[0][w], tail0 += sh[1][w];
    moves += sh[1][w];
  }

  const int share = (moves + a.cluster - 1) / a.cluster;
  const int m0 = min(moves, part * share), m1 = min(moves, m0 + share);
  const int pieces = a.hd / 8;  // 16-byte pieces of a K or V row
  uint4* kr = reinterpret_cast<uint4*>(a.kc + base * a.hd);
  uint4* vr = reinterpret_cast<uint4*>(a.vc + base * a.hd);
  int* hole = u.list.hole;
  int* from = u.list.from;
  bool met = a.cluster == 1;
  for (int at = m0; at < m1; at += kEvMoves) {
    const int count = min(kEvMoves, m1 - at);
    __syncthreads();  // the histograms, or the lists of the round before, are done with
    int h = hole0 - at, t = tail0 - at;
    for (int w = w0; w < w1; ++w) {
      const uint32_t b = bits[w], low = below_n(w);
      const uint32_t bh = ~b & low, bt = b & ~low, below = (1u << lane) - 1u;
      const int i = h + __popc(bh & below), j = t + __popc(bt & below);
      if ((bh >> lane & 1u) && i >= 0 && i < count) hole[i] = w * 32 + lane;
      if ((bt >> lane & 1u) && j >= 0 && j < count) from[j] = w * 32 + lane;
      h += __popc(bh);
      t += __popc(bt);
    }
    __syncthreads();
    constexpr int U = 4;  // rows' pieces in flight per thread: eight 16-byte loads
    const int all = count * pieces;
    for (int i0 = tid; i0 < all; i0 += U * kEvThreads) {
      uint4 k4[U], v4[U];
      int d[U];
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const int i = i0 + q * kEvThreads;
        if (i < all) {
          const int j = i / pieces, c = i - j * pieces;
          const size_t s = (size_t)from[j] * pieces + c;
          d[q] = hole[j] * pieces + c;
          k4[q] = kr[s];
          v4[q] = vr[s];
        }
      }
#pragma unroll
      for (int q = 0; q < U; ++q)
        if (i0 + q * kEvThreads < all) {
          kr[d[q]] = k4[q];
          vr[d[q]] = v4[q];
        }
    }
    if (!met) ev_cluster_wait();
    met = true;
    for (int j = tid; j < count; j += kEvThreads) {
      mass_out[hole[j]] = mass[from[j]];
      pos_out[hole[j]] = pos[from[j]];
    }
  }
  if (!met) ev_cluster_wait();
  if (mass_out != mass)  // separate outputs: the survivors that stayed in place
    for (int e = part * kEvThreads + tid; e < n; e += a.cluster * kEvThreads)
      if (bits[e >> 5] >> (e & 31) & 1u) {
        mass_out[e] = mass[e];
        pos_out[e] = pos[e];
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
  // CTAs per (row, head): enough for two per SM, and 64 moves at least for each
  const uint32_t pairs = M * num_kv_heads, most = std::min<uint32_t>(a.budget, max_seq - a.budget);
  uint32_t c = 1;
  while (c < 8 && 2 * c * pairs <= 4 * (uint32_t)num_sms() && most >= 128 * c) c *= 2;
  a.cluster = (int)c;
  if ((uint64_t)pairs * c > 0x7fffffffu) return fail(ORCH_ERR_UNSUPPORTED, "cache_evict: too many rows and heads");
  const dim3 grid(pairs * c), cl(c > 1 ? c : 0, c > 1 ? 1 : 0, c > 1 ? 1 : 0);
  if (staged <= (size_t)kEvStaged)
    ORCH_CUDA(launch_k(cache_evict_kernel<true>, grid, dim3(kEvThreads), staged, as_stream(stream), cl, a));
  else
    ORCH_CUDA(launch_k(cache_evict_kernel<false>, grid, dim3(kEvThreads), bits, as_stream(stream), cl, a));
  return check_launch("cache_evict");
}
