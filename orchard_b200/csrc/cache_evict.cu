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

constexpr int kEvMoves = 2048;  // moves listed at a time
constexpr int kEvBins = 2048;
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

// Four consecutive entries, 16-byte loads where rows are aligned for them.
struct EvFour {
  float m[4];
  int p[4];
};
__device__ __forceinline__ EvFour ev_load(const float* mass, const int* pos, int e, int len, bool vec) {
  EvFour r;
  if (vec && e + 4 <= len) {
    const float4 f = *reinterpret_cast<const float4*>(mass + e);
    const int4 i = *reinterpret_cast<const int4*>(pos + e);
    r.m[0] = f.x, r.m[1] = f.y, r.m[2] = f.z, r.m[3] = f.w;
    r.p[0] = i.x, r.p[1] = i.y, r.p[2] = i.z, r.p[3] = i.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r.m[j] = e + j < len ? mass[e + j] : 0.f;
      r.p[j] = e + j < len ? pos[e + j] : -0x7fffffff - 1;
    }
  }
  return r;
}

// use(e, load(e)) for this thread's groups of four entries, U loads requested before the first
// is used.
template <int U, int NT, typename Load, typename Use>
__device__ __forceinline__ void ev_sweep(int len, Load load, Use use) {
  for (int e = 4 * threadIdx.x; e < len; e += 4 * U * NT) {
    decltype(load(0)) v[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (e + 4 * i * NT < len) v[i] = load(e + 4 * i * NT);
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (e + 4 * i * NT < len) use(e + 4 * i * NT, v[i]);
  }
}

// STAGED: the keys stay in shared memory; caches too long for that read mass and position
// again in every pass.
template <int NT, bool STAGED>
__global__ void __launch_bounds__(NT, 1024 / NT) cache_evict_kernel(const EvArgs a) {
  constexpr int NW = NT / 32, BPT = kEvBins / NT;  // warps, bins per thread
  extern __shared__ __align__(16) uint32_t ev_smem[];  // survivors, a bit per entry; then the keys
  __shared__ union {
    __align__(16) int hist[3][kEvBins];
    struct {
      int hole[kEvMoves], from[kEvMoves];
    } list;
  } u;
  __shared__ int sh[2][NW];
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
    for (int r = tid; r < m; r += NT) twice |= a.slots[r] == slot;
  const int n = min(len, a.budget);
  const size_t base = ((size_t)slot * a.nkv + kv) * a.max_seq;
  const float* mass = a.mass + base;
  const int* pos = a.pos + base;
  float* mass_out = a.mass_out + base;
  int* pos_out = a.pos_out + base;
  const bool vec = (((uintptr_t)mass | (uintptr_t)pos) & 15) == 0;
  uint32_t* bits = ev_smem;
  uint4* keys = reinterpret_cast<uint4*>(ev_smem + (a.max_seq + 127) / 128 * 4);  // four entries each
  auto entries = [&](int e) { return ev_load(mass, pos, e, len, vec); };

  // newest position; the keys of all masses, if they fit (kEvDrop past the last entry)
  int newest = -0x7fffffff - 1;
  for (int i = tid * 4; i < 3 * kEvBins; i += NT * 4)
    *reinterpret_cast<int4*>(&u.hist[0][0] + i) = make_int4(0, 0, 0, 0);
  ev_sweep<4, NT>(len, entries, [&](int e, const EvFour& v) {
    uint32_t k[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      newest = max(newest, v.p[j]);
      k[j] = e + j < len ? ev_key(v.m[j]) : kEvDrop;
    }
    if (STAGED) keys[e >> 2] = make_uint4(k[0], k[1], k[2], k[3]);
  });
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (lane == 0) sh[0][warp] = newest;
  if (__syncthreads_or(twice)) {
    if (tid == 0) atomicOr(a.check, 8u);
    return;
  }
  if (kv == 0 && part == 0 && tid == 0) a.lens_out[m] = n;
  const bool vec_out = (((uintptr_t)mass_out | (uintptr_t)pos_out) & 15) == 0;
  auto copy = [&](int e, const EvFour& v, uint32_t which) {  // masses and positions into place
    if (vec_out && which == 15u) {
      *reinterpret_cast<float4*>(mass_out + e) = make_float4(v.m[0], v.m[1], v.m[2], v.m[3]);
      *reinterpret_cast<int4*>(pos_out + e) = make_int4(v.p[0], v.p[1], v.p[2], v.p[3]);
      return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (which >> j & 1u) {
        mass_out[e + j] = v.m[j];
        pos_out[e + j] = v.p[j];
      }
  };
  if (n == len || n == 0) {
    if (part == 0 && mass_out != mass)
      ev_sweep<4, NT>(n, entries, [&](int e, const EvFour& v) { copy(e, v, e + 4 <= n ? 15u : (1u << (n - e)) - 1u); });
    return;
  }
  newest = __reduce_max_sync(0xffffffffu, sh[0][lane % NW]);
  // protected: positions above newest - recent
  const int guard = (int)max((long long)newest - a.recent + 1, -0x80000000ll);
  const bool any = a.recent != 0u;

  // The set that the cut falls into is the unprotected entries (inner: the protected ones, when
  // they alone fill n). Keys outside it become kEvKeep or kEvDrop; the set's first digits are
  // counted on the way, as if it were the unprotected ones.
  bool inner = false;
  auto make = [&](const uint4& raw, const EvFour& v, int& count) {
    const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t k[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool g = any && v.p[j] >= guard && r[j] != kEvDrop;
      k[j] = g == inner ? r[j] : g ? kEvKeep : kEvDrop;
      count += g;
    }
    return make_uint4(k[0], k[1], k[2], k[3]);
  };
  auto raw_keys = [&](int e, const EvFour& v) {
    uint32_t k[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) k[j] = e + j < len ? ev_key(v.m[j]) : kEvDrop;
    return make_uint4(k[0], k[1], k[2], k[3]);
  };
  auto tally = [&](int* hist, const uint4& k4, int shift, uint32_t mask, int above, uint32_t prefix) {
    const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k[j] - 1u < kEvKeep - 1u && (above == 32 || k[j] >> above == prefix)) atomicAdd(&hist[k[j] >> shift & mask], 1);
  };
  int cnt = 0;
  ev_sweep<4, NT>(len, entries, [&](int e, const EvFour& v) {
    const uint4 k = make(STAGED ? keys[e >> 2] : raw_keys(e, v), v, cnt);
    if (STAGED) keys[e >> 2] = k;
    tally(u.hist[0], k, 21, 2047u, 32, 0u);
  });
  cnt = __reduce_add_sync(0xffffffffu, cnt);
  if (lane == 0) sh[1][warp] = cnt;
  __syncthreads();
  const int guarded = __reduce_add_sync(0xffffffffu, lane < NW ? sh[1][lane] : 0);
  int want = n - guarded;  // of the set
  if (guarded >= n) {      // uniform: the protected entries compete among themselves
    inner = true;
    want = n;
    for (int i = tid; i < kEvBins; i += NT) u.hist[0][i] = 0;
    __syncthreads();
    ev_sweep<4, NT>(len, entries, [&](int e, const EvFour& v) {
      int c = 0;
      const uint4 k = make(raw_keys(e, v), v, c);
      if (STAGED) keys[e >> 2] = k;
      tally(u.hist[0], k, 21, 2047u, 32, 0u);
    });
    __syncthreads();
  }
  auto key4 = [&](int e) {
    if (STAGED) return keys[e >> 2];
    const EvFour v = entries(e);
    int c = 0;
    return make(raw_keys(e, v), v, c);
  };

  // radix select: entries whose key >> shift is above cut stay, and the first `want` equal to it
  uint32_t cut = 0;
  int shift = 21, equal = 0;
#pragma unroll 1
  for (int d = 0;; ++d) {
    const int* hist = u.hist[d];
    int s[BPT], sum = 0;  // from the largest bin down
#pragma unroll
    for (int i = 0; i < BPT; i += 4) {
      const int4 h4 = *reinterpret_cast<const int4*>(hist + kEvBins - 4 - i - BPT * tid);
      s[i] = h4.w, s[i + 1] = h4.z, s[i + 2] = h4.y, s[i + 3] = h4.x;
      sum += h4.x + h4.y + h4.z + h4.w;
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sh[d & 1][warp] = incl;
    __syncthreads();
    int before = incl - sum + __reduce_add_sync(0xffffffffu, lane < warp ? sh[d & 1][lane] : 0);
    if (before < want && want <= before + sum) {
#pragma unroll
      for (int i = 0; i < BPT; ++i) {
        if (before < want && want <= before + s[i]) {
          pick[0] = kEvBins - 1 - BPT * tid - i;
          pick[1] = want - before;
          pick[2] = s[i];
        }
        before += s[i];
      }
    }
    __syncthreads();
    cut = d == 0 ? (uint32_t)pick[0] : cut << (d == 2 ? 10 : 11) | (uint32_t)pick[0];
    want = pick[1];
    equal = pick[2];
    if (d == 2 || want == equal) break;  // every bit used, or the whole bucket stays
    const int next = d == 0 ? 10 : 0;
    ev_sweep<4, NT>(len, key4, [&](int, const uint4& k) { tally(u.hist[d + 1], k, next, d == 0 ? 2047u : 1023u, shift, cut); });
    shift = next;
    __syncthreads();
  }

  // `last`: the index of the want-th equal key, the last of them that stays
  int last = len;
  if (want < equal) {  // each warp looks through a contiguous run of entries, 32 at a time
    const int run = ((len + NW - 1) / NW + 31) / 32 * 32, e0 = min(len, warp * run), e1 = min(len, e0 + run);
    auto same = [&](int e) {
      const int at = min(e, len - 1);
      const uint4 k4 = key4(at & ~3);
      const uint32_t k = (e & 2) ? ((e & 1) ? k4.w : k4.z) : ((e & 1) ? k4.y : k4.x);
      return __ballot_sync(0xffffffffu, e < e1 && k != kEvDrop && k >> shift == cut);
    };
    int ties = 0;
    for (int e = e0; e < e1; e += 32) ties += __popc(same(e + lane));
    __syncthreads();
    if (lane == 0) sh[0][warp] = ties;
    __syncthreads();
    int before = __reduce_add_sync(0xffffffffu, lane < warp ? sh[0][lane] : 0);
    if (before < want && want <= before + ties) {
      for (int e = e0; e < e1; e += 32) {
        const uint32_t b = same(e + lane);
        const int c = __popc(b);
        if (before < want && want <= before + c && lane == 0) pick[0] = e + (int)__fns(b, 0, want - before);
        before += c;
      }
    }
    __syncthreads();
    last = pick[0];
  }

  // survivors, a byte of eight bits per thread and step
  uint8_t* bytes = reinterpret_cast<uint8_t*>(bits);
  const int words = (len + 31) / 32;
  for (int e = 8 * tid; e < words * 32; e += 8 * NT) {
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (e + 4 * i >= len) continue;
      const uint4 k4 = key4(e + 4 * i);
      const uint32_t k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t kk = k[j] >> shift;
        const bool stay = kk > cut || (kk == cut && k[j] != kEvDrop && e + 4 * i + j <= last);
        b |= (uint32_t)stay << (4 * i + j);
      }
    }
    bytes[e >> 3] = (uint8_t)b;
  }
  __syncthreads();
  if (a.cluster > 1) ev_cluster_arrive();  // mass and positions have been read

  // Holes (dropped, below n) and tails (kept, at or above n) are numbered in order: a thread
  // takes a run of words. There are as many of the one as of the other.
  const int run = (words + NT - 1) / NT, w0 = min(words, tid * run), w1 = min(words, w0 + run);
  auto below_n = [&](int w) { return w * 32 + 32 <= n ? 0xffffffffu : w * 32 >= n ? 0u : (1u << (n - w * 32)) - 1u; };
  int holes = 0, tails = 0;
  for (int w = w0; w < w1; ++w) {
    const uint32_t b = bits[w], low = below_n(w);
    holes += __popc(~b & low);
    tails += __popc(b & ~low);
  }
  int hole0 = holes, tail0 = tails;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, hole0, o), y = __shfl_up_sync(0xffffffffu, tail0, o);
    if (lane >= o) hole0 += x, tail0 += y;
  }
  if (lane == 31) {
    sh[0][warp] = hole0;
    sh[1][warp] = tail0;
  }
  hole0 -= holes;
  tail0 -= tails;
  __syncthreads();
  hole0 += __reduce_add_sync(0xffffffffu, lane < warp ? sh[0][lane] : 0);
  tail0 += __reduce_add_sync(0xffffffffu, lane < warp ? sh[1][lane] : 0);
  const int moves = __reduce_add_sync(0xffffffffu, lane < NW ? sh[1][lane] : 0);

  const int share = (moves + a.cluster - 1) / a.cluster;
  const int m0 = min(moves, part * share), m1 = min(moves, m0 + share);
  const int pieces = a.hd / 8;  // 16-byte pieces of a K or V row
  const int log2p = (pieces & (pieces - 1)) == 0 ? __ffs(pieces) - 1 : -1;
  uint4* kr = reinterpret_cast<uint4*>(a.kc + base * a.hd);
  uint4* vr = reinterpret_cast<uint4*>(a.vc + base * a.hd);
  int* hole = u.list.hole;
  int* from = u.list.from;
  bool met = a.cluster == 1;
  for (int at = m0; at < m1; at += kEvMoves) {
    const int count = min(kEvMoves, m1 - at);
    if (at > m0) __syncthreads();  // the lists of the round before are done with
    int h = hole0 - at, t = tail0 - at;
    for (int w = w0; w < w1; ++w) {
      const uint32_t b = bits[w], low = below_n(w);
      for (uint32_t x = ~b & low; x != 0u; x &= x - 1u, ++h)
        if (h >= 0 && h < count) hole[h] = w * 32 + __ffs(x) - 1;
      for (uint32_t x = b & ~low; x != 0u; x &= x - 1u, ++t)
        if (t >= 0 && t < count) from[t] = w * 32 + __ffs(x) - 1;
    }
    __syncthreads();
    constexpr int U = 4;  // pieces in flight per thread: eight 16-byte loads
    const int all = count * pieces;
    for (int i0 = tid; i0 < all; i0 += U * NT) {
      uint4 k4[U], v4[U];
      int d[U];
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const int i = i0 + q * NT;
        if (i < all) {
          const int j = log2p >= 0 ? i >> log2p : i / pieces, c = i - j * pieces;
          const size_t s = (size_t)from[j] * pieces + c;
          d[q] = hole[j] * pieces + c;
          k4[q] = kr[s];
          v4[q] = vr[s];
        }
      }
#pragma unroll
      for (int q = 0; q < U; ++q)
        if (i0 + q * NT < all) {
          kr[d[q]] = k4[q];
          vr[d[q]] = v4[q];
        }
    }
    if (!met) ev_cluster_wait();
    met = true;
    for (int j = tid; j < count; j += NT) {
      const float mv = mass[from[j]];
      const int pv = pos[from[j]];
      mass_out[hole[j]] = mv;
      pos_out[hole[j]] = pv;
    }
  }
  if (!met) ev_cluster_wait();
  if (mass_out != mass) {  // separate outputs: the survivors that stayed in place
    const int part4 = ((n + a.cluster - 1) / a.cluster + 3) / 4 * 4, e0 = min(n, part * part4), e1 = min(n, e0 + part4);
    ev_sweep<4, NT>(e1 - e0, [&](int e) { return entries(e0 + e); },
                    [&](int e, const EvFour& v) {
                      const uint32_t here = e0 + e + 4 <= n ? 15u : (1u << (n - e0 - e)) - 1u;
                      copy(e0 + e, v, bits[(e0 + e) >> 5] >> ((e0 + e) & 31) & here);
                    });
  }
}

template <int NT, bool STAGED>
int ev_launch(const EvArgs& a, size_t smem, cudaStream_t st) {
  static bool attr_done[64] = {};
  const int dev = device_index();
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    ORCH_CUDA(cudaFuncSetAttribute(cache_evict_kernel<NT, STAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvStaged));
    attr_done[dev] = true;
  }
  const unsigned c = (unsigned)a.cluster;
  ORCH_CUDA(launch_k(cache_evict_kernel<NT, STAGED>, dim3((unsigned)a.M * a.nkv * c), dim3(NT), smem, st,
                     c > 1 ? dim3(c, 1, 1) : dim3(0, 0, 0), a));
  return check_launch("cache_evict");
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
  ORCH_REQUIRE((((uintptr_t)mass | (uintptr_t)positions | (uintptr_t)lens | (uintptr_t)slots | (uintptr_t)mass_out |
                 (uintptr_t)positions_out | (uintptr_t)lens_out) & 3) == 0,
               "cache_evict: mass, positions, lens and slots must be 4-byte aligned");
  ORCH_REQUIRE(lens_out != lens, "cache_evict: lens_out must not be lens (heads read it while others finish)");
  ORCH_REQUIRE((mass_out == mass) == (positions_out == positions),
               "cache_evict: mass and positions are both updated in place, or neither");
  if (max_seq > kEvMaxLen) return fail(ORCH_ERR_UNSUPPORTED, "cache_evict: max_seq above 1,000,000");
  if ((uint64_t)M * num_kv_heads > 0x7fffffffu) return fail(ORCH_ERR_UNSUPPORTED, "cache_evict: too many rows and heads");
  // Outputs are in place or lie apart from everything that other CTAs may still read.
  const size_t rows = (size_t)M * 4, entries = (size_t)num_slots * num_kv_heads * max_seq * 4;
  const auto meet = [](const void* a, size_t an, const void* b, size_t bn) {
    return a != nullptr && b != nullptr && (uintptr_t)a < (uintptr_t)b + bn && (uintptr_t)b < (uintptr_t)a + an;
  };
  const bool place = mass_out == mass;
  ORCH_REQUIRE(!meet(lens_out, rows, lens, rows) && !meet(lens_out, rows, slots, rows) && !meet(lens_out, rows, mass, entries) &&
                   !meet(lens_out, rows, positions, entries) && !meet(lens_out, rows, mass_out, entries) &&
                   !meet(lens_out, rows, positions_out, entries) &&
                   (place || (!meet(mass_out, entries, mass, entries) && !meet(positions_out, entries, positions, entries) &&
                              !meet(mass_out, entries, positions_out, entries) && !meet(mass_out, entries, positions, entries) &&
                              !meet(positions_out, entries, mass, entries))),
               "cache_evict: outputs overlap inputs or each other");
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
  const size_t bits = ((size_t)max_seq + 127) / 128 * 16, staged = bits + ((size_t)max_seq + 3) / 4 * 16;
  // CTAs per (row, head): twice as many while all of them run at once, two per SM (8 x 32 heads,
  // 1,024 -> 512: 23.7 us with one, 32.3 with two, which no longer do; 9 x 32, 2,048 -> 1,024: 41.6 and
  // 47.6; 4 x 32, 16,384 -> 4,096: 96.8 with two, 109.6 with four. Rows that lose nothing leave at once,
  // which the host cannot see: 32 x 8 heads of 1 to 1,537 -> 1,024 take 17.4 with one, 15.4 with two),
  // each with at least 128 moves (a step of one entry: 8.6 us with one, 19 with two)
  const uint32_t pairs = M * num_kv_heads, most = std::min<uint32_t>(a.budget, max_seq - a.budget);
  uint32_t c = 1;
  while (c < 8 && c * (uint64_t)pairs <= (uint64_t)num_sms() && most >= 256 * c) c *= 2;
  a.cluster = (int)c;
  if ((uint64_t)pairs * c > 0x7fffffffu) return fail(ORCH_ERR_UNSUPPORTED, "cache_evict: too many rows and heads");
  return staged <= (size_t)kEvStaged ? ev_launch<512, true>(a, staged, as_stream(stream))
                                     : ev_launch<512, false>(a, bits, as_stream(stream));
}
