// What the kernels of attention over shared prefixes have in common (attention_prefix.cu: the
// mma.sync tiles, the own entries and the join; attention_prefix_tc.cu: the tcgen05 tiles of
// prefixes with many query rows).
#pragma once

#include "orch_common.cuh"

namespace orch {

constexpr int kApKeys = 64;         // keys per block
constexpr int kApMaxUnitRows = 128;  // rows of a unit
constexpr uint32_t kApMaxLen = 1u << 29;  // entries of a slot: twice that stays an int
constexpr float kApShift = 10.f;    // P is held as 2^10 e^(s - max)

struct ApArgs {
  const __half* q;
  const __half* kp;
  const __half* vp;
  const int4* units;  // (row0, rows, prefix slot, prefix length)
  int num_units, max_prefix, prefix_cap, num_prefix;
  const __half* kc;
  const __half* vc;
  const int* lens;
  const int* slots;
  int max_own, max_seq, num_slots;
  float* mass;
  __half* out;
  int M, nh, nkv, G;
  int tr_p, tr_sh;       // query rows of a prefix tile, and their logarithm
  int tiles_p, tiles_o;  // row tiles of all units (as many as disjoint ones can have) / per row
  int S_p, S_o;          // key ranges of a prefix / of a row's own entries
  int blk_p;             // keys that a range of a prefix is a multiple of
  int tc;                // the prefix part runs in its own kernel (attention_prefix_tc.cu)
  int blocks_p;          // CTAs of the prefix part
  int row;               // few rows and keys: a CTA per row and K/V head takes all of them
  int direct;            // the output is written by the attention kernel: nothing to join
  float* acc;            // [M * nh][S][HD]
  float2* stat;          // [M * nh][S]: (max, sum), in powers of two
  float* scores;         // [M * nh][lds], with mass only
  int lds;
  uint32_t* check;
};

__device__ __forceinline__ float ap_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Keys per range when n keys are cut into at most S ranges of whole blocks.
__host__ __device__ __forceinline__ int ap_range(int n, int S, int block = kApKeys) {
  const int per = (n + S - 1) / S;
  return (per + block - 1) / block * block;
}

// A unit's prefix is one of the call's; with max_prefix 0 there are none, and its number does not matter.
__device__ __forceinline__ bool ap_unit_prefix_ok(const ApArgs& a, const int4& u) {
  return a.max_prefix == 0 || (u.z >= 0 && u.z < a.num_prefix);
}
// A unit that names rows, a prefix and a length inside what the call was given.
__device__ __forceinline__ bool ap_unit_ok(const ApArgs& a, const int4& u) {
  return u.y >= 1 && u.y <= kApMaxUnitRows && u.x >= 0 && u.x < a.M && u.y <= a.M - u.x && u.w >= 0 &&
         u.w <= a.max_prefix && ap_unit_prefix_ok(a, u);
}
// Row tiles of a unit; a rejected one has none.
__device__ __forceinline__ int ap_unit_tiles(const ApArgs& a, const int4& u) {
  return ap_unit_ok(a, u) ? (u.y * a.G + a.tr_p - 1) >> a.tr_sh : 0;
}
// Reports the rejected units. Whole CTAs call.
__device__ __forceinline__ void ap_report_units(const ApArgs& a) {
  for (int i = threadIdx.x; i < a.num_units; i += blockDim.x) {
    const int4 u = a.units[i];
    if (!ap_unit_ok(a, u)) atomicOr(a.check, ap_unit_prefix_ok(a, u) ? 2u : 8u);
  }
}
// Row tile t of all units, in their order: its unit (in u) and its first query row, or -1 past
// the last tile. Whole warps call.
__device__ __forceinline__ int ap_find_tile(const ApArgs& a, int t, int4& u) {
  const int lane = threadIdx.x & 31;
  for (int u0 = 0; u0 < a.num_units; u0 += 32) {
    int4 v = make_int4(0, 0, 0, 0);
    int tiles = 0;
    if (u0 + lane < a.num_units) {
      v = a.units[u0 + lane];
      tiles = ap_unit_tiles(a, v);
    }
    int end = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= o) end += x;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, t < end);
    if (hit != 0u) {
      const int l = __ffs(hit) - 1;
      u = make_int4(__shfl_sync(0xffffffffu, v.x, l), __shfl_sync(0xffffffffu, v.y, l), __shfl_sync(0xffffffffu, v.z, l),
                    __shfl_sync(0xffffffffu, v.w, l));
      return (t - __shfl_sync(0xffffffffu, end - tiles, l)) * a.tr_p;
    }
    t -= __shfl_sync(0xffffffffu, end, 31);
  }
  return -1;
}
// Whether the tiles of row m's query rows are among the tiles_p that the grid has. They are, unless
// units overlap: those of disjoint units are at most tiles_p. Whole warps call.
__device__ __forceinline__ bool ap_row_has_tile(const ApArgs& a, int m) {
  const int lane = threadIdx.x & 31;
  long long before = 0;
  for (int u0 = 0; u0 < a.num_units; u0 += 32) {
    int tiles = 0, own = -1;
    if (u0 + lane < a.num_units) {
      const int4 v = a.units[u0 + lane];
      tiles = ap_unit_tiles(a, v);
      if (tiles > 0 && m >= v.x && m - v.x < v.y) own = ((m - v.x) * a.G + a.G - 1) >> a.tr_sh;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, own >= 0);
    const int l = hit != 0u ? __ffs(hit) - 1 : 32;
    before += __reduce_add_sync(0xffffffffu, lane < l ? tiles : 0);
    if (hit != 0u) return before + __shfl_sync(0xffffffffu, own, l) < a.tiles_p;
  }
  return true;  // in no unit
}
// The row's cache slot and own length, or false when either lies outside the cache.
__device__ __forceinline__ bool ap_row(const ApArgs& a, int m, int& slot, int& len) {
  slot = a.slots ? a.slots[m] : m;
  len = a.lens[m];
  return slot >= 0 && slot < a.num_slots && len >= 0 && len <= a.max_own;
}

// The prefix part on tcgen05 tiles of kApTcRows query rows, or twice as many (head_dim 64 or 128).
constexpr int kApTcRows = 128, kApTcKeys = 128;
int ap_tc_launch(const ApArgs& a, int hd, cudaStream_t st);

}  // namespace orch
