// Attention of a batch whose rows share long prefixes, each prefix held once, beside every
// row's own cache entries; optionally the weight each own entry received is added to a
// running mass (the input of orch_cache_evict).
//
// Mathematics. Row m, head h, K/V head kv = h / G (G = num_heads / num_kv_heads):
//   s_j = q . k_j / sqrt(hd) over the prefix keys, then the row's own entries,
//   out = sum_j e^(s_j - max) v_j / sum_j e^(s_j - max).
// The sums over disjoint key ranges combine: a range keeps (max, sum, weighted V), and the
// ranges are joined by rescaling each with e^(its max - the common max).
//
// Work. A "unit" names consecutive rows and the prefix they share. One CTA takes a range of
// one prefix's keys for one K/V head and a tile of the unit's query rows (rows x G heads of
// that K/V head), so the prefix is read once for all of them; another CTA takes a range of
// one row's own entries for its G heads. Both run the same tensor-core tile: S = Q K^T in
// m16n8k16 MMAs (exact products of fp16 values, fp32 sums), an online softmax in fp32, O += P V
// with P in two fp16 terms, as in the prefill kernel: hi = fp16(p), lo = fp16(p - hi), a product
// each. One term alone would be off by up to 2^-11 of each weight, as much as the rounding of the
// fp16 output (64 x 32 heads behind 4,096 entries: 72.4 us a call, 71.8 with one term; 32 x 8 heads
// x 4, tracked: 41.7 and 39.6). The sums l take the fp32 weights, and P is scaled by 2^10 so that
// weights down to 2^-24 of the largest are normal numbers.
//
// Layout of a CTA: 4 warps. A tile of 64 rows gives each warp 16 rows and all 64 keys of a
// block; a tile of 16 or 32 rows splits the block's keys over 4 or 2 warps instead, whose
// (max, sum, O) meet in shared memory at the end, so few rows still keep every warp at work.
// K and V blocks of 64 keys are copied by cp.async into a double buffer.
#include <algorithm>
#include <cmath>

#include "attention_prefix.cuh"

namespace orch {

namespace {

// Half-element offset of 16-byte piece c of row r in a tile of HD-wide rows: pieces are permuted
// within 128 bytes so that the eight rows of an ldmatrix fall in distinct banks.
template <int HD>
__device__ __forceinline__ int ap_at(int r, int c) {
  return r * HD + ((HD == 32 ? c ^ ((r >> 1) & 3) : c ^ (r & 7)) << 3);
}

// The keys of a tile: rows [j0, j1) at k / v, then rows [0, n2) at k2 / v2. srow, with own2 naming
// the stretch it belongs to, takes the scores of the own entries (rows are the G heads).
struct ApKeys {
  const __half* k;
  const __half* v;
  int j0, j1;
  const __half* k2;
  const __half* v2;
  int n2;
  float* srow;
  bool own2;
};

// One tile: query rows i0 .. i0 + n - 1 of the (row, head of kv) pairs starting at row m0, over
// `keys`; partials go to range `split`. The statistics of the rows stay in shared memory.
template <int HD, int WR>
__device__ __forceinline__ void ap_tile(const ApArgs& a, int m0, int i0, int n, int kv, const ApKeys& keys, int split) {
  constexpr int WK = 4 / WR, TR = 16 * WR, TILE = kApKeys * HD, KT = kApKeys / 8 / WK;
  extern __shared__ __align__(16) uint8_t ap_smem[];
  __half* buf = reinterpret_cast<__half*>(ap_smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int wrow = warp % WR, wkey = warp / WR;
  const int nb1 = (keys.j1 - keys.j0 + kApKeys - 1) / kApKeys, nb = nb1 + (keys.n2 + kApKeys - 1) / kApKeys;
  // block b's first row and the end of its stretch
  auto first = [&](int b) { return b < nb1 ? keys.j0 + b * kApKeys : (b - nb1) * kApKeys; };
  auto end = [&](int b) { return b < nb1 ? keys.j1 : keys.n2; };

  // A thread copies piece c8 of rows r0, r0 + RS, ..: RS keeps the permutation of the pieces, so
  // their places in shared memory and in the cache are a constant apart.
  constexpr int CPR = HD / 8, RS = 128 / CPR;  // 16-byte pieces per row, rows per pass of the CTA
  static_assert(RS % 8 == 0, "the permutation repeats every eight rows");
  const int r0 = tid / CPR, c8 = tid % CPR, at0 = ap_at<HD>(r0, c8);
  auto issue = [&](int b) {
    __half* kd = buf + (b & 1) * 2 * TILE + at0;
    const int k0 = first(b), left = end(b) - k0 - r0;  // rows from r0 on
    const size_t off = left > 0 ? (size_t)(k0 + r0) * HD + c8 * 8 : 0;
    const __half* kb = (b < nb1 ? keys.k : keys.k2) + off;
    const __half* vb = (b < nb1 ? keys.v : keys.v2) + off;
#pragma unroll
    for (int j = 0; j < kApKeys / RS; ++j) {
      const bool ok = j * RS < left;
      const int step = ok ? j * RS * HD : 0;  // rows past the end are filled with zeros, not read
      cp_async16(kd + j * RS * HD, kb + step, ok);
      cp_async16(kd + TILE + j * RS * HD, vb + step, ok);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  issue(0);

  // Q rows through buffer 1, then into registers as A fragments
  __half* qs = buf + 2 * TILE;
  for (int i = tid; i < TR * (HD / 8); i += 128) {
    const int r = i / (HD / 8), c8 = i % (HD / 8);
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (r < n) {
      const int m = m0 + (i0 + r) / a.G, h = kv * a.G + (i0 + r) % a.G;
      v = *reinterpret_cast<const uint4*>(a.q + ((size_t)m * a.nh + h) * HD + c8 * 8);
    }
    *reinterpret_cast<uint4*>(qs + ap_at<HD>(r, c8)) = v;
  }
  __syncthreads();
  const int qr = wrow * 16 + g;  // this thread's rows: qr and qr + 8
  uint32_t qa[HD / 16][4];
#pragma unroll
  for (int kk = 0; kk < HD / 16; ++kk) {
    qa[kk][0] = *reinterpret_cast<const uint32_t*>(qs + ap_at<HD>(qr, 2 * kk) + 2 * c);
    qa[kk][1] = *reinterpret_cast<const uint32_t*>(qs + ap_at<HD>(qr + 8, 2 * kk) + 2 * c);
    qa[kk][2] = *reinterpret_cast<const uint32_t*>(qs + ap_at<HD>(qr, 2 * kk + 1) + 2 * c);
    qa[kk][3] = *reinterpret_cast<const uint32_t*>(qs + ap_at<HD>(qr + 8, 2 * kk + 1) + 2 * c);
  }
  __syncthreads();  // buffer 1 is free for block 1

  float o[HD / 8][4];
#pragma unroll
  for (int d = 0; d < HD / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
  float m0r = -INFINITY, m1r = -INFINITY, l0 = 0.f, l1 = 0.f;
  const float scale = rsqrtf((float)HD) * 1.4426950408889634f;  // scores in powers of two
  const int lm = lane >> 3, lr = lane & 7;

  for (int b = 0; b < nb; ++b) {
    if (b + 1 < nb) {
      issue(b + 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    const __half* ks = buf + (b & 1) * 2 * TILE;
    const __half* vs = ks + TILE;
    const int kt0 = wkey * KT;  // first 8-key tile of this warp

    float sc[KT][4];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; kk += 2) {
        uint32_t bb[4];
        ldmatrix4(ks + ap_at<HD>(8 * (kt0 + t) + lr, 2 * kk + lm), bb);
        mma_16816(sc[t], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], bb[0], bb[1]);
        mma_16816(sc[t], qa[kk + 1][0], qa[kk + 1][1], qa[kk + 1][2], qa[kk + 1][3], bb[2], bb[3]);
      }
    }
    float bm0 = -INFINITY, bm1 = -INFINITY;
    const int k0 = first(b), k1 = end(b);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool ok = k0 + 8 * (kt0 + t) + 2 * c + e < k1;
        sc[t][e] = ok ? sc[t][e] * scale : -INFINITY;
        sc[t][2 + e] = ok ? sc[t][2 + e] * scale : -INFINITY;
        bm0 = fmaxf(bm0, sc[t][e]);
        bm1 = fmaxf(bm1, sc[t][2 + e]);
      }
    if (keys.srow != nullptr && (b >= nb1) == keys.own2) {  // the own entries' scores, for their weights
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = k0 + 8 * (kt0 + t) + 2 * c + e;
          if (key < k1) {
            if (qr < n) keys.srow[(size_t)(i0 + qr) * a.lds + key] = sc[t][e];
            if (qr + 8 < n) keys.srow[(size_t)(i0 + qr + 8) * a.lds + key] = sc[t][2 + e];
          }
        }
    }
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      bm0 = fmaxf(bm0, __shfl_xor_sync(0xffffffffu, bm0, x));
      bm1 = fmaxf(bm1, __shfl_xor_sync(0xffffffffu, bm1, x));
    }
    // a warp's keys may all lie past j1: its maximum is then still -inf and stands for 0
    const float mn0 = fmaxf(m0r, bm0), mn1 = fmaxf(m1r, bm1);
    const float r0 = mn0 == -INFINITY ? 0.f : mn0 - kApShift, r1 = mn1 == -INFINITY ? 0.f : mn1 - kApShift;
    const float al0 = ap_exp2(m0r - (mn0 == -INFINITY ? 0.f : mn0)), al1 = ap_exp2(m1r - (mn1 == -INFINITY ? 0.f : mn1));
    m0r = mn0;
    m1r = mn1;
    float rs0 = 0.f, rs1 = 0.f;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      sc[t][0] = ap_exp2(sc[t][0] - r0);
      sc[t][1] = ap_exp2(sc[t][1] - r0);
      sc[t][2] = ap_exp2(sc[t][2] - r1);
      sc[t][3] = ap_exp2(sc[t][3] - r1);
      rs0 += sc[t][0] + sc[t][1];
      rs1 += sc[t][2] + sc[t][3];
    }
    l0 = l0 * al0 + rs0;
    l1 = l1 * al1 + rs1;
    if (__any_sync(0xffffffffu, al0 != 1.f || al1 != 1.f)) {  // a maximum moved (a NaN factor counts)
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) {
        o[d][0] *= al0;
        o[d][1] *= al0;
        o[d][2] *= al1;
        o[d][3] *= al1;
      }
    }
#pragma unroll
    for (int j = 0; j < KT / 2; ++j) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float p0 = sc[2 * j + (x >> 1)][2 * (x & 1)], p1 = sc[2 * j + (x >> 1)][2 * (x & 1) + 1];
        const __half2 h = __floats2half2_rn(p0, p1);
        const float2 f = __half22float2(h);
        hi[x] = h2_bits(h);
        lo[x] = h2_bits(__floats2half2_rn(p0 - f.x, p1 - f.y));
      }
#pragma unroll
      for (int d = 0; d < HD / 8; d += 2) {
        uint32_t bb[4];
        ldmatrix4_t(vs + ap_at<HD>(8 * kt0 + 16 * j + 8 * (lm & 1) + lr, d + (lm >> 1)), bb);
        mma_16816(o[d], hi[0], hi[1], hi[2], hi[3], bb[0], bb[1]);
        mma_16816(o[d + 1], hi[0], hi[1], hi[2], hi[3], bb[2], bb[3]);
        mma_16816(o[d], lo[0], lo[1], lo[2], lo[3], bb[0], bb[1]);
        mma_16816(o[d + 1], lo[0], lo[1], lo[2], lo[3], bb[2], bb[3]);
      }
    }
    __syncthreads();  // buffer b & 1 is free for block b + 2
  }
#pragma unroll
  for (int x = 1; x <= 2; x <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, x);
    l1 += __shfl_xor_sync(0xffffffffu, l1, x);
  }

  // the tile's rows in shared memory: warp wkey's part of O [row][HD] and (max, sum) per row
  constexpr int OP = HD + 4;
  float* os = reinterpret_cast<float*>(ap_smem);        // [WK][TR][OP]
  float2* ss = reinterpret_cast<float2*>(os + WK * TR * OP);  // [WK][TR]
  {
    float* w = os + (size_t)(wkey * TR + qr) * OP + 2 * c;
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) {
      *reinterpret_cast<float2*>(w + 8 * d) = make_float2(o[d][0], o[d][1]);
      *reinterpret_cast<float2*>(w + 8 * OP + 8 * d) = make_float2(o[d][2], o[d][3]);
    }
    if (c == 0) {
      ss[wkey * TR + qr] = make_float2(m0r, l0);
      ss[wkey * TR + qr + 8] = make_float2(m1r, l1);
    }
  }
  __syncthreads();
  constexpr int LPR = HD / 4;  // threads per row, four values each
  const int S = a.S_p + a.S_o;
  for (int i = tid; i < n * LPR; i += 128) {
    const int r = i / LPR, d = (i % LPR) * 4;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < WK; ++w) mx = fmaxf(mx, ss[w * TR + r].x);
    float l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WK; ++w) {
      const float2 st = ss[w * TR + r];
      const float f = st.x == -INFINITY ? 0.f : ap_exp2(st.x - mx);
      const float4 ov = *reinterpret_cast<const float4*>(os + (size_t)(w * TR + r) * OP + d);
      l = fmaf(f, st.y, l);
      v[0] = fmaf(f, ov.x, v[0]);
      v[1] = fmaf(f, ov.y, v[1]);
      v[2] = fmaf(f, ov.z, v[2]);
      v[3] = fmaf(f, ov.w, v[3]);
    }
    const size_t mh = (size_t)(m0 + (i0 + r) / a.G) * a.nh + kv * a.G + (i0 + r) % a.G;
    if (a.direct) {
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      uint2 h;
      h.x = h2_bits(__floats2half2_rn(v[0] * inv, v[1] * inv));
      h.y = h2_bits(__floats2half2_rn(v[2] * inv, v[3] * inv));
      *reinterpret_cast<uint2*>(a.out + mh * HD + d) = h;
    } else {
      *reinterpret_cast<float4*>(a.acc + (mh * S + split) * HD + d) = make_float4(v[0], v[1], v[2], v[3]);
      if (d == 0) a.stat[mh * S + split] = make_float2(mx, l);
    }
  }
  // the only row (attn_prefix_row_kernel): its own entries' weights (n is G here)
  if (a.direct && keys.srow != nullptr) {
    __syncthreads();  // scores written; O no longer needed
    float2* tot = reinterpret_cast<float2*>(ap_smem);
    if (tid < n) {
      float mx = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < WK; ++w) mx = fmaxf(mx, ss[w * TR + tid].x);
#pragma unroll
      for (int w = 0; w < WK; ++w) l += ss[w * TR + tid].x == -INFINITY ? ss[w * TR + tid].y : ap_exp2(ss[w * TR + tid].x - mx) * ss[w * TR + tid].y;
      tot[tid] = make_float2(mx == -INFINITY ? 0.f : mx - kApShift, l == 0.f ? 0.f : 1.0f / l);
    }
    __syncthreads();
    const int len = keys.n2;
    float* mass = a.mass + ((size_t)(a.slots ? a.slots[m0] : m0) * a.nkv + kv) * a.max_seq;
    for (int e = tid; e < len; e += 128) {
      float w = 0.f;
      for (int h = 0; h < n; ++h) w = fmaf(ap_exp2(keys.srow[(size_t)h * a.lds + e] - tot[h].x), tot[h].y, w);
      mass[e] = e == len - 1 ? w : mass[e] + w;
    }
  }
}

// The same tile for one warp: the G <= 16 heads of a K/V head of row m over the row's own entries
// [j0, j1), 16 keys at a time through the warp's own ring of two stages. Where there are enough
// rows and heads, four of these per CTA need no barrier and no join across warps, and a quarter of
// the CTAs (measured at kApWarpKeys).
template <int HD>
__device__ __forceinline__ void ap_warp(const ApArgs& a, int m, int kv, const __half* k, const __half* v, int j0, int j1,
                                        int split, float* srow) {
  constexpr int KEYS = 16, TILE = KEYS * HD, CPR = HD / 8, RS = 32 / CPR;  // 16-byte pieces per row, rows per pass
  extern __shared__ __align__(16) uint8_t ap_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  __half* buf = reinterpret_cast<__half*>(ap_smem) + warp * 4 * TILE;  // [stage][K, V][key][dim]
  const int nb = (j1 - j0 + KEYS - 1) / KEYS, r0 = lane / CPR, c8 = lane % CPR, n = a.G;

  auto issue = [&](int b) {
    __half* kd = buf + (b & 1) * 2 * TILE;
    const int left = j1 - j0 - b * KEYS - r0;  // rows from r0 on
    const size_t off = left > 0 ? (size_t)(j0 + b * KEYS + r0) * HD + c8 * 8 : 0;
#pragma unroll
    for (int j = 0; j < KEYS / RS; ++j) {
      const bool ok = j * RS < left;
      const int step = ok ? j * RS * HD : 0, at = ap_at<HD>(r0 + j * RS, c8);  // past the end: zeros, not read
      cp_async16(kd + at, k + off + step, ok);
      cp_async16(kd + TILE + at, v + off + step, ok);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  issue(0);
  // Q straight into A fragments: rows g and g + 8
  uint32_t qa[HD / 16][4];
  {
    const __half* q = a.q + ((size_t)m * a.nh + kv * n + g) * HD + 2 * c;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        qa[kk][x] = g + 8 * (x & 1) < n ? *reinterpret_cast<const uint32_t*>(q + (x & 1) * 8 * HD + 16 * kk + (x >> 1) * 8) : 0u;
  }
  float o[HD / 8][4];
#pragma unroll
  for (int d = 0; d < HD / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  const float scale = rsqrtf((float)HD) * 1.4426950408889634f;  // scores in powers of two
  const int lm = lane >> 3, lr = lane & 7;

  for (int b = 0; b < nb; ++b) {
    if (b + 1 < nb) {
      issue(b + 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    const __half* ks = buf + (b & 1) * 2 * TILE;
    const __half* vs = ks + TILE;
    float sc[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; kk += 2) {
        uint32_t bb[4];
        ldmatrix4(ks + ap_at<HD>(8 * t + lr, 2 * kk + lm), bb);
        mma_16816(sc[t], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], bb[0], bb[1]);
        mma_16816(sc[t], qa[kk + 1][0], qa[kk + 1][1], qa[kk + 1][2], qa[kk + 1][3], bb[2], bb[3]);
      }
    }
    float bm0 = -INFINITY, bm1 = -INFINITY;
    const int k0 = j0 + b * KEYS + 2 * c;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int key = k0 + 8 * t + e;
        const bool ok = key < j1;
        sc[t][e] = ok ? sc[t][e] * scale : -INFINITY;
        sc[t][2 + e] = ok ? sc[t][2 + e] * scale : -INFINITY;
        bm0 = fmaxf(bm0, sc[t][e]);
        bm1 = fmaxf(bm1, sc[t][2 + e]);
        if (srow != nullptr && ok) {
          if (g < n) srow[(size_t)g * a.lds + key] = sc[t][e];
          if (g + 8 < n) srow[(size_t)(g + 8) * a.lds + key] = sc[t][2 + e];
        }
      }
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      bm0 = fmaxf(bm0, __shfl_xor_sync(0xffffffffu, bm0, x));
      bm1 = fmaxf(bm1, __shfl_xor_sync(0xffffffffu, bm1, x));
    }
    const float mn0 = fmaxf(m0, bm0), mn1 = fmaxf(m1, bm1);
    const float f0 = mn0 == -INFINITY ? 0.f : mn0 - kApShift, f1 = mn1 == -INFINITY ? 0.f : mn1 - kApShift;
    const float al0 = ap_exp2(m0 - (mn0 == -INFINITY ? 0.f : mn0)), al1 = ap_exp2(m1 - (mn1 == -INFINITY ? 0.f : mn1));
    m0 = mn0;
    m1 = mn1;
    uint32_t hi[4], lo[4];
    float rs0 = 0.f, rs1 = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float f = (x & 1) ? f1 : f0;
      const float p0 = ap_exp2(sc[x >> 1][2 * (x & 1)] - f), p1 = ap_exp2(sc[x >> 1][2 * (x & 1) + 1] - f);
      if (x & 1)
        rs1 += p0 + p1;
      else
        rs0 += p0 + p1;
      const __half2 h = __floats2half2_rn(p0, p1);
      const float2 w = __half22float2(h);
      hi[x] = h2_bits(h);
      lo[x] = h2_bits(__floats2half2_rn(p0 - w.x, p1 - w.y));
    }
    l0 = l0 * al0 + rs0;
    l1 = l1 * al1 + rs1;
    if (__any_sync(0xffffffffu, al0 != 1.f || al1 != 1.f)) {  // a maximum moved (a NaN factor counts)
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) {
        o[d][0] *= al0;
        o[d][1] *= al0;
        o[d][2] *= al1;
        o[d][3] *= al1;
      }
    }
#pragma unroll
    for (int d = 0; d < HD / 8; d += 2) {
      uint32_t bb[4];
      ldmatrix4_t(vs + ap_at<HD>(8 * (lm & 1) + lr, d + (lm >> 1)), bb);
      mma_16816(o[d], hi[0], hi[1], hi[2], hi[3], bb[0], bb[1]);
      mma_16816(o[d + 1], hi[0], hi[1], hi[2], hi[3], bb[2], bb[3]);
      mma_16816(o[d], lo[0], lo[1], lo[2], lo[3], bb[0], bb[1]);
      mma_16816(o[d + 1], lo[0], lo[1], lo[2], lo[3], bb[2], bb[3]);
    }
    __syncwarp();  // stage b & 1 is free for block b + 2
  }
#pragma unroll
  for (int x = 1; x <= 2; x <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, x);
    l1 += __shfl_xor_sync(0xffffffffu, l1, x);
  }
  const int S = a.S_p + a.S_o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + 8 * h;
    if (r >= n) continue;
    const float mx = h ? m1 : m0, l = h ? l1 : l0;
    const size_t mh = (size_t)m * a.nh + kv * n + r;
    if (a.direct) {
      const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
      for (int d = 0; d < HD / 8; ++d)
        *reinterpret_cast<__half2*>(a.out + mh * HD + 8 * d + 2 * c) = __floats2half2_rn(o[d][2 * h] * inv, o[d][2 * h + 1] * inv);
    } else {
#pragma unroll
      for (int d = 0; d < HD / 8; ++d)
        *reinterpret_cast<float2*>(a.acc + (mh * S + split) * HD + 8 * d + 2 * c) = make_float2(o[d][2 * h], o[d][2 * h + 1]);
      if (c == 0) a.stat[mh * S + split] = make_float2(mx, l);
    }
  }
}

// WRP, WRO: warps along the rows of a prefix tile and of an own tile (WRP 0: no prefix here; WRO 0:
// own entries by single warps).
template <int HD, int WRP, int WRO>
__device__ __forceinline__ void ap_work(const ApArgs& a) {
  int b = blockIdx.x;
  if (a.num_units > 0) {  // the first CTA reports the rejected units
    if (b == 0) {
      ap_report_units(a);
      return;
    }
    --b;
  }
  if (WRP > 0 && b < a.blocks_p) {  // a range of a prefix for a tile of the unit's query rows
    // row tiles fastest: the tiles that read the same keys run together
    const int tile = b % a.tiles_p;
    b /= a.tiles_p;
    const int kv = b % a.nkv, split = b / a.nkv;
    int4 u;
    const int i0 = ap_find_tile(a, tile, u);
    if (i0 < 0) return;
    const int n = min(a.tr_p, u.y * a.G - i0);
    const int per = ap_range(u.w, a.S_p, a.blk_p), j0 = split * per, j1 = min(u.w, j0 + per);
    if (j0 >= j1) return;
    const size_t base = ((size_t)u.z * a.nkv + kv) * a.prefix_cap * HD;
    ap_tile<HD, WRP ? WRP : 1>(a, u.x, i0, n, kv, ApKeys{a.kp + base, a.vp + base, j0, j1, nullptr, nullptr, 0, nullptr, false},
                   split);
    return;
  }
  b -= a.blocks_p;  // a range of one row's own entries for the G heads of a K/V head
  if constexpr (WRO == 0) {
    b = b * 4 + (int)(threadIdx.x >> 5);  // K/V heads fastest: a CTA's warps mostly share a row
    const int kv = b % a.nkv;
    b /= a.nkv;
    const int split = b % a.S_o, m = b / a.S_o;
    if (m >= a.M) return;
    const bool first = (threadIdx.x & 31) == 0;
    int slot, len;
    if (!ap_row(a, m, slot, len)) {
      if (first) atomicOr(a.check, slot < 0 || slot >= a.num_slots ? 8u : 2u);
      return;
    }
    const int per = ap_range(len, a.S_o), j0 = split * per, j1 = min(len, j0 + per);
    if (j0 >= j1) {
      if (a.direct && len == 0)  // nothing to attend to
        for (int i = threadIdx.x & 31; i < a.G * HD; i += 32)
          a.out[((size_t)m * a.nh + kv * a.G) * HD + i] = __float2half_rn(0.f);
      return;
    }
    const size_t base = ((size_t)slot * a.nkv + kv) * a.max_seq * HD;
    ap_warp<HD>(a, m, kv, a.kc + base, a.vc + base, j0, j1, a.S_p + split,
                      a.mass ? a.scores + ((size_t)m * a.nh + kv * a.G) * a.lds : nullptr);
    return;
  }
  constexpr int WR = WRO ? WRO : 1;
  const int tile = b % a.tiles_o;
  b /= a.tiles_o;
  const int split = b % a.S_o;
  b /= a.S_o;
  const int kv = b % a.nkv, m = b / a.nkv;
  int slot, len;
  if (!ap_row(a, m, slot, len)) {
    if (threadIdx.x == 0) atomicOr(a.check, slot < 0 || slot >= a.num_slots ? 8u : 2u);
    return;
  }
  constexpr int tr = 16 * WR;
  const int i0 = tile * tr, n = min(tr, a.G - i0);
  const int per = ap_range(len, a.S_o), j0 = split * per, j1 = min(len, j0 + per);
  if (j0 >= j1) {
    if (a.direct && len == 0)  // nothing to attend to
      for (int i = threadIdx.x; i < n * HD; i += 128)
        a.out[((size_t)m * a.nh + kv * a.G + i0) * HD + i] = __float2half_rn(0.f);
    return;
  }
  const size_t base = ((size_t)slot * a.nkv + kv) * a.max_seq * HD;
  float* srow = a.mass ? a.scores + ((size_t)m * a.nh + kv * a.G) * a.lds : nullptr;
  ap_tile<HD, WR>(a, m, i0, n, kv, ApKeys{a.kc + base, a.vc + base, j0, j1, nullptr, nullptr, 0, srow, false},
                 a.S_p + split);
}

template <int HD, int WRP, int WRO>
__global__ void __launch_bounds__(128, 3) attn_prefix_kernel(const ApArgs a) {
  pdl_trigger();
  // Beside the prefix's own kernel, launched just before: that kernel waited for everything
  // earlier before it let this one start, and the two share no output, so they run together.
  // The first CTA stays until it has ended, so that whoever waits for this grid waits for both.
  if (!a.tc) pdl_wait();
  ap_work<HD, WRP, WRO>(a);
  if (a.tc && blockIdx.x == 0) pdl_wait();
}

// The prefix of row m: its slot and length (0: none). False when the row's unit was rejected, the
// row is in two, or (TILES) overlapping units left its tile no CTA. (Called by whole warps.)
template <bool TILES>
__device__ __forceinline__ bool ap_row_prefix(const ApArgs& a, int m, int& pslot, int& plen) {
  constexpr int kMany = 1 << 26;
  const int lane = threadIdx.x & 31;
  int bad = 0, in = 0, z = 0, w = 0, tiles = 0;
  for (int u0 = 0; u0 < a.num_units; u0 += 32) {
    const int i = u0 + lane;
    if (i < a.num_units) {
      const int4 u = a.units[i];
      if (TILES) tiles = min(tiles + ap_unit_tiles(a, u), kMany);
      if (m >= u.x && (long long)m < (long long)u.x + u.y) {
        if (ap_unit_ok(a, u)) {
          z = u.z, w = u.w;
          ++in;
        } else {
          bad = 1;
        }
      }
    }
  }
  in = (int)__reduce_add_sync(0xffffffffu, (unsigned)in);
  if (in > 1 && lane == 0) atomicOr(a.check, 2u);
  pslot = (int)__reduce_add_sync(0xffffffffu, (unsigned)z);  // one lane's at most, when in <= 1
  plen = (int)__reduce_add_sync(0xffffffffu, (unsigned)w);
  if (__any_sync(0xffffffffu, bad) || in > 1) return false;
  if (TILES && plen > 0 && (__reduce_add_sync(0xffffffffu, (unsigned)tiles) > (unsigned)a.tiles_p || __any_sync(0xffffffffu, tiles == kMany)) &&
      !ap_row_has_tile(a, m)) {
    if (lane == 0) atomicOr(a.check, 2u);
    return false;
  }
  return true;
}

// Ranges of row m that hold keys: prefix ranges 0 .. np - 1, own ranges S_p .. S_p + no - 1.
// False when the row or its unit was rejected. (Called by whole warps.)
__device__ __forceinline__ bool ap_ranges(const ApArgs& a, int m, int& slot, int& len, int& np, int& no) {
  int pslot, plen;
  const bool ok = ap_row(a, m, slot, len);
  if (!ap_row_prefix<true>(a, m, pslot, plen) || !ok) return false;
  np = plen > 0 ? (plen + ap_range(plen, a.S_p, a.blk_p) - 1) / ap_range(plen, a.S_p, a.blk_p) : 0;
  no = len > 0 ? (len + ap_range(len, a.S_o) - 1) / ap_range(len, a.S_o) : 0;
  return true;
}

// Few rows and few keys: a CTA takes one row's G heads of a K/V head through the prefix and the
// own entries and writes the output itself, in one launch.
template <int HD, int WRO>
__global__ void __launch_bounds__(128, 3) attn_prefix_row_kernel(const ApArgs a) {
  pdl_trigger();
  pdl_wait();
  const int tile = blockIdx.x % a.tiles_o, b = blockIdx.x / a.tiles_o, kv = b % a.nkv, m = b / a.nkv;
  if (blockIdx.x == 0) ap_report_units(a);  // once, whether or not a row is in them
  int slot, len, pslot, plen;
  const bool row = ap_row(a, m, slot, len);
  if (!row && threadIdx.x == 0) atomicOr(a.check, slot < 0 || slot >= a.num_slots ? 8u : 2u);
  if (!ap_row_prefix<false>(a, m, pslot, plen) || !row) return;
  constexpr int tr = 16 * WRO;
  const int i0 = tile * tr, n = min(tr, a.G - i0);
  if (plen + len == 0) {  // nothing to attend to
    for (int i = threadIdx.x; i < n * HD; i += 128)
      a.out[((size_t)m * a.nh + kv * a.G + i0) * HD + i] = __float2half_rn(0.f);
    return;
  }
  const size_t base = ((size_t)slot * a.nkv + kv) * a.max_seq * HD, pb = ((size_t)pslot * a.nkv + kv) * a.prefix_cap * HD;
  float* srow = a.mass && len > 0 ? a.scores + ((size_t)m * a.nh + kv * a.G) * a.lds : nullptr;
  ap_tile<HD, WRO>(a, m, i0, n, kv, ApKeys{a.kp + pb, a.vp + pb, 0, plen, a.kc + base, a.vc + base, len, srow, true}, 0);
}

template <int V>
struct alignas(4 * V) ApVec {
  float v[V];
};

// The common maximum and sum of row-head mh over its ranges; `first` is this lane's record (range
// `lane`), read before it was known which ranges hold keys. (Called by whole warps.)
__device__ __forceinline__ float2 ap_total(const ApArgs& a, size_t mh, int np, int no, float2 first) {
  const int lane = threadIdx.x & 31, S = a.S_p + a.S_o;
  const float2* st = a.stat + mh * S;
  auto live = [&](int s) { return s < np || (s >= a.S_p && s < a.S_p + no); };
  if (lane >= S || !live(lane)) first = make_float2(-INFINITY, 0.f);
  float mx = first.x;
  for (int s = lane + 32; s < S; s += 32)
    if (live(s)) mx = fmaxf(mx, st[s].x);
  mx = warp_max(mx);
  // a range whose maximum is -inf has sum 0, or NaN where a key was NaN: that one is kept
  float l = first.x == -INFINITY ? first.y : ap_exp2(first.x - mx) * first.y;
  for (int s = lane + 32; s < S; s += 32)
    if (live(s)) l += st[s].x == -INFINITY ? st[s].y : ap_exp2(st[s].x - mx) * st[s].y;
  return make_float2(mx, warp_sum(l));
}

// Joins the ranges: one warp per (row, head) for the output; with mass, further CTAs each
// take kMassEntries entries of one (row, K/V head).
constexpr int kMassEntries = 512;
constexpr int kMassHeads = 4;  // heads of a K/V head taken at once, a warp each

template <int HD>
__global__ void __launch_bounds__(128) attn_prefix_join_kernel(const ApArgs a, int blocks_out, int chunks) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int S = a.S_p + a.S_o;
  if (blockIdx.x < blocks_out) {
    const int mh = blockIdx.x * 4 + warp;
    if (mh >= a.M * a.nh) return;
    // The first ranges' records are requested before it is known which of them hold keys, so
    // that the kernel waits on L2 once; what a range without keys left there is not used.
    constexpr int V = HD / 32, U = 12;  // values per lane, ranges requested ahead
    const float* ac = a.acc + (size_t)mh * S * HD + lane * V;
    const float2* st = a.stat + (size_t)mh * S;
    ApVec<V> pre[U];
#pragma unroll
    for (int s = 0; s < U; ++s)
      if (s < S) pre[s] = *reinterpret_cast<const ApVec<V>*>(ac + (size_t)s * HD);
    float2 sl = lane < S ? st[lane] : make_float2(0.f, 0.f);
    int slot, len, np, no;
    if (!ap_ranges(a, mh / a.nh, slot, len, np, no)) return;
    auto live = [&](int s) { return s < np || (s >= a.S_p && s < a.S_p + no); };
    const float2 tot = ap_total(a, mh, np, no, sl);
    auto weight = [&](float m) { return m == -INFINITY ? 0.f : ap_exp2(m - tot.x); };
    const float wl = lane < S && live(lane) ? weight(sl.x) : 0.f;
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.f;
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const float f = __shfl_sync(0xffffffffu, wl, s);
      if (live(s))
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = fmaf(f, pre[s].v[i], v[i]);
    }
#pragma unroll 4
    for (int s = U; s < S; ++s) {
      const float f = s < 32 ? __shfl_sync(0xffffffffu, wl, s & 31) : live(s) ? weight(st[s].x) : 0.f;
      if (live(s)) {
        const ApVec<V> x = *reinterpret_cast<const ApVec<V>*>(ac + (size_t)s * HD);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = fmaf(f, x.v[i], v[i]);
      }
    }
    const float inv = tot.y == 0.f ? 0.f : 1.0f / tot.y;  // nothing to attend to: zeros
    __half* op = a.out + (size_t)mh * HD + lane * V;
    if (V == 4) {
      uint2 h;
      h.x = h2_bits(__floats2half2_rn(v[0] * inv, v[1 % V] * inv));
      h.y = h2_bits(__floats2half2_rn(v[2 % V] * inv, v[3 % V] * inv));
      *reinterpret_cast<uint2*>(op) = h;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) op[i] = __float2half_rn(v[i] * inv);
    }
    return;
  }
  // Weights of the own entries. The first of the rows that share a slot takes them all, in row
  // order, so the sums have one order.
  int b = blockIdx.x - blocks_out;
  const int chunk = b % chunks;
  b /= chunks;
  const int kv = b % a.nkv, m = b / a.nkv;
  int slot, len, np, no;
  if (!ap_ranges(a, m, slot, len, np, no)) return;
  constexpr int E = kMassEntries / 128;  // entries per thread
  const int e0 = chunk * kMassEntries;
  float* mass = a.mass + ((size_t)slot * a.nkv + kv) * a.max_seq;
  // the scores of kMassHeads heads of row r, requested before their totals are known
  float sv[kMassHeads][E];
  auto fetch = [&](int r, int h0) {
    const float* sr = a.scores + ((size_t)r * a.nh + kv * a.G + h0) * a.lds;
#pragma unroll
    for (int j = 0; j < kMassHeads; ++j)
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int e = e0 + threadIdx.x + 128 * i;
        sv[j][i] = j < a.G - h0 && e < len ? sr[(size_t)j * a.lds + e] : -INFINITY;
      }
  };
  __shared__ int any;
  __shared__ float2 tots[kMassHeads];
  if (threadIdx.x == 0) any = 0;
  // requested before anything is known of other rows: this row's scores and records, the masses
  fetch(m, 0);
  const int S1 = a.S_p + a.S_o;
  auto record = [&](int r, int h) {
    return h < a.G && lane < S1 ? a.stat[((size_t)r * a.nh + kv * a.G + h) * S1 + lane] : make_float2(0.f, 0.f);
  };
  float2 rec = record(m, warp);
  float old[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int e = e0 + threadIdx.x + 128 * i;
    old[i] = e < len ? mass[e] : 0.f;
  }
  __syncthreads();
  int mine = 0;  // whether another row of the call has this slot: 1 an earlier one, 2 a later one
  for (int r = threadIdx.x; r < a.M; r += 128)
    if (r != m && (a.slots ? a.slots[r] : r) == slot) mine |= r < m ? 1 : 2;
  if (mine) atomicOr(&any, mine);
  __syncthreads();
  // an earlier row of the slot that was itself rejected takes nothing: look for a valid one
  if (any & 1) {
    for (int r = 0; r < m; ++r) {
      if ((a.slots ? a.slots[r] : r) != slot) continue;
      int s2, l2, p2, o2;
      if (ap_ranges(a, r, s2, l2, p2, o2)) return;
    }
  }
  const int last = (any & 2) ? a.M - 1 : m;
  for (int r = m; r <= last; ++r) {
    if (r != m) {
      int s2;
      if ((a.slots ? a.slots[r] : r) != slot || !ap_ranges(a, r, s2, len, np, no) || e0 >= len) continue;
      fetch(r, 0);
      rec = record(r, warp);
#pragma unroll
      for (int i = 0; i < E; ++i) {  // what the rows before have left there
        const int e = e0 + threadIdx.x + 128 * i;
        old[i] = e < len ? mass[e] : 0.f;
      }
    } else if (e0 >= len) {
      continue;
    }
    float w[E];
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = 0.f;
    for (int h0 = 0; h0 < a.G; h0 += kMassHeads) {
      const int hs = min(kMassHeads, a.G - h0);
      if (h0 > 0) fetch(r, h0);
      __syncthreads();  // the totals of the heads before are done with
      if (h0 > 0) rec = record(r, h0 + warp);
      if (warp < hs) {  // the heads' totals, a warp each
        const float2 tot = ap_total(a, (size_t)r * a.nh + kv * a.G + h0 + warp, np, no, rec);
        if (lane == 0) tots[warp] = make_float2(tot.x == -INFINITY ? 0.f : tot.x - kApShift, tot.y == 0.f ? 0.f : 1.0f / tot.y);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kMassHeads; ++j)
        if (j < hs)
#pragma unroll
          for (int i = 0; i < E; ++i) w[i] = fmaf(ap_exp2(sv[j][i] - tots[j].x), tots[j].y, w[i]);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int e = e0 + threadIdx.x + 128 * i;
      if (e < len) mass[e] = e == len - 1 ? w[i] : old[i] + w[i];
    }
  }
}

// How a call is cut: rows per tile, key ranges, workspace. The same for the size query.
struct ApPlan {
  int G, wr_p, wr_o, tiles_p, tiles_o, S_p, S_o, blk_p, tr_p, tc, row, by_warp, direct, lds;
  size_t acc_floats, stat_floats, score_floats;
  size_t bytes() const { return (acc_floats + stat_floats + score_floats) * sizeof(float); }
};

constexpr uint32_t kApDirectPairs = 64, kApDirectKeys = 192;  // rows x K/V heads, keys of a row: one launch
// The tcgen05 tiles take the prefix where units have more than 32 query rows and there are 256 blocks
// of 128 x 128 (query rows, keys) over all heads, or where units have more than 16 (a tile is then
// mostly empty) and 1,024 blocks. A third launch and their start cost ~5 us: 16 rows x 8 heads x 4
// behind 2,048 entries (64 query rows, 128 blocks) 18.8 us with them, 13.6 without; 64 x 32 heads
// behind 512 (128 blocks) 24.8 and 23.2, behind 1,024 27.9 and 26.9, behind 4,096 37.6 and 51.6; 64 x 8
// x 4 behind 2,048 (256 blocks of 256 query rows) 28.4 and 29.3. 32 rows x 32 heads behind 1,024
// (256 blocks) 21.6 and 20.2, behind 4,096 (1,024) 33.6 and 37.2; two units of them behind 1,024 (512)
// 28.7 and 26.2, behind 2,048 (1,024) 34.3 and 36.3. 16 units of 8 x 32 heads behind 1,024: 84.8 and 57.8.
constexpr int kApTcRowsFrom = 32, kApTcBlocks = 256, kApTcFewFrom = 16, kApTcFewBlocks = 1024;
// Own entries of a row up to which single warps take them, where their warps (two per SM or more)
// fill the SMs, and up to which they always do. 64 x 32 heads of up to 64, 128 and 256 entries: 10.4,
// 16.8 and 30.5 us by warps, 19.9, 23.6 and 31.6 by tiles; 4 x 8 heads x 4 of up to 256: 10.3 and
// 6.1; behind a prefix of 256, 32 x 8 heads x 4 of up to 64: 10.5 and 11.3, 16 x 32: 9.4 and 11.1
// (without one 32 x 8 x 4: 5.4 and 4.7).
constexpr uint32_t kApWarpKeys = 256, kApWarpAlways = 64;

int ap_wr(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }

ApPlan ap_plan(uint32_t M, uint32_t nh, uint32_t nkv, uint32_t hd, uint32_t num_units, uint32_t max_prefix,
               uint32_t max_own, int track) {
  ApPlan p;
  p.G = (int)(nh / nkv);
  // query rows of a unit, as if all were as large
  const bool some = num_units > 0 && max_prefix > 0;
  const int rows_p = (int)std::min<uint32_t>(some ? (uint32_t)(((uint64_t)M + num_units - 1) / num_units) : M, kApMaxUnitRows) * p.G;
  const size_t blocks_k = nkv * (size_t)((max_prefix + 127) / 128);
  p.tc = some && hd != 32 &&
         ((rows_p > kApTcRowsFrom && blocks_k * (((size_t)M * p.G + 127) / 128) >= (size_t)kApTcBlocks) ||
          (rows_p > kApTcFewFrom && blocks_k * num_units >= (size_t)kApTcFewBlocks));
  p.blk_p = p.tc ? kApTcKeys : kApKeys;
  p.wr_p = std::min(ap_wr(rows_p), hd == 32 || p.G > 32 ? 4 : 2);  // 64 rows of 64 or 128 dims spill
  p.wr_o = ap_wr(p.G);
  p.tr_p = !p.tc ? 16 * p.wr_p : rows_p > kApTcRows ? 2 * kApTcRows : kApTcRows;
  // Units that share out at most M rows have at most this many tiles, and about `likely`; where
  // they overlap they may have more, and rows past these tiles are rejected (ap_row_has_tile).
  const size_t q_rows = (size_t)M * p.G;
  p.tiles_p = some ? (int)std::min<size_t>((q_rows + (size_t)num_units * (p.tr_p - 1)) / p.tr_p, 0x7fffffff) : 0;
  const size_t likely = std::max<size_t>((q_rows + p.tr_p - 1) / p.tr_p, num_units);
  p.tiles_o = (p.G + 16 * p.wr_o - 1) / (16 * p.wr_o);
  // Two rounds of three CTAs per SM at most; ranges long enough to pay for their start and their
  // record, shorter ones only where there are few CTAs (16 x 32 heads, prefix 1,000, own entries up
  // to 128: 14.6 us with ranges of 256 and 128 keys at least, 16.0 with 128 and 64).
  const int want = 6 * num_sms();
  const auto ranges = [&](size_t ctas, uint32_t keys, int least) {
    const size_t s = (want + ctas - 1) / std::max<size_t>(ctas, 1);
    return (int)std::max<size_t>(1, std::min<size_t>(s, (keys + least - 1) / least));
  };
  const size_t items = nkv * likely;
  p.S_p = 0;
  if (p.tc) {
    // One CTA per SM, and the own entries' CTAs run on the other SMs meanwhile: the cut whose
    // estimated time is least, in us. A block is taken to cost 1.5 (128 rows; 1.4 alone) or 2.7 (256;
    // 2.5 alone), a range's start and end 5, and an SM gets through ~35 KB of own entries per us (they
    // are taken to be half as long as they may be).
    const double sms = num_sms(), blocks = (max_prefix + kApTcKeys - 1) / kApTcKeys;
    const double own = (double)M * nkv * max_own * 2.0 * hd / 35e3, block = p.tr_p > kApTcRows ? 2.7 : 1.5;
    double best = 0;
    for (int c = 1; c <= (int)std::min(blocks, sms); ++c) {
      const double n = (double)items * c, run = std::ceil(blocks / c) * block + 5.0;
      const double tc = std::ceil(n / sms) * run, beside = n < sms ? (sms - n) * tc : 0.0;
      const double cost = tc + std::max(0.0, own - beside) / sms;
      if (p.S_p == 0 || cost < best) p.S_p = c, best = cost;
    }
  } else if (some) {
    p.S_p = ranges(items, max_prefix, items * (max_prefix / 256) >= (size_t)num_sms() / 2 ? 256 : 128);
  }
  const size_t own_items = (size_t)M * nkv * p.tiles_o;
  p.by_warp = p.G <= 16 && max_own <= (own_items >= 2 * (size_t)num_sms() ? kApWarpKeys : kApWarpAlways);
  p.S_o = p.by_warp ? (int)std::max<size_t>(1, std::min<size_t>((12 * (size_t)num_sms() + own_items - 1) / own_items, max_own / 128))
                    : ranges(own_items, max_own, own_items >= (size_t)num_sms() ? 128 : 64);
  // Few CTAs with little to read: splitting would cost a second launch and more than it saves (2 x
  // 2 heads of 32 keys: 3.2 us in one launch, 4.9 in two; one row of 32 heads x 577 keys, tracked:
  // 15.9 and 9.7). Weights only for a single row: rows that share a slot need an order.
  p.row = (size_t)M * nkv <= kApDirectPairs && (some ? max_prefix : 0) + (uint64_t)max_own <= kApDirectKeys &&
             (!track || (M == 1 && p.tiles_o == 1));
  if (p.row) p.tc = 0;
  // one range per row in all, and no unit that could reject a row: nothing to join either
  p.direct = p.row || (num_units == 0 && p.S_o == 1 && !track);
  const size_t mh = (size_t)M * nh, S = p.S_p + p.S_o;
  p.acc_floats = p.direct ? 0 : mh * S * hd;
  p.stat_floats = p.direct ? 0 : (mh * S * 2 + 3) / 4 * 4;
  p.lds = (int)((max_own + 3) / 4 * 4);
  p.score_floats = track ? mh * p.lds : 0;
  return p;
}

template <int HD, int WRP, int WRO>
int ap_launch_shape(ApArgs a, cudaStream_t st) {
  constexpr int kSmem = 4 * kApKeys * HD * 2;
  constexpr int kJoin = 64 * (HD + 4) * 4 + 64 * 8;  // WK x TR = 64 rows of O and their statistics
  constexpr int smem = kSmem > kJoin ? kSmem : kJoin;
  static bool attr_done[64] = {};
  const int dev = device_index();
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    ORCH_CUDA(cudaFuncSetAttribute(attn_prefix_kernel<HD, WRP, WRO>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    ORCH_CUDA(cudaFuncSetAttribute(attn_prefix_row_kernel<HD, WRO ? WRO : 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attr_done[dev] = true;
  }
  const dim3 none(0, 0, 0);
  if (a.row) {
    ORCH_CUDA(launch_k_serial(attn_prefix_row_kernel<HD, WRO ? WRO : 1>, dim3((unsigned)(a.M * a.nkv * a.tiles_o)), dim3(128), smem,
                              st, none, a));
    return check_launch("attention_prefix");
  }
  if (a.tc) {
    const int rc = ap_tc_launch(a, HD, st);
    if (rc != ORCH_OK) return rc;
    a.blocks_p = 0;
  }
  const size_t own = (size_t)a.M * a.nkv * a.S_o * a.tiles_o, blocks = (size_t)a.blocks_p + (WRO ? own : (own + 3) / 4) + (a.num_units > 0);
  if (blocks > 0x7fffffffu) return fail(ORCH_ERR_UNSUPPORTED, "attention_prefix: too many rows and heads for one launch");
  ORCH_CUDA(launch_k_pdl(a.tc != 0, attn_prefix_kernel<HD, WRP, WRO>, dim3((unsigned)blocks), dim3(128), smem, st, none, a));
  if (a.direct) return check_launch("attention_prefix");
  const int blocks_out = (int)(((size_t)a.M * a.nh + 3) / 4);
  const int chunks = a.mass ? (a.max_own + kMassEntries - 1) / kMassEntries : 0;
  const size_t jb = (size_t)blocks_out + (size_t)a.M * a.nkv * chunks;
  if (jb > 0x7fffffffu) return fail(ORCH_ERR_UNSUPPORTED, "attention_prefix: too many rows and heads for one launch");
  ORCH_CUDA(launch_k(attn_prefix_join_kernel<HD>, dim3((unsigned)jb), dim3(128), 0, st, none, a, blocks_out,
                     std::max(chunks, 1)));
  return check_launch("attention_prefix");
}

// A tile of a unit has at least the rows of a tile of one row, so wr_p >= wr_o; with head_dim 64
// or 128 it has 64 rows only where a row's heads already fill that.
template <int HD>
int ap_launch(const ApArgs& a, const ApPlan& plan, cudaStream_t st) {
  const int p = a.tc || a.row || a.blocks_p == 0 ? 0 : plan.wr_p;
  const int o = plan.by_warp ? 0 : plan.wr_o;
  if (p == 0)
    return o == 0 ? ap_launch_shape<HD, 0, 0>(a, st) : o == 1 ? ap_launch_shape<HD, 0, 1>(a, st)
         : o == 2 ? ap_launch_shape<HD, 0, 2>(a, st) : ap_launch_shape<HD, 0, 4>(a, st);
  if (p == 1) return o == 0 ? ap_launch_shape<HD, 1, 0>(a, st) : ap_launch_shape<HD, 1, 1>(a, st);
  if (p == 2)
    return o == 0 ? ap_launch_shape<HD, 2, 0>(a, st) : o == 1 ? ap_launch_shape<HD, 2, 1>(a, st) : ap_launch_shape<HD, 2, 2>(a, st);
  if constexpr (HD == 32) {
    if (o == 0) return ap_launch_shape<HD, 4, 0>(a, st);
    if (o == 1) return ap_launch_shape<HD, 4, 1>(a, st);
    if (o == 2) return ap_launch_shape<HD, 4, 2>(a, st);
  }
  return ap_launch_shape<HD, 4, 4>(a, st);
}

bool ap_shape_ok(uint32_t M, uint32_t nh, uint32_t nkv, uint32_t hd) {
  return nh > 0 && nkv > 0 && nh % nkv == 0 && nh <= 65535 && (hd == 32 || hd == 64 || hd == 128) &&
         (uint64_t)M * nh <= 0x7fffffffu;
}

}  // namespace

}  // namespace orch

using namespace orch;

extern "C" size_t orch_attention_prefix_workspace_bytes(uint32_t M, uint32_t num_heads, uint32_t num_kv_heads,
                                                        uint32_t head_dim, uint32_t num_units, uint32_t max_prefix,
                                                        uint32_t max_own, int track) {
  if (M == 0 || !ap_shape_ok(M, num_heads, num_kv_heads, head_dim)) return 0;
  return ap_plan(M, num_heads, num_kv_heads, head_dim, num_units, max_prefix, max_own, track).bytes();
}

// No counterpart in the reference, which attends per sequence over a host cache
// (orchard/model.py:112-144): the rows there share no keys and keep every position.
extern "C" int orch_attention_prefix(const void* q, const void* prefix_k, const void* prefix_v, const int32_t* units,
                                     uint32_t num_units, uint32_t max_prefix, uint32_t prefix_cap, uint32_t num_prefix,
                                     const void* k_cache, const void* v_cache, const int32_t* lens,
                                     const int32_t* slots, uint32_t max_own, uint32_t max_seq, uint32_t num_slots,
                                     float* mass, void* out, uint32_t M, uint32_t num_heads, uint32_t num_kv_heads,
                                     uint32_t head_dim, void* workspace, size_t workspace_bytes, void* stream) {
  if (M == 0) return ORCH_OK;
  ORCH_REQUIRE(q && k_cache && v_cache && lens && out, "attention_prefix: null pointer");
  ORCH_REQUIRE(num_units == 0 || max_prefix == 0 || (prefix_k && prefix_v && units), "attention_prefix: null prefix");
  ORCH_REQUIRE(num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0,
               "attention_prefix: num_heads must be a multiple of num_kv_heads");
  ORCH_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128, "attention_prefix: head_dim must be 32, 64 or 128");
  ORCH_REQUIRE(max_seq > 0 && max_seq <= kApMaxLen && num_slots > 0 && num_slots <= 0x7fffffffu && max_own <= max_seq,
               "attention_prefix: bad cache shape (max_own must not exceed max_seq)");
  ORCH_REQUIRE(num_units == 0 || max_prefix == 0 ||
                   (max_prefix <= prefix_cap && prefix_cap <= kApMaxLen && num_prefix > 0 && num_prefix <= 0x7fffffffu),
               "attention_prefix: bad prefix shape (max_prefix must not exceed prefix_cap)");
  ORCH_REQUIRE(num_units <= M, "attention_prefix: more units than rows (a row belongs to one at most)");
  ORCH_REQUIRE((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)prefix_k |
                 (uintptr_t)prefix_v | (uintptr_t)units | (uintptr_t)workspace) & 15) == 0,
               "attention_prefix: buffers must be 16-byte aligned");
  ORCH_REQUIRE((((uintptr_t)lens | (uintptr_t)slots | (uintptr_t)mass) & 3) == 0,
               "attention_prefix: lens, slots and mass must be 4-byte aligned");
  if (!ap_shape_ok(M, num_heads, num_kv_heads, head_dim))
    return fail(ORCH_ERR_UNSUPPORTED, "attention_prefix: too many rows and heads");
  const ApPlan p = ap_plan(M, num_heads, num_kv_heads, head_dim, num_units, max_prefix, max_own, mass != nullptr);
  ORCH_REQUIRE(workspace_bytes >= p.bytes() && (p.bytes() == 0 || workspace != nullptr),
               "attention_prefix: workspace too small");
  ApArgs a;
  a.q = static_cast<const __half*>(q);
  a.kp = static_cast<const __half*>(prefix_k);
  a.vp = static_cast<const __half*>(prefix_v);
  a.units = reinterpret_cast<const int4*>(units);
  a.num_units = units ? (int)num_units : 0;  // with max_prefix 0 they may be left out
  a.max_prefix = (int)max_prefix;
  a.prefix_cap = (int)prefix_cap;
  a.num_prefix = (int)num_prefix;
  a.kc = static_cast<const __half*>(k_cache);
  a.vc = static_cast<const __half*>(v_cache);
  a.lens = lens;
  a.slots = slots;
  a.max_own = (int)max_own;
  a.max_seq = (int)max_seq;
  a.num_slots = (int)num_slots;
  a.mass = mass;
  a.out = static_cast<__half*>(out);
  a.M = (int)M;
  a.nh = (int)num_heads;
  a.nkv = (int)num_kv_heads;
  a.G = p.G;
  a.tiles_p = p.tiles_p;
  a.tiles_o = p.tiles_o;
  a.S_p = p.S_p;
  a.blk_p = p.blk_p;
  a.tr_p = p.tr_p;
  for (a.tr_sh = 0; 1 << a.tr_sh < p.tr_p; ++a.tr_sh) {
  }
  a.tc = p.tc;
  a.S_o = p.S_o;
  const uint64_t blocks_p = (uint64_t)num_kv_heads * p.tiles_p * p.S_p;
  if (p.tc && (uint64_t)num_prefix * num_kv_heads * prefix_cap > 0x7fffff00u)
    return fail(ORCH_ERR_UNSUPPORTED, "attention_prefix: more than 2^31 prefix entries over all heads");
  if (blocks_p > 0x7fffffffu) return fail(ORCH_ERR_UNSUPPORTED, "attention_prefix: too many units for one launch");
  a.blocks_p = (int)blocks_p;
  a.direct = p.direct;
  a.row = p.row;
  a.acc = static_cast<float*>(workspace);
  a.stat = reinterpret_cast<float2*>(a.acc + p.acc_floats);
  a.scores = a.acc + p.acc_floats + p.stat_floats;
  a.lds = p.lds;
  ORCH_CHECK_WORD(a.check);
  cudaStream_t st = as_stream(stream);
  switch (head_dim) {
    case 32: return ap_launch<32>(a, p, st);
    case 64: return ap_launch<64>(a, p, st);
    default: return ap_launch<128>(a, p, st);
  }
}
