// The prefix part of orch_attention_prefix on the 5th-generation tensor cores, for units with
// many query rows: S = Q K^T and O += P V as tcgen05.mma with fp32 accumulators in tensor
// memory, 128 query rows (rows x heads of one K/V head) by 128 keys at a time.
//
// Mathematics as in attention_prefix.cu. With 128 rows a block is 12.6 MFLOP (the scores, and V
// with each of the weights' two terms) against 64 KB of K and V, past what mma.sync tiles sustain.
// Per block the products take ~1,580 cycles of the tensor pipe (24 of 66) and the 16,384
// exponentials 1,024 cycles of the special-function units; two groups of four warps keep both busy,
// one turning scores into weights while the tensor pipe works for the other. A unit of up to 128
// query rows gives the groups alternate blocks of keys; with more (PAIR) a CTA takes 256 rows, a
// group 128 of them and every block: each block then serves twice the rows, which halves the
// traffic from L2. 128 CTAs at once take 1.4 us per block with 128 rows, 2.5 with 256; head_dim 64
// 1.3 and 2.1.
//  * a producer thread brings K and V blocks by TMA (128-byte swizzle; K rows are the K-major
//    operand of Q K^T, V rows the MN-major operand of P V), two slots each;
//  * one warp issues the products, a lane elected at each;
//  * a thread of a group owns one query row and holds a block's 128 scores in registers: maximum,
//    weights and sum need no shuffles. A row's weights are scaled by `ref`, which moves only when
//    a maximum exceeds it by more than 2^7 (held weights then reach 2^15 at most; any scale
//    gives the same quotient); then the accumulator is rescaled before the block's product.
//    Each weight is held in two fp16 terms, hi = fp16(p) and lo = fp16(p - hi), 22 bits together:
//    one alone would be off by up to 2^-11 of the weight, as much as the output's own rounding.
// The weights of a block lie over the scores they came from, whose 128 columns their two terms
// fill. Alternate blocks share one accumulator and take three score buffers in turn: the scores of
// block i + 2 go where block i - 1's weights were, under way while block i's become weights;
// `ref` passes from block to block through shared memory right after each maximum. With PAIR each
// group has its own accumulator and one buffer.
// The CTA writes one record per row for the join. Keys past the range are masked, their V rows
// zeroed in shared memory (whatever lies there in the prefix region could be a NaN).
//
// Tensor memory (512 columns): score buffers at 0, 128 and 256 and the accumulator at 384, or
// (PAIR) at 0 and 128, accumulators at 256 and 256 + HD. Each 32 keys of a buffer's weights have
// the 16 columns of their hi terms, then the 16 of their lo terms. Every mbarrier wait is bounded;
// one that runs out sets device check bit 256.
#include "attention_prefix.cuh"
#include "tcgen05.cuh"

namespace orch {

namespace {

constexpr int kPtThreads = 320;  // two groups of four warps, the producer, the issuer
constexpr float kPtShift = 8.f, kPtGrow = 7.f;

template <int HD, bool PAIR>
struct PtCfg {
  static constexpr int Rows = PAIR ? 2 * kApTcRows : kApTcRows;
  static constexpr int Atom = kApTcRows * 128;  // 128 rows of one 64-dim swizzle atom
  static constexpr int Tile = Atom * (HD / 64);  // 128 rows of Q, or a block of K or V
  static constexpr int OffK = Tile * (Rows / kApTcRows), OffV = OffK + 2 * Tile, OffBar = OffV + 2 * Tile;
  static constexpr int OP = HD + 4;  // row pitch of the accumulators' staging (floats)
  static constexpr int OffStat = Rows * OP * 4;
  static constexpr int Bytes = (OffStat + 2 * kApTcRows * 8 > OffBar ? OffStat + 2 * kApTcRows * 8 : OffBar);
  static constexpr int OffRef = Bytes + 256;  // a row's ref (floats), behind the barriers
  static constexpr int OffRec = OffRef + kApTcRows * 4;  // a row's number among all (row, head) pairs
  static constexpr int Smem = OffRec + Rows * 4;
  static constexpr int Bufs = PAIR ? 2 : 3;                                  // score buffers of 128 columns
  static constexpr uint32_t ColO = PAIR ? 256 : 384, StepO = PAIR ? HD : 0;  // accumulator of group g
};

__device__ __forceinline__ void pt_groups_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int HD, bool PAIR>
__global__ void __launch_bounds__(kPtThreads, 1)
    attn_prefix_tc_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                          const ApArgs a) {
  using C = PtCfg<HD, PAIR>;
  constexpr uint32_t kIdescS = umma_idesc_f16<kApTcKeys>(), kIdescO = umma_idesc_f16<HD>() | kIdescBMn;
  extern __shared__ __align__(1024) uint8_t sm[];
  uint8_t* sK = sm + C::OffK;
  uint8_t* sV = sm + C::OffV;
  uint64_t* kfull = reinterpret_cast<uint64_t*>(sm + C::Bytes);
  uint64_t* vfull = kfull + 2;
  // Of a score buffer; a buffer's phases are its blocks. (Barriers by the block's parity would not
  // do: three blocks are under way, and a parity names one of two phases.)
  uint64_t* sready = vfull + 2;   // scores written: also (not PAIR) the K slot is free
  uint64_t* pready = sready + 3;  // [buffer][half]: weights of the block's first and last 64 keys
  uint64_t* pvdone = pready + 6;  // weights used: also (not PAIR) the V slot is free
  uint64_t* refset = pvdone + 3;  // [group][warp of the group]: the rows' ref after its block
  uint64_t* kfree = refset + 8;   // [slot], PAIR: the last group's product has read the slot
  uint64_t* vfree = kfree + 2;
  uint64_t* drain = vfree + 2;  // every product issued has ended
  uint64_t* qfull = drain + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(qfull + 1);
  volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);

  float* refs = reinterpret_cast<float*>(sm + C::OffRef);

  pdl_wait();
  // The own entries' kernel, launched next, may start once every CTA is here; it does not read
  // what this kernel writes, and everything before this kernel has completed.
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int b = blockIdx.x;  // row tiles fastest: the tiles that read the same keys run together
  const int tile = b % a.tiles_p;
  b /= a.tiles_p;
  const int kv = b % a.nkv, split = b / a.nkv;
  int4 u;
  const int i0 = ap_find_tile(a, tile, u);
  if (i0 < 0) return;
  const int n = min(C::Rows, u.y * a.G - i0);
  const int per = ap_range(u.w, a.S_p, a.blk_p), j0 = split * per, j1 = min(u.w, j0 + per);
  if (j0 >= j1) return;
  const int nb = (j1 - j0 + kApTcKeys - 1) / kApTcKeys;

  if (warp == 8) tmem_alloc(tmem_slot, 512);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&kfull[i], 1);
      mbar_init(&vfull[i], 1);
      mbar_init(&kfree[i], 1);
      mbar_init(&vfree[i], 1);
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(&sready[i], 1);
      mbar_init(&pready[2 * i], 4);  // one lane per warp of the group
      mbar_init(&pready[2 * i + 1], 4);
      mbar_init(&pvdone[i], 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&refset[i], 1);
    mbar_init(drain, 1);
    mbar_init(qfull, 8);  // one lane per warp of the groups
    *failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int grp = warp >> 2, row = (warp & 3) * 32 + lane;
  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
  const int groups = PAIR && n <= kApTcRows ? 1 : 2;  // groups at work; the last one frees the slots
  const int mine = grp >= groups ? 0 : PAIR ? nb : (nb - grp + 1) / 2;  // blocks of this group
  float ref = -INFINITY, l = 0.f;
  if (warp == 8) {
    if (lane == 0) {
      const int y0 = (u.z * a.nkv + kv) * a.prefix_cap + j0;
      int ik = 0, iv = 0;
      auto load = [&](uint8_t* to, const CUtensorMap* map, uint64_t* bar, int i) {
        mbar_expect_tx(bar, (uint32_t)C::Tile);
        for (int d = 0; d < HD / 64; ++d) tma_load_2d(to + (i & 1) * C::Tile + d * C::Atom, map, bar, d * 64, y0 + i * kApTcKeys);
      };
      // A slot is free after the products of two blocks before; in the order in which they end. The
      // barriers waited for pass once for each use of a slot, so none can be two phases ahead (a
      // parity would name the wrong one): the next use is this thread's own.
      auto load_k = [&](int i) {
        uint64_t* bar = PAIR ? &kfree[i & 1] : &sready[(i - 2) % 3];
        const int phase = PAIR ? (i >> 1) - 1 : (i - 2) / 3;
        if (i >= 2 && !mbar_wait_f(bar, (uint32_t)phase & 1, failed)) return false;
        load(sK, &tmk, &kfull[i & 1], i);
        ik = i + 1;
        return true;
      };
      auto load_v = [&](int i) {
        uint64_t* bar = PAIR ? &vfree[i & 1] : &pvdone[(i - 2) % 3];
        const int phase = PAIR ? (i >> 1) - 1 : (i - 2) / 3;
        if (i >= 2 && !mbar_wait_f(bar, (uint32_t)phase & 1, failed)) return false;
        load(sV, &tmv, &vfull[i & 1], i);
        iv = i + 1;
        return true;
      };
      bool ok = load_k(0);
      for (int i = 0; ok && i < nb; ++i) {
        if (PAIR)
          ok = load_v(i) && (i + 1 >= nb || load_k(i + 1));
        else
          ok = (i + 1 >= nb || load_k(i + 1)) && load_v(i);
      }
      if (!ok) *failed = 1;
      // whoever gave up, no load may still be in flight when the CTA ends
      for (int i = max(0, ik - 2); i < ik; ++i) mbar_wait(&kfull[i & 1], (uint32_t)(i >> 1) & 1);
      for (int i = max(0, iv - 2); i < iv; ++i) mbar_wait(&vfull[i & 1], (uint32_t)(i >> 1) & 1);
    }
    __syncwarp();
  } else if (warp == 9) {
    // every lane waits and computes the descriptors, an elected one issues
    auto wait = [&](uint64_t* bar, int phase) {
      return __all_sync(0xffffffffu, mbar_wait_f(bar, (uint32_t)phase & 1, failed)) != 0;
    };
    // The waits for K and V (`arrived`) are placed where products are running, not before them.
    auto arrived = [&](uint64_t* full, int i) { return i >= nb || wait(&full[i & 1], i >> 1); };
    // block i's scores into buffer b, from rows 128 g of the tile (PAIR: g is b) or all of them
    auto scores = [&](int b, int i) {
      tc_fence_after();
      uint8_t* q = sm + (PAIR ? b * C::Tile : 0);
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
        umma_f16_ss_warp(tmem + b * 128, sw128_desc(smem_u32(q + (kk >> 2) * C::Atom)) + 2 * (kk & 3),
                         sw128_desc(smem_u32(sK + (i & 1) * C::Tile + (kk >> 2) * C::Atom)) + 2 * (kk & 3), kIdescS, kk > 0);
      umma_commit_warp(&sready[b]);
      if (PAIR && b == groups - 1 && i + 2 < nb) umma_commit_warp(&kfree[i & 1]);
    };
    // accumulator of buffer b's group += weights of block i . V, as the two halves of the weights come
    auto weigh = [&](int b, int i, int phase) {
      const uint32_t d = tmem + C::ColO + (PAIR ? b * C::StepO : 0), p = tmem + b * 128;
      const uint64_t v = sw128_desc_mn(smem_u32(sV + (i & 1) * C::Tile), C::Atom);  // 16 keys are 2,048 B
      const int steps = (min(kApTcKeys, j1 - j0 - i * kApTcKeys) + 15) / 16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!wait(&pready[2 * b + h], phase)) return false;
        tc_fence_after();
        if (steps >= 4 * h + 4) {
#pragma unroll
          for (int kk = 4 * h; kk < 4 * h + 4; ++kk) {
            umma_f16_ta_warp(d, p + (kk >> 1) * 32 + (kk & 1) * 8, v + kk * 128, kIdescO, i > 0 || kk > 0);
            umma_f16_ta_warp(d, p + (kk >> 1) * 32 + (kk & 1) * 8 + 16, v + kk * 128, kIdescO, 1);
          }
        } else {  // the last block: steps of 16 keys past the range are left out
          for (int kk = 4 * h; kk < steps; ++kk) {
            umma_f16_ta_warp(d, p + (kk >> 1) * 32 + (kk & 1) * 8, v + kk * 128, kIdescO, i > 0 || kk > 0);
            umma_f16_ta_warp(d, p + (kk >> 1) * 32 + (kk & 1) * 8 + 16, v + kk * 128, kIdescO, 1);
          }
        }
      }
      umma_commit_warp(&pvdone[b]);
      if (PAIR && b == groups - 1 && i + 2 < nb) umma_commit_warp(&vfree[i & 1]);
      return true;
    };
    bool ok = arrived(kfull, 0) && wait(qfull, 0);
    if (ok) scores(0, 0);
    if (PAIR) {
      if (ok && groups > 1) scores(1, 0);
      ok = ok && arrived(vfull, 0);
      for (int i = 0; ok && i < nb; ++i)
        for (int g = 0; ok && g < groups; ++g) {
          ok = weigh(g, i, i) && (g > 0 || arrived(kfull, i + 1));
          if (!ok || i + 1 >= nb) continue;
          // the next scores overwrite the weights: wait until they have been used
          ok = wait(&pvdone[g], i);
          if (!ok) break;
          scores(g, i + 1);
          if (g == groups - 1) ok = arrived(vfull, i + 1);
        }
    } else {
      ok = ok && arrived(kfull, 1);
      if (ok && nb > 1) scores(1, 1);
      ok = ok && arrived(vfull, 0);
      int b = 0, b2 = 2, phase = 0, before = 0;  // block i's buffer and phase, block i + 2's buffer, block i - 1's phase
      for (int i = 0; ok && i < nb; ++i) {
        if (i + 2 < nb) {  // into the buffer of block i - 1, once its weights have been used
          ok = arrived(kfull, i + 2) && (i == 0 || wait(&pvdone[b2], before));
          if (ok) scores(b2, i + 2);
        }
        ok = ok && weigh(b, i, phase) && arrived(vfull, i + 1);
        b2 = b;
        before = phase;
        if (++b == 3) b = 0, ++phase;
      }
    }
    if (!ok) *failed = 1;
    // Whoever gave up, no product may still be running when tensor memory is freed; some may have no
    // commit of their own (a block's first half, when its second half's weights did not come).
    umma_commit_warp(drain);
    mbar_wait(drain, 0);
    __syncwarp();
  } else {
    if (tid < n) reinterpret_cast<int*>(sm + C::OffRec)[tid] = (u.x + (i0 + tid) / a.G) * a.nh + kv * a.G + (i0 + tid) % a.G;
    // Q rows into their swizzled places: 16-byte piece c of a 128-byte row r at c ^ (r & 7).
    // Up to eight pieces per thread are requested before the first is stored.
    constexpr int Pieces = C::Rows * (HD / 8) / 256, Batch = Pieces < 8 ? Pieces : 8;
    static_assert(C::Rows * (HD / 8) % (256 * Batch) == 0, "whole batches");
#pragma unroll
    for (int x0 = 0; x0 < Pieces; x0 += Batch) {
      uint4 v[Batch];
#pragma unroll
      for (int x = 0; x < Batch; ++x) {
        const int i = tid + (x0 + x) * 256, r = i / (HD / 8), c = i % (HD / 8);
        v[x] = make_uint4(0u, 0u, 0u, 0u);
        if (r < n) {
          const int m = u.x + (i0 + r) / a.G, h = kv * a.G + (i0 + r) % a.G;
          v[x] = *reinterpret_cast<const uint4*>(a.q + ((size_t)m * a.nh + h) * HD + c * 8);
        }
      }
#pragma unroll
      for (int x = 0; x < Batch; ++x) {
        const int i = tid + (x0 + x) * 256, r = i / (HD / 8), c = i % (HD / 8);
        *reinterpret_cast<uint4*>(sm + (r >> 7) * C::Tile + (c >> 3) * C::Atom + (r & 127) * 128 + ((c & 7) ^ (r & 7)) * 16) = v[x];
      }
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(qfull);

    const float scale = rsqrtf((float)HD) * 1.4426950408889634f;  // scores in powers of two
    const uint32_t to = tmem + lanes + C::ColO + grp * C::StepO;
    const int q = warp & 3;
    auto wait = [&](uint64_t* bar, int phase) {
      return __all_sync(0xffffffffu, mbar_wait_f(bar, (uint32_t)phase & 1, failed)) != 0;
    };
    // the product of block i with its V has ended
    auto product = [&](int i) { return PAIR ? wait(&pvdone[grp], i) : wait(&pvdone[i % 3], i / 3); };
    for (int k = 0; k < mine; ++k) {
      const int i = PAIR ? k : 2 * k + grp, keys = min(kApTcKeys, j1 - j0 - i * kApTcKeys);
      const int before = grp ? k : k - 1;  // the other group's last block before this one
      const int buf = PAIR ? grp : i % 3;
      const uint32_t ts = tmem + lanes + buf * 128;
      if (!wait(&sready[buf], PAIR ? i : i / 3)) {
        *failed = 1;
        break;
      }
      tc_fence_after();
      uint32_t s[2][64];
      tmem_ld64(ts, s[0]);
      tmem_ld64(ts + 64, s[1]);
      if (keys < kApTcKeys) {
#pragma unroll
        for (int e = 0; e < 128; ++e)
          if (e >= keys) s[e >> 6][e & 63] = 0xff800000u;  // -inf
      }
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 128; ++e) m4[e & 3] = fmaxf(m4[e & 3], __uint_as_float(s[e >> 6][e & 63]));
      const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * scale;
      float in = ref;
      if (!PAIR && i > 0) {
        if (!wait(&refset[(grp ^ 1) * 4 + q], before)) {
          *failed = 1;
          break;
        }
        in = refs[row];
      }
      const float now = mx > in + kPtGrow || i == 0 ? mx : in;
      if (!PAIR) {
        refs[row] = now;
        __syncwarp();
        if (lane == 0) mbar_arrive(&refset[grp * 4 + q]);
      }
      if (__any_sync(0xffffffffu, i > 0 && now != in)) {
        // This block moves the scale: every earlier product has to be in the accumulator. (With
        // PAIR it is: these scores came after it. Otherwise block i - 1's may not be; its barrier's
        // phase before, block i - 4's, has ended, as these scores came after block i - 3's product.)
        if (!PAIR && !product(i - 1)) {
          *failed = 1;
          break;
        }
        tc_fence_after();
        const float f = now == in ? 1.f : ap_exp2(in - now);
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(to + 32 * c, o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmem_st32(to + 32 * c, o);
        }
      }
      if (now != ref) l *= ap_exp2(ref - now);
      ref = now;
      const float off = now == -INFINITY ? 0.f : now - kPtShift;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      bool good = true;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t p[32];  // hi terms of 32 keys, then their lo terms
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float p0 = ap_exp2(fmaf(__uint_as_float(s[h][32 * c + 2 * e]), scale, -off));
            const float p1 = ap_exp2(fmaf(__uint_as_float(s[h][32 * c + 2 * e + 1]), scale, -off));
            sum[(2 * e) & 3] += p0;
            sum[(2 * e + 1) & 3] += p1;
            const __half2 hi = __floats2half2_rn(p0, p1);
            const float2 f = __half22float2(hi);
            p[e] = h2_bits(hi);
            p[16 + e] = h2_bits(__floats2half2_rn(p0 - f.x, p1 - f.y));
          }
          tmem_st32(ts + 64 * h + 32 * c, p);
        }
        if (h == 0 && keys < kApTcKeys) {  // the V rows of the last step that lie past the range
          good = wait(&vfull[i & 1], i >> 1);
          if (!good) break;
          const int end = (keys + 15) / 16 * 16, pieces = (end - keys) * (HD / 8);
          for (int x = row; x < pieces; x += 128) {
            const int r = keys + x / (HD / 8), c = x % (HD / 8);
            *reinterpret_cast<uint4*>(sV + (i & 1) * C::Tile + (c >> 3) * C::Atom + r * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pready[2 * buf + h]);
      }
      if (!good) {
        *failed = 1;
        break;
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
    if (mine > 0 && !product(PAIR ? nb - 1 : 2 * mine - 2 + grp)) *failed = 1;
    tc_fence_before();
  }
  if (grp < 2) {
    pt_groups_sync();  // both groups' products have ended: every slot is free
    tc_fence_after();
    const bool good = __all_sync(0xffffffffu, !*failed);
    float* os = reinterpret_cast<float*>(sm);  // [rows][OP]
    float2* ss = reinterpret_cast<float2*>(sm + C::OffStat);  // [group][128]: (ref, sum)
    if (good && (!PAIR || mine > 0)) {
      // PAIR: a group's own accumulator; otherwise half of the columns each
      constexpr int Steps = PAIR ? HD / 32 : HD / 64;
      const int col0 = PAIR ? 0 : grp * (HD / 2);
      float* w = os + ((PAIR ? grp * kApTcRows : 0) + row) * C::OP + col0;
#pragma unroll
      for (int c = 0; c < Steps; ++c) {
        uint32_t o[32];
        tmem_ld32(tmem + lanes + C::ColO + grp * C::StepO + col0 + 32 * c, o);
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          *reinterpret_cast<uint4*>(w + 32 * c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      }
      ss[grp * kApTcRows + row] = make_float2(ref, l);
    }
    pt_groups_sync();
    constexpr int LPR = HD / 4;  // threads per row, four values each
    const int S = a.S_p + a.S_o;
    // the other kernels' records hold weights as 2^kApShift e^(s - max): the same scale here
    const float g = exp2f(kApShift - kPtShift);
    const int* recs = reinterpret_cast<const int*>(sm + C::OffRec);
#pragma unroll 4
    for (int i = tid; i < (good ? n * LPR : 0); i += 256) {
      const int r = i / LPR, d = (i % LPR) * 4;
      const float4 ov = *reinterpret_cast<const float4*>(os + r * C::OP + d);
      *reinterpret_cast<float4*>(a.acc + ((size_t)recs[r] * S + split) * HD + d) = make_float4(ov.x * g, ov.y * g, ov.z * g, ov.w * g);
    }
    if (good && tid < n) {
      const int r = tid;
      float2 st = ss[r];
      if (!PAIR) {  // the groups' sums, at the last block's ref
        const float at = refs[r];
        const float2 s1 = nb > 1 ? ss[kApTcRows + r] : make_float2(at, 0.f);
        st.y = (st.x == at ? st.y : st.y * ap_exp2(st.x - at)) + (s1.x == at ? s1.y : s1.y * ap_exp2(s1.x - at));
        st.x = at;
      }
      a.stat[(size_t)recs[r] * S + split] = make_float2(st.x, st.y * g);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_dealloc(tmem, 512);
  if (tid == 0 && *failed) atomicOr(a.check, 256u);
}

template <int HD, bool PAIR>
int pt_launch(const ApArgs& a, cudaStream_t st) {
  using C = PtCfg<HD, PAIR>;
  static bool attr_done[64] = {};
  const int dev = device_index();
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    ORCH_CUDA(cudaFuncSetAttribute(attn_prefix_tc_kernel<HD, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::Smem));
    attr_done[dev] = true;
  }
  if (!encode_fn()) return fail(ORCH_ERR_CUDA, "attention_prefix: no tensor-map encoder");
  const uint64_t rows = (uint64_t)a.num_prefix * a.nkv * a.prefix_cap;
  CUtensorMap mk, mv;
  if (!encode2d(&mk, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.kp, HD, rows, HD * 2, 64, kApTcKeys, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode2d(&mv, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.vp, HD, rows, HD * 2, 64, kApTcKeys, CU_TENSOR_MAP_SWIZZLE_128B))
    return fail(ORCH_ERR_CUDA, "attention_prefix: tensor map");
  ORCH_CUDA(launch_k_serial(attn_prefix_tc_kernel<HD, PAIR>, dim3((unsigned)a.blocks_p), dim3(kPtThreads), C::Smem, st,
                            dim3(0, 0, 0), mk, mv, a));
  return check_launch("attention_prefix");
}

}  // namespace

int ap_tc_launch(const ApArgs& a, int hd, cudaStream_t st) {
  const bool pair = a.tr_p > kApTcRows;
  if (hd == 64) return pair ? pt_launch<64, true>(a, st) : pt_launch<64, false>(a, st);
  return pair ? pt_launch<128, true>(a, st) : pt_launch<128, false>(a, st);
}

}  // namespace orch
