// The prefix part of orch_attention_prefix on the 5th-generation tensor cores, for units with
// many query rows: S = Q K^T and O += P V as tcgen05.mma with fp32 accumulators in tensor
// memory, 128 query rows (rows x heads of one K/V head) by 128 keys at a time.
//
// Mathematics as in attention_prefix.cu. With 128 rows a block is 8.4 MFLOP against 64 KB of K
// and V, past what mma.sync tiles sustain; here the matrix products take ~1,050 cycles of the
// tensor pipe and the 16,384 exponentials 1,024 cycles of the special-function units, so the
// two are kept busy by two groups of four warps that take alternate blocks: while one group
// turns its scores into weights, the tensor pipe works for the other.
//  * a producer thread brings K and V blocks by TMA (128-byte swizzle; K rows are the K-major
//    operand of Q K^T, V rows the MN-major operand of P V), two slots each;
//  * one thread issues the products; group w's scores, weights and accumulator have their own
//    tensor-memory columns, the weights (fp16) over the scores they came from;
//  * a thread of a group owns one query row: maximum, weights and sum need no shuffles. The
//    accumulator is rescaled only when the row's maximum has grown by more than 2^7 since the
//    value it is scaled by (held weights then reach 2^15 at most, and stay normal down to
//    2^-22 of the largest); any scale gives the same quotient.
// The groups' two accumulators meet in shared memory at the end, and the CTA writes one record
// of its key range for the join. Keys past the range are masked, their V rows zeroed in shared
// memory (whatever lies there in the prefix region could be a NaN).
//
// Tensor memory (512 columns): scores 0 and 1 at 0 and 128, accumulators at 256 and 256 + HD.
// Every mbarrier wait is bounded; one that runs out sets device check bit 256.
#include "attention_prefix.cuh"
#include "tcgen05.cuh"

namespace orch {

namespace {

constexpr int kPtThreads = 320;  // two groups of four warps, the producer, the issuer
constexpr float kPtShift = 8.f, kPtGrow = 7.f;

template <int HD>
struct PtCfg {
  static constexpr int Atom = kApTcRows * 128;  // 128 rows of one 64-dim swizzle atom
  static constexpr int Tile = Atom * (HD / 64);  // Q, or a block of K or V
  static constexpr int OffK = Tile, OffV = OffK + 2 * Tile, OffBar = OffV + 2 * Tile;
  static constexpr int OP = HD + 4;  // row pitch of the accumulators' staging (floats)
  static constexpr int OffStat = 2 * kApTcRows * OP * 4;
  static constexpr int Bytes = (OffStat + 2 * kApTcRows * 8 > OffBar ? OffStat + 2 * kApTcRows * 8 : OffBar);
  static constexpr int Smem = 1024 + Bytes + 256;
  static constexpr uint32_t O0 = 256;
};

__device__ __forceinline__ void pt_groups_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int HD>
__global__ void __launch_bounds__(kPtThreads, 1)
    attn_prefix_tc_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                          const ApArgs a) {
  using C = PtCfg<HD>;
  constexpr uint32_t kIdescS = umma_idesc_f16<kApTcKeys>(), kIdescO = umma_idesc_f16<HD>() | kIdescBMn;
  extern __shared__ uint8_t pt_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pt_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sK = sm + C::OffK;
  uint8_t* sV = sm + C::OffV;
  uint64_t* kfull = reinterpret_cast<uint64_t*>(sm + C::Bytes);
  uint64_t* vfull = kfull + 2;
  uint64_t* sready = vfull + 2;  // scores written: also, the K slot is free
  uint64_t* pready = sready + 2;
  uint64_t* pvdone = pready + 2;  // weights used: also, the V slot and the scores' columns are free
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pvdone + 2);
  volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);

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
  if (!ap_unit_ok(a, u)) {
    if (tid == 0) atomicOr(a.check, u.z < 0 || u.z >= a.num_prefix ? 8u : 2u);
    return;
  }
  const int n = min(kApTcRows, u.y * a.G - i0);
  const int per = ap_range(u.w, a.S_p, a.blk_p), j0 = split * per, j1 = min(u.w, j0 + per);
  if (j0 >= j1) return;
  const int nb = (j1 - j0 + kApTcKeys - 1) / kApTcKeys;

  if (warp == 8) tmem_alloc(tmem_slot, 512);
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&kfull[i], 1);
      mbar_init(&vfull[i], 1);
      mbar_init(&sready[i], 1);
      mbar_init(&pready[i], 4);  // one elected lane per warp of the group
      mbar_init(&pvdone[i], 1);
    }
    *failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // Q rows into their swizzled places: 16-byte piece c of a 128-byte row r at c ^ (r & 7)
  for (int i = tid; i < kApTcRows * (HD / 8); i += kPtThreads) {
    const int r = i / (HD / 8), c = i % (HD / 8);
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (r < n) {
      const int m = u.x + (i0 + r) / a.G, h = kv * a.G + (i0 + r) % a.G;
      v = *reinterpret_cast<const uint4*>(a.q + ((size_t)m * a.nh + h) * HD + c * 8);
    }
    *reinterpret_cast<uint4*>(sm + (c >> 3) * C::Atom + r * 128 + ((c & 7) ^ (r & 7)) * 16) = v;
  }
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int grp = warp >> 2, row = (warp & 3) * 32 + lane;
  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
  const int mine = grp < 2 ? (nb - grp + 1) / 2 : 0;  // blocks of this group
  float ref = -INFINITY, l = 0.f;
  if (warp == 8) {
    if (lane == 0) {
      const int y0 = (u.z * a.nkv + kv) * a.prefix_cap + j0;
      int ik = 0, iv = 0;
      for (int i = 0; i < nb && !*failed; ++i) {
        const int w = i & 1;
        const uint32_t ph = (uint32_t)((i >> 1) - 1) & 1;
        if (i >= 2 && !mbar_wait_f(&sready[w], ph, failed)) {
          *failed = 1;
          break;
        }
        mbar_expect_tx(&kfull[w], (uint32_t)C::Tile);
        for (int d = 0; d < HD / 64; ++d) tma_load_2d(sK + w * C::Tile + d * C::Atom, &tmk, &kfull[w], d * 64, y0 + i * kApTcKeys);
        ik = i + 1;
        if (i >= 2 && !mbar_wait_f(&pvdone[w], ph, failed)) {
          *failed = 1;
          break;
        }
        mbar_expect_tx(&vfull[w], (uint32_t)C::Tile);
        for (int d = 0; d < HD / 64; ++d) tma_load_2d(sV + w * C::Tile + d * C::Atom, &tmv, &vfull[w], d * 64, y0 + i * kApTcKeys);
        iv = i + 1;
      }
      if (*failed) {  // loads still in flight when the others gave up
        for (int i = max(0, ik - 2); i < ik; ++i) mbar_wait(&kfull[i & 1], (uint32_t)(i >> 1) & 1);
        for (int i = max(0, iv - 2); i < iv; ++i) mbar_wait(&vfull[i & 1], (uint32_t)(i >> 1) & 1);
      }
    }
    __syncwarp();
  } else if (warp == 9) {
    if (lane == 0) {
      int issued_s[2] = {0, 0}, issued_o[2] = {0, 0};
      auto scores = [&](int i) {
        const int w = i & 1;
        if (!mbar_wait_f(&kfull[w], (uint32_t)(i >> 1) & 1, failed)) return false;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          umma_f16_ss(tmem + w * 128, sw128_desc(smem_u32(sm + (kk >> 2) * C::Atom)) + 2 * (kk & 3),
                      sw128_desc(smem_u32(sK + w * C::Tile + (kk >> 2) * C::Atom)) + 2 * (kk & 3), kIdescS, kk > 0);
        umma_commit(&sready[w]);
        ++issued_s[w];
        return true;
      };
      bool ok = scores(0) && (nb < 2 || scores(1));
      for (int i = 0; ok && i < nb; ++i) {
        const int w = i & 1;
        const uint32_t ph = (uint32_t)(i >> 1) & 1;
        ok = mbar_wait_f(&pready[w], ph, failed) && mbar_wait_f(&vfull[w], ph, failed);
        if (!ok) break;
        tc_fence_after();
        // the last block's keys past the range: whole steps of 16 are left out
        const int steps = min(kApTcKeys, (j1 - j0 - i * kApTcKeys + 15) / 16 * 16) / 16;
        for (int kk = 0; kk < steps; ++kk)
          umma_f16_ta(tmem + C::O0 + w * HD, tmem + w * 128 + kk * 8,
                      sw128_desc_mn(smem_u32(sV + w * C::Tile + kk * 2048), C::Atom), kIdescO, (i >= 2 || kk > 0) ? 1u : 0u);
        umma_commit(&pvdone[w]);
        ++issued_o[w];
        if (i + 2 < nb) {
          // the next scores overwrite the weights: wait until they have been used
          ok = mbar_wait_f(&pvdone[w], ph, failed) && scores(i + 2);
        }
      }
      if (!ok) {
        *failed = 1;
        for (int w = 0; w < 2; ++w) {  // products still running
          if (issued_s[w]) mbar_wait(&sready[w], (uint32_t)(issued_s[w] - 1) & 1);
          if (issued_o[w]) mbar_wait(&pvdone[w], (uint32_t)(issued_o[w] - 1) & 1);
        }
      }
    }
    __syncwarp();
  } else {
    const float scale = rsqrtf((float)HD) * 1.4426950408889634f;  // scores in powers of two
    const uint32_t ts = tmem + lanes + grp * 128, to = tmem + lanes + C::O0 + grp * HD;
    for (int k = 0; k < mine; ++k) {
      const int i = 2 * k + grp, keys = min(kApTcKeys, j1 - j0 - i * kApTcKeys);
      if (!__all_sync(0xffffffffu, mbar_wait_f(&sready[grp], (uint32_t)k & 1, failed))) {
        *failed = 1;
        break;
      }
      tc_fence_after();
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t s[32];
        tmem_ld32(ts + 32 * c, s);
        if (keys == kApTcKeys) {
#pragma unroll
          for (int e = 0; e < 32; ++e) mx = fmaxf(mx, __uint_as_float(s[e]));
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (32 * c + e < keys) mx = fmaxf(mx, __uint_as_float(s[e]));
        }
      }
      mx *= scale;
      const bool grow = k > 0 && mx > ref + kPtGrow;
      if (__any_sync(0xffffffffu, grow)) {  // rescale the accumulator (its last product is done)
        const float f = grow ? ap_exp2(ref - mx) : 1.f;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(to + 32 * c, o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmem_st32(to + 32 * c, o);
        }
        l *= f;
      }
      if (k == 0 || grow) ref = mx;
      const float off = ref == -INFINITY ? 0.f : ref - kPtShift;
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t s[32], p[16];
        tmem_ld32(ts + 32 * c, s);
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float v = ap_exp2(fmaf(__uint_as_float(s[e]), scale, -off));
          s[e] = __float_as_uint(keys == kApTcKeys || 32 * c + e < keys ? v : 0.f);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p0 = __uint_as_float(s[2 * e]), p1 = __uint_as_float(s[2 * e + 1]);
          sum += p0 + p1;
          p[e] = h2_bits(__floats2half2_rn(p0, p1));
        }
        tmem_st16(ts + 16 * c, p);  // over scores already read
      }
      l += sum;
      if (keys < kApTcKeys) {  // the V rows of the last step that lie past the range
        if (!__all_sync(0xffffffffu, mbar_wait_f(&vfull[grp], (uint32_t)k & 1, failed))) {
          *failed = 1;
          break;
        }
        const int end = (keys + 15) / 16 * 16, pieces = (end - keys) * (HD / 8);
        for (int x = row; x < pieces; x += 128) {
          const int r = keys + x / (HD / 8), c = x % (HD / 8);
          *reinterpret_cast<uint4*>(sV + grp * C::Tile + (c >> 3) * C::Atom + r * 128 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pready[grp]);
    }
    if (mine > 0 && !*failed && !mbar_wait_f(&pvdone[grp], (uint32_t)(mine - 1) & 1, failed)) *failed = 1;
    tc_fence_after();
  }
  if (grp < 2) {
    pt_groups_sync();  // both groups' products have ended: every slot is free
    const bool good = __all_sync(0xffffffffu, !*failed);
    float* os = reinterpret_cast<float*>(sm);  // [2][128][OP]
    float2* ss = reinterpret_cast<float2*>(sm + C::OffStat);
    if (mine > 0 && good) {
      float* w = os + (size_t)(grp * kApTcRows + row) * C::OP;
      const uint32_t to = tmem + lanes + C::O0 + grp * HD;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(to + 32 * c, o);
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          *reinterpret_cast<uint4*>(w + 32 * c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      }
      ss[grp * kApTcRows + row] = make_float2(ref, l);
    }
    pt_groups_sync();
    constexpr int LPR = HD / 4;  // threads per row, four values each
    const int S = a.S_p + a.S_o, parts = nb > 1 ? 2 : 1;
    for (int i = tid; i < n * LPR && good; i += 256) {
      const int r = i / LPR, d = (i % LPR) * 4;
      const float mx = parts > 1 ? fmaxf(ss[r].x, ss[kApTcRows + r].x) : ss[r].x;
      float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
      for (int p = 0; p < parts; ++p) {
        const float2 st = ss[p * kApTcRows + r];
        const float f = st.x == -INFINITY ? 0.f : ap_exp2(st.x - mx);
        const float4 ov = *reinterpret_cast<const float4*>(os + (size_t)(p * kApTcRows + r) * C::OP + d);
        sum = fmaf(f, st.y, sum);
        v[0] = fmaf(f, ov.x, v[0]);
        v[1] = fmaf(f, ov.y, v[1]);
        v[2] = fmaf(f, ov.z, v[2]);
        v[3] = fmaf(f, ov.w, v[3]);
      }
      // the other kernels' records hold weights as 2^kApShift e^(s - max): the same scale here
      const float g = exp2f(kApShift - kPtShift);
      const size_t mh = (size_t)(u.x + (i0 + r) / a.G) * a.nh + kv * a.G + (i0 + r) % a.G;
      *reinterpret_cast<float4*>(a.acc + (mh * S + split) * HD + d) = make_float4(v[0] * g, v[1] * g, v[2] * g, v[3] * g);
      if (d == 0) a.stat[mh * S + split] = make_float2(mx, sum * g);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) tmem_dealloc(tmem, 512);
  if (tid == 0 && *failed) atomicOr(a.check, 256u);
}

template <int HD>
int pt_launch(const ApArgs& a, cudaStream_t st) {
  using C = PtCfg<HD>;
  static bool attr_done[64] = {};
  const int dev = device_index();
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    ORCH_CUDA(cudaFuncSetAttribute(attn_prefix_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::Smem));
    attr_done[dev] = true;
  }
  if (!encode_fn()) return fail(ORCH_ERR_CUDA, "attention_prefix: no tensor-map encoder");
  const uint64_t rows = (uint64_t)a.num_prefix * a.nkv * a.prefix_cap;
  CUtensorMap mk, mv;
  if (!encode2d(&mk, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.kp, HD, rows, HD * 2, 64, kApTcKeys, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode2d(&mv, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.vp, HD, rows, HD * 2, 64, kApTcKeys, CU_TENSOR_MAP_SWIZZLE_128B))
    return fail(ORCH_ERR_CUDA, "attention_prefix: tensor map");
  ORCH_CUDA(launch_k_serial(attn_prefix_tc_kernel<HD>, dim3((unsigned)a.blocks_p), dim3(kPtThreads), C::Smem, st,
                            dim3(0, 0, 0), mk, mv, a));
  return check_launch("attention_prefix");
}

}  // namespace

int ap_tc_launch(const ApArgs& a, int hd, cudaStream_t st) { return hd == 64 ? pt_launch<64>(a, st) : pt_launch<128>(a, st); }

}  // namespace orch
