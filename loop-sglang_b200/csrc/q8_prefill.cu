// Causal attention of prompts over the 8-bit paged KV cache (q8.cuh) on the 5th-generation
// tensor cores.
//
// A CTA takes one KV head of one request and 256 of its packed query rows (row = position *
// group + head in the group, so grouped heads share the keys), as two tiles of 128, and walks
// the keys in tiles of 64 up to the last row's causal limit:
//   warps 8-11  widen the codes to f16 tiles in shared memory (K as it lies, V transposed, both
//               K-major with a 128-byte swizzle) and leave each key's scales beside them;
//   warp 12     issues the tcgen05 products S = Q K^T and O += P V^T into TMEM, the score of
//               one tile of rows while the other's softmax runs;
//   warps 0-7   a thread per row: softmax of S from TMEM, P to shared memory as f16.
// Bound: the tensor cores, then the exponentials (16 a clock and SM) and shared memory, in that
// order of the floor.
//
// u = S * k_scale + log2(v_scale) in the log2 domain, w = exp2(u - m) is softmax weight times
// value scale at once, and the row's sum takes w / v_scale: the value scales cost no
// instruction, and the largest contribution is near 1 whatever the scales. Codes are exact in
// f16; q is scaled by one power of two per CTA to f16 (8 bits of 11); w is rounded to f16; all
// sums are fp32. O is rescaled only when a row's maximum grew by more than 2^8.
#include <atomic>

#include "mbarrier.cuh"
#include "q8_prefill.cuh"

namespace lsb {
namespace {

constexpr int kRows = 128;      // query rows per tile, two tiles per CTA
constexpr int kKeys = 64;       // keys per tile
constexpr int kStages = 2;      // K and V tiles in flight
constexpr int kSoftWarps = 8;   // four per tile of rows (TMEM lanes 32w .. belong to warp w % 4)
constexpr int kWidenWarps = 4;
constexpr int kWidenThreads = 32 * kWidenWarps;
constexpr int kThreads = 32 * (kSoftWarps + kWidenWarps + 1);
constexpr float kLow = -1e30f;      // below every score
constexpr float kGrowth = 8.f;      // rescale O when a maximum grew by more (log2)
constexpr float kWeightBits = 6.f;  // weights are scaled by 2^6: at most 2^14 before a rescale

struct KeyScales {  // of one key, or of four with one scale
  float ks, lv, iv, unused;
};

template <int D>
struct Smem {
  static constexpr int kSlabs = (D + 63) / 64;           // 64 dims are a swizzled row
  static constexpr int kQ = kSlabs * kRows * 128;        // bytes of one Q tile
  static constexpr int kK = kSlabs * kKeys * 128;
  static constexpr int kV = D * 128;                     // a row per dim, 64 keys
  static constexpr int kP = kRows * 128;
  static constexpr int q = 0;
  static constexpr int k = q + 2 * kQ;
  static constexpr int v = k + kStages * kK;
  static constexpr int pp = v + kStages * kV;
  static constexpr int scales = pp + 2 * kP;
  static constexpr int slots = scales + kStages * kKeys * 16;
  static constexpr int total = slots + 2 * kKeys * 4;
};

// 128-byte swizzle: 16-byte chunk c of row r of a tile whose rows are 128 bytes.
__device__ __forceinline__ int swizzled(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// K-major operand, 128-byte swizzle: rows of 128 bytes, 8-row atoms 1024 bytes apart.
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
  return ((addr >> 4) & 0x3FFFull) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                     bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)));
}

__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tmem_load16(uint32_t addr, float* f) {
  uint32_t* r = reinterpret_cast<uint32_t*>(f);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const float* f) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(f);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_load_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_store_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// This thread's shared-memory stores, for the tensor cores to read.
__device__ __forceinline__ void fence_operands() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Whether one of a word's four codes is NaN (e4m3 0x7f and 0xff; int8 has none).
template <bool INT8>
__device__ __forceinline__ bool has_nan(uint32_t w) {
  return !INT8 && (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
}

// Tensor-core instruction descriptor: f16 operands, fp32 accumulator, 128 rows, n columns.
__host__ __device__ constexpr uint32_t f16_shape(int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kRows >> 4) << 24);
}

template <int D, bool INT8>
__global__ void __launch_bounds__(kThreads, 1) q8_prefill_kernel(Q8PrefillParams p) {
  using S = Smem<D>;
  constexpr int CHUNKS = D / 16;  // 16-byte chunks of codes per row
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t s_kfull[kStages], s_kempty[kStages], s_vfull[kStages],
      s_vempty[kStages], s_sfull[2], s_pfull[2], s_odone[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_item[2];
  __shared__ uint32_t s_amax;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int kvh = blockIdx.y;

  // ---- which request and which 256 packed rows: blocks of a request, the last one (the most
  // keys) first
  if (warp == 0) {
    int left = blockIdx.x, req = -1, blk = 0;
    for (int base = 0; base < p.num_reqs && req < 0; base += 32) {
      const int r = base + lane;
      int64_t n = 0;
      if (r < p.num_reqs) n = static_cast<int64_t>(p.cu_seqlens_q[r + 1]) - p.cu_seqlens_q[r];
      const int mine = n > 0 ? static_cast<int>((n * p.group + 2 * kRows - 1) / (2 * kRows)) : 0;
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, left < incl);
      if (hit) {
        const int at = __ffs(hit) - 1;
        req = base + at;
        blk = __shfl_sync(0xffffffffu, mine, at) - 1 -
              (left - __shfl_sync(0xffffffffu, incl - mine, at));
      }
      left -= __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      s_item[0] = req;
      s_item[1] = blk;
      s_amax = 0;
      for (int i = 0; i < kStages; ++i) {
        mbar_init(&s_kfull[i], kWidenThreads);
        mbar_init(&s_vfull[i], kWidenThreads);
        mbar_init(&s_kempty[i], 1);
        mbar_init(&s_vempty[i], 1);
      }
      for (int g = 0; g < 2; ++g) {
        mbar_init(&s_sfull[g], 1);
        mbar_init(&s_pfull[g], kRows);
        mbar_init(&s_odone[g], 1);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  __syncthreads();
  const int req = s_item[0];
  if (req < 0) return;
  const int64_t q_begin = p.cu_seqlens_q[req];
  const int64_t n = p.cu_seqlens_q[req + 1] - q_begin;
  int64_t kv_len = p.cache_seqlens[req];
  if (kv_len > p.max_seqlen) {
    if (tid == 0 && p.error_flag) atomicOr(p.error_flag, LSB_DEVERR_SEQLEN);
    kv_len = p.max_seqlen;
  }
  if (kv_len < 0) kv_len = 0;
  const int64_t packed = n * p.group, row0 = static_cast<int64_t>(s_item[1]) * 2 * kRows;
  const int64_t before = kv_len - n;  // the row at position j sees keys 0 .. before + j
  // tiles of keys that each tile of rows walks: up to its last row's limit
  int tiles[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const int64_t from = row0 + g * kRows;
    int64_t last = from + kRows < packed ? from + kRows : packed;
    int64_t see = from < packed ? before + (last - 1) / p.group + 1 : 0;
    if (see > kv_len) see = kv_len;
    tiles[g] = see > 0 ? static_cast<int>((see + kKeys - 1) / kKeys) : 0;
  }
  const int ntiles = max(tiles[0], tiles[1]);

  if (warp == kSoftWarps + kWidenWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&s_tmem)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }

  // ---- the query rows, a thread each: largest finite element of the CTA to [2^7, 2^8)
  const int g = warp >> 2;  // tile of rows (softmax warps)
  const int trow = tid & (kRows - 1);
  const int64_t prow = row0 + g * kRows + trow;  // packed row
  const bool real = warp < kSoftWarps && prow < packed;
  const int64_t pos = real ? prow / p.group : 0;
  const int head = kvh * p.group + (real ? static_cast<int>(prow - pos * p.group) : 0);
  const int64_t qrow = q_begin + pos;
  const bool mine = real && qrow < p.rows;
  {
    uint4 raw[D / 8];
    uint32_t amax = 0;
    if (mine) {
      const bf16* src = p.q + qrow * p.q_stride + static_cast<int64_t>(head) * D;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) raw[c] = *reinterpret_cast<const uint4*>(src + 8 * c);
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t a = (w[e] << 16) & 0x7fffffffu, b = w[e] & 0x7fff0000u;
          if (a < kInfBits) amax = max(amax, a);
          if (b < kInfBits) amax = max(amax, b);
        }
      }
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    if (lane == 0 && amax) atomicMax(&s_amax, amax);
    fence_before();
    __syncthreads();
    fence_after();
    amax = s_amax;
    const int ex = amax == 0 ? 134 : max(static_cast<int>(amax >> 23), 16);
    const float up = __uint_as_float(static_cast<uint32_t>(254 + 7 - ex) << 23);
    if (warp < kSoftWarps) {
      uint8_t* const qt = smem + S::q + g * S::kQ;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        uint4 h = make_uint4(0, 0, 0, 0);
        if (mine) {
          float f[8];
          unpack8(*reinterpret_cast<const bf16x8*>(&raw[c]), f);
          h.x = pack_f16(f[0] * up, f[1] * up);
          h.y = pack_f16(f[2] * up, f[3] * up);
          h.z = pack_f16(f[4] * up, f[5] * up);
          h.w = pack_f16(f[6] * up, f[7] * up);
        }
        *reinterpret_cast<uint4*>(qt + (c >> 3) * (kRows * 128) + swizzled(trow, c & 7)) = h;
      }
      fence_operands();
    }
    __syncthreads();
  }
  const uint32_t tmem = s_tmem;
  const uint32_t smem0 = smem_u32(smem);
  const uint32_t score_at = tmem, out_at = tmem + 2 * kKeys;  // S: 64 columns a tile; O: D

  if (warp == kSoftWarps + kWidenWarps) {
    // ---- products, one thread
    if (lane == 0 && ntiles > 0) {
      auto scores = [&](int gg, int i) {
        if (!mbar_wait(&s_kfull[i % kStages], (i / kStages) & 1, p.error_flag)) return false;
        fence_after();
        const uint32_t a = smem0 + S::q + gg * S::kQ, b = smem0 + S::k + (i % kStages) * S::kK;
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
          umma(score_at + gg * kKeys, operand(a + (s >> 2) * (kRows * 128)) + 2 * (s & 3),
               operand(b + (s >> 2) * (kKeys * 128)) + 2 * (s & 3), f16_shape(kKeys), s > 0);
        umma_commit(&s_sfull[gg]);
        return true;
      };
      // the last tile of rows to use key tile i frees it
      auto last_user = [&](int i) { return i < tiles[1] ? 1 : 0; };
      bool ok = true;
      for (int gg = 0; gg < 2 && ok; ++gg)
        if (tiles[gg] > 0) {
          ok = scores(gg, 0);
          if (last_user(0) == gg) umma_commit(&s_kempty[0]);
        }
      for (int i = 0; i < ntiles && ok; ++i) {
        for (int gg = 0; gg < 2 && ok; ++gg) {
          if (i >= tiles[gg]) continue;
          ok = mbar_wait(&s_pfull[gg], i & 1, p.error_flag);
          if (!ok) break;
          fence_after();
          if (i + 1 < tiles[gg]) {
            ok = scores(gg, i + 1);
            if (!ok) break;
            if (last_user(i + 1) == gg) umma_commit(&s_kempty[(i + 1) % kStages]);
          }
          ok = mbar_wait(&s_vfull[i % kStages], (i / kStages) & 1, p.error_flag);
          if (!ok) break;
          fence_after();
          const uint32_t a = smem0 + S::pp + gg * S::kP, b = smem0 + S::v + (i % kStages) * S::kV;
#pragma unroll
          for (int s = 0; s < kKeys / 16; ++s)
            umma(out_at + gg * D, operand(a) + 2 * s, operand(b) + 2 * s, f16_shape(D),
                 i > 0 || s > 0);
          umma_commit(&s_odone[gg]);
          if (last_user(i) == gg) umma_commit(&s_vempty[i % kStages]);
        }
      }
    }
  } else if (warp >= kSoftWarps) {
    // ---- codes to f16 tiles
    const int wt = tid - 32 * kSoftWarps;
    int32_t* const slots = reinterpret_cast<int32_t*>(smem + S::slots);
    const bool pow2 = (p.page_size & (p.page_size - 1)) == 0;
    const int pshift = __ffs(p.page_size) - 1;
    const int32_t* const pages = p.page_table + req * p.pt_stride;
    const float up_inv = [&] {
      const uint32_t amax = s_amax;
      const int ex = amax == 0 ? 134 : max(static_cast<int>(amax >> 23), 16);
      return __uint_as_float(static_cast<uint32_t>(ex - 7) << 23);
    }();
    const float c_log2 = p.scale_log2 * up_inv;
    // slot of each key of tile i, -1 for none (past the context or outside the pool)
    auto find_slots = [&](int i) {
      if (wt < kKeys) {
        const int64_t key = static_cast<int64_t>(i) * kKeys + wt;
        int32_t slot = -1;
        if (i < ntiles && key < kv_len) {
          const int64_t pg = pow2 ? key >> pshift : key / p.page_size;
          const int64_t s = static_cast<int64_t>(pages[pg]) * p.page_size + (key - pg * p.page_size);
          if (s >= 0 && s < p.num_slots) slot = static_cast<int32_t>(s);
          else if (p.error_flag) atomicOr(p.error_flag, LSB_DEVERR_SLOT);
        }
        slots[(i & 1) * kKeys + wt] = slot;
      }
    };
    // K: 16 codes of key krow(j); V: 8 codes (dims 8 vd ..) of the 8 keys 8 vo ..
    constexpr int KLOADS = kKeys * CHUNKS / kWidenThreads;
    constexpr int VDIMS = D / 8;                       // groups of 8 dims
    constexpr int VLOADS = (8 * VDIMS + kWidenThreads - 1) / kWidenThreads;  // 1 (D = 32 .. 128)
    static_assert(VLOADS == 1 && KLOADS >= 1, "tile shape");
    const int vo = wt & 7, vd = wt >> 3;
    uint4 kraw[2][KLOADS];
    uint2 vraw[2][8];
    float kscale[2], vscale[2];  // of key wt (threads 0 .. 63)
    auto fetch = [&](int i, int b) {
      const int32_t* const sl = slots + (i & 1) * kKeys;
#pragma unroll
      for (int j = 0; j < KLOADS; ++j) {
        const int idx = j * kWidenThreads + wt, key = idx / CHUNKS, c = idx - key * CHUNKS;
        const int32_t s = sl[key];
        kraw[b][j] = make_uint4(0, 0, 0, 0);
        if (s >= 0)
          kraw[b][j] =
              *reinterpret_cast<const uint4*>(p.k + s * p.slot_stride + kvh * D + 16 * c);
      }
      if (vd < VDIMS) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int32_t s = sl[8 * vo + j];
          vraw[b][j] = make_uint2(0, 0);
          if (s >= 0)
            vraw[b][j] =
                *reinterpret_cast<const uint2*>(p.v + s * p.slot_stride + kvh * D + 8 * vd);
        }
      }
      if (wt < kKeys) {
        const int32_t s = sl[wt];
        kscale[b] = vscale[b] = 0.f;
        if (s >= 0) {
          const int64_t at = static_cast<int64_t>(s >> p.block_shift) * p.hkv + kvh;
          kscale[b] = p.ks[at];
          vscale[b] = p.vs[at];
        }
      }
    };
    auto group_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(kWidenThreads) : "memory"); };
    // whether all of these warps' threads are well (they give up a wait together)
    auto group_and = [](bool ok) {
      uint32_t all;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
          "barrier.cta.red.and.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(all)
          : "r"(static_cast<uint32_t>(ok)), "n"(kWidenThreads)
          : "memory");
      return all != 0;
    };
    auto convert = [&](int i, int b) -> bool {
      const int st = i % kStages;
      const uint32_t parity = ((i / kStages) & 1) ^ 1;
      const int32_t* const sl = slots + (i & 1) * kKeys;
      if (!group_and(mbar_wait(&s_kempty[st], parity, p.error_flag))) return false;
      uint8_t* const kt = smem + S::k + st * S::kK;
#pragma unroll
      for (int j = 0; j < KLOADS; ++j) {
        const int idx = j * kWidenThreads + wt, key = idx / CHUNKS, c = idx - key * CHUNKS;
        const uint32_t w[4] = {kraw[b][j].x, kraw[b][j].y, kraw[b][j].z, kraw[b][j].w};
        uint4 h[2];
        q8_decode4<INT8>(w[0], h[0].x, h[0].y);
        q8_decode4<INT8>(w[1], h[0].z, h[0].w);
        q8_decode4<INT8>(w[2], h[1].x, h[1].y);
        q8_decode4<INT8>(w[3], h[1].z, h[1].w);
        uint8_t* const slab = kt + (c >> 2) * (kKeys * 128);
        const int cc = 2 * (c & 3), odd = (c >> 2) & 1;  // the second slab's halves swapped in
        // time: the stores of 8 lanes then fall in different banks
        *reinterpret_cast<uint4*>(slab + swizzled(key, cc + odd)) = odd ? h[1] : h[0];
        *reinterpret_cast<uint4*>(slab + swizzled(key, cc + 1 - odd)) = odd ? h[0] : h[1];
      }
      fence_operands();
      mbar_arrive(&s_kfull[st]);
      if (!group_and(mbar_wait(&s_vempty[st], parity, p.error_flag))) return false;
      // Keys that some row of the CTA must not see although others do: a NaN code would reach
      // it through 0 * NaN, so it becomes 0 and the key's scale NaN (which only rows that see
      // the key take in)
      const bool diagonal = (i + 1) * static_cast<int64_t>(kKeys) > before + row0 / p.group + 1;
      bool bad[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) bad[j] = false;
      if (vd < VDIMS) {
        if (!INT8 && diagonal) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            bad[j] = has_nan<INT8>(vraw[b][j].x) || has_nan<INT8>(vraw[b][j].y);
            if (bad[j]) vraw[b][j] = make_uint2(0, 0);
          }
        }
        uint8_t* const vt = smem + S::v + st * S::kV;
#pragma unroll
        for (int w = 0; w < 2; ++w) {  // dims 8 vd + 4 w ..
          uint32_t pairs[4][4];        // [dim][key pair]
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a = w ? vraw[b][2 * j].y : vraw[b][2 * j].x;
            const uint32_t c = w ? vraw[b][2 * j + 1].y : vraw[b][2 * j + 1].x;
            q8_decode4<INT8>(__byte_perm(a, c, 0x5140), pairs[0][j], pairs[1][j]);
            q8_decode4<INT8>(__byte_perm(a, c, 0x7362), pairs[2][j], pairs[3][j]);
          }
#pragma unroll
          for (int d = 0; d < 4; ++d)
            *reinterpret_cast<uint4*>(vt + swizzled(8 * vd + 4 * w + d, vo)) =
                make_uint4(pairs[d][0], pairs[d][1], pairs[d][2], pairs[d][3]);
        }
      }
      KeyScales* const sc = reinterpret_cast<KeyScales*>(smem + S::scales) + st * kKeys;
      if (wt < kKeys) {
        const float vs = vscale[b];
        KeyScales x;
        x.unused = 0.f;
        const float held = fmaxf(vs, 7.888609e-31f);  // 2^-100: less counts as that
        x.ks = kscale[b] * c_log2;
        x.lv = vs != vs ? vs : log2_fast(held);
        x.iv = 1.f / held;
        if (sl[wt] < 0) {
          x.ks = 0.f;
          x.lv = -INFINITY;
          x.iv = 0.f;
        }
        sc[wt] = x;
      }
      if (!INT8 && diagonal) {
        group_sync();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (bad[j]) sc[8 * vo + j].lv = __uint_as_float(kNanBits);
      }
      fence_operands();
      mbar_arrive(&s_vfull[st]);
      return true;
    };
    if (ntiles > 0) {
      find_slots(0);
      group_sync();
      fetch(0, 0);
      find_slots(1);
      group_sync();
      for (int i = 0; i < ntiles; i += 2) {
        if (i + 1 < ntiles) fetch(i + 1, 1);
        if (!convert(i, 0)) break;
        group_sync();
        find_slots(i + 2);
        group_sync();
        if (i + 1 >= ntiles) break;
        if (i + 2 < ntiles) fetch(i + 2, 0);
        if (!convert(i + 1, 1)) break;
        group_sync();
        find_slots(i + 3);
        group_sync();
      }
    }
  } else {
    // ---- softmax: a thread per row
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = score_at + g * kKeys + lanes, o_at = out_at + g * D + lanes;
    uint8_t* const pt = smem + S::pp + g * S::kP;
    const int64_t limit = mine ? before + pos : -1;  // last key this row sees
    const bool four = p.block_shift >= 2;            // four neighbouring keys have one scale
    float m = kLow, sum = 0.f;
    bool ok = true;
    for (int i = 0; i < tiles[g]; ++i) {
      const int st = i % kStages;
      ok = __all_sync(0xffffffffu, mbar_wait(&s_sfull[g], i & 1, p.error_flag) &&
                                       mbar_wait(&s_vfull[st], (i / kStages) & 1, p.error_flag));
      if (!ok) break;
      fence_after();
      float x[kKeys];
#pragma unroll
      for (int c = 0; c < kKeys; c += 16) tmem_load16(s_at + c, x + c);
      tmem_load_wait();
      const KeyScales* const sc = reinterpret_cast<const KeyScales*>(smem + S::scales) + st * kKeys;
      float top = m;
      if (four) {
#pragma unroll
        for (int k = 0; k < kKeys; k += 4) {
          const KeyScales f = sc[k];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[k + e] = fmaf(x[k + e], f.ks, f.lv);
        }
      } else {
#pragma unroll
        for (int k = 0; k < kKeys; ++k) {
          const KeyScales f = sc[k];
          x[k] = fmaf(x[k], f.ks, f.lv);
        }
      }
      const int64_t sees = limit - static_cast<int64_t>(i) * kKeys;  // last visible key in the tile
      if (sees < kKeys - 1) {
#pragma unroll
        for (int k = 0; k < kKeys; ++k)
          if (k > sees) x[k] = -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < kKeys; ++k) top = fmaxf(top, x[k]);
      // P's buffer and O are free once the product before is done
      if (i > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&s_odone[g], (i - 1) & 1, p.error_flag));
        if (!ok) break;
        fence_after();
      }
      const bool grows = top > m + kGrowth;
      if (__any_sync(0xffffffffu, grows)) {
        const float f = grows ? exp2_fast(m - top) : 1.f;
        if (grows) m = top;
        sum *= f;
        if (i > 0) {
#pragma unroll
          for (int c = 0; c < D; c += 16) {
            float o[16];
            tmem_load16(o_at + c, o);
            tmem_load_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] *= f;
            tmem_store16(o_at + c, o);
          }
          tmem_store_wait();
        }
      }
      const float shift = kWeightBits - m;
#pragma unroll
      for (int k = 0; k < kKeys; ++k) x[k] = exp2_fast(x[k] + shift);
      float part[4] = {0.f, 0.f, 0.f, 0.f};
      if (four) {
#pragma unroll
        for (int k = 0; k < kKeys; k += 4)
          part[(k >> 2) & 3] =
              fmaf(x[k] + x[k + 1] + (x[k + 2] + x[k + 3]), sc[k].iv, part[(k >> 2) & 3]);
      } else {
#pragma unroll
        for (int k = 0; k < kKeys; ++k) part[k & 3] = fmaf(x[k], sc[k].iv, part[k & 3]);
      }
      sum += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
      for (int c = 0; c < kKeys / 8; ++c)
        *reinterpret_cast<uint4*>(pt + swizzled(trow, c)) =
            make_uint4(pack_f16(x[8 * c], x[8 * c + 1]), pack_f16(x[8 * c + 2], x[8 * c + 3]),
                       pack_f16(x[8 * c + 4], x[8 * c + 5]), pack_f16(x[8 * c + 6], x[8 * c + 7]));
      fence_operands();
      fence_before();
      mbar_arrive(&s_pfull[g]);
    }
    // ---- output
    if (ok && tiles[g] > 0)
      ok = __all_sync(0xffffffffu, mbar_wait(&s_odone[g], (tiles[g] - 1) & 1, p.error_flag));
    if (ok) {
      fence_after();
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      bf16* const dst = p.out + qrow * p.out_stride + static_cast<int64_t>(head) * D;
#pragma unroll
      for (int c = 0; c < D; c += 16) {
        float o[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = 0.f;
        if (tiles[g] > 0) {
          tmem_load16(o_at + c, o);
          tmem_load_wait();
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = sum == 0.f ? 0.f : o[e] * inv;
        if (mine) {
          const bf16x8 lo = pack8(o), hi = pack8(o + 8);
          *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(&lo);
          *reinterpret_cast<uint4*>(dst + c + 8) = *reinterpret_cast<const uint4*>(&hi);
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == kSoftWarps + kWidenWarps) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

template <int D, bool INT8>
int launch_dim(const Q8PrefillParams& p, cudaStream_t stream) {
  auto kernel = q8_prefill_kernel<D, INT8>;
  static std::atomic<uint64_t> allowed{0};  // devices whose limit is raised already
  int dev = 0;
  LSB_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    LSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  Smem<D>::total));
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  // blocks of 256 packed rows over all requests: at most one more each than the rows fill
  const int64_t blocks = (p.rows * p.group + 2 * kRows - 1) / (2 * kRows) + p.num_reqs;
  LSB_REQUIRE(blocks < (int64_t(1) << 31) && p.hkv < 65536, "paged_attention_q8: grid too large");
  kernel<<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(p.hkv)), kThreads,
           Smem<D>::total, stream>>>(p);
  return check_launch("lsb_paged_attention_q8 (prompt)");
}

}  // namespace

int launch_q8_prefill(const Q8PrefillParams& p, int head_dim, bool int8, cudaStream_t stream) {
  switch (head_dim) {
    case 32: return int8 ? launch_dim<32, true>(p, stream) : launch_dim<32, false>(p, stream);
    case 64: return int8 ? launch_dim<64, true>(p, stream) : launch_dim<64, false>(p, stream);
    case 96: return int8 ? launch_dim<96, true>(p, stream) : launch_dim<96, false>(p, stream);
    case 128: return int8 ? launch_dim<128, true>(p, stream) : launch_dim<128, false>(p, stream);
  }
  return fail(LSB_ERR_UNSUPPORTED, "lsb_paged_attention_q8: head_dim %d", head_dim);
}

}  // namespace lsb
