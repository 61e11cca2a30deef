// Causal attention of prompts over the 8-bit paged KV cache (q8.cuh) on the 5th-generation
// tensor cores.
//
// A CTA takes one KV head of one request and 256 of its packed query rows (row = position *
// group + head in the group, so grouped heads share the keys), as two tiles of 128, and walks
// the keys in tiles of 64 up to the last row's causal limit:
//   warps 14-15 bring the codes of K and V into shared memory with cp.async;
//   warps 8-11  widen them to f16 tiles (K as it lies, V transposed, both K-major with a
//               128-byte swizzle) and leave each key's scales beside them;
//   warps 12-13 issue the tcgen05 products, a warp per tile of rows: S = Q K^T two key tiles
//               ahead into TMEM, and O += P V^T with P from TMEM, where it replaces its own S;
//   warps 0-7   a thread per row: softmax of S, P back to TMEM as f16.
// Bound per key tile and CTA: 1024 cycles of products and as many of exponentials (16 a clock
// and SM); shared memory feeds the first product with 96 KB (768 cycles for its 512).
//
// u = S * k_scale + log2(v_scale) in the log2 domain, w = exp2(u - m) is softmax weight times
// value scale at once, and the row's sum takes w / v_scale: the value scales cost no
// instruction, and the largest contribution is near 1 whatever the scales. Codes are exact in
// f16; q is scaled by one power of two per tile of rows to f16 (8 bits of 11); w is rounded to
// f16; all sums are fp32. O is rescaled only when a row's maximum grew by more than 2^8.
#include <atomic>

#include "mbarrier.cuh"
#include "q8_prefill.cuh"

namespace lsb {
namespace {

constexpr int kRows = 128;      // query rows per tile, two tiles per CTA
constexpr int kKeys = 64;       // keys per tile
constexpr int kStages = 3;      // K and V tiles in flight
constexpr int kRawStages = 3;   // tiles of codes on their way or being widened
constexpr int kSoftWarps = 8;   // four per tile of rows (TMEM lanes 32w .. belong to warp w % 4)
constexpr int kWidenWarps = 4;
constexpr int kWidenThreads = 32 * kWidenWarps;
constexpr int kThreads = 32 * (kSoftWarps + kWidenWarps + 4);  // whole warpgroups
// registers per thread of the three kinds of warpgroups: (2 * 168 + 96 + 64) * 128 <= 64 K
constexpr int kSoftRegs = 168, kWidenRegs = 96, kIssueRegs = 64;
constexpr float kLow = -1e30f;      // below every score
constexpr float kGrowth = 8.f;      // rescale O when a maximum grew by more (log2)
constexpr float kWeightBits = 6.f;  // weights are scaled by 2^6: at most 2^14 before a rescale

// A key's scales (or those of four keys with one): the factor of its scores, log2 and inverse
// of its value scale.
struct alignas(16) KeyScales {
  float ks, lv, iv, unused;
};

template <int D>
struct Smem {
  static constexpr int kSlabs = (D + 63) / 64;           // 64 dims are a swizzled row
  static constexpr int kQ = kSlabs * kRows * 128;        // bytes of one Q tile
  static constexpr int kK = kSlabs * kKeys * 128;
  static constexpr int kV = D * 128;                     // a row per dim, 64 keys
  static constexpr int q = 0;
  static constexpr int k = q + 2 * kQ;
  static constexpr int v = k + kStages * kK;
  static constexpr int kRawK = kKeys * D;                // codes of a tile as they are
  static constexpr int kRawV = kKeys * q8_row_bytes<D>();
  static constexpr int raw_k = v + kStages * kV;
  static constexpr int raw_v = raw_k + kRawStages * kRawK;
  static constexpr int scales = raw_v + kRawStages * kRawV;
  static constexpr int raw_scales = scales + kStages * kKeys * 16;  // K's, then V's
  static constexpr int valid = raw_scales + kRawStages * kKeys * 8;
  static constexpr int total = valid + kRawStages * 8;
};

// Codes of K as they are copied: by slabs of 64 dims (chunks 0-3, 4-7), a slab's rows together.
template <int D>
__device__ __forceinline__ int raw_k_offset(int r, int c) {
  constexpr int kSecond = D > 64 ? D - 64 : 0;  // bytes of a row in the second slab
  return c < 4 ? r * (D < 64 ? D : 64) + 16 * c : kKeys * 64 + r * kSecond + 16 * (c - 4);
}

// 128-byte swizzle: 16-byte chunk c of row r of a tile whose rows are 128 bytes.
__device__ __forceinline__ int swizzled(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// K-major operand, 128-byte swizzle: rows of 128 bytes, 8-row atoms 1024 bytes apart. The low
// word of its descriptor (16 elements further along K: + 2); the high word is kOperandHigh.
__device__ __forceinline__ uint32_t operand(uint32_t addr) {
  return ((addr >> 4) & 0x3FFFu) | (1u << 16);
}
constexpr uint32_t kOperandHigh = 64u | (1u << 14) | (2u << 29);

__device__ __forceinline__ void umma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                     bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "n"(kOperandHigh));
}
// The same with the left operand in TMEM (a lane per row, two f16 per column).
__device__ __forceinline__ void umma_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                          bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "n"(kOperandHigh));
}
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(yes));
  return yes != 0;
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
// (nothing is read where it is not valid: the bytes are zeroed)
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 4 : 0)
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

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The bytes of a word that are NaN codes (e4m3 0x7f and 0xff; int8 has none), as 0xff.
template <bool INT8>
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  if (INT8) return 0;
  return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
}

// 32 rows x 16 bytes, transposed: lane (g, t) gets column g (r[0]) and g + 8 (r[1]) of rows
// 4t .. 4t + 3, and the same of rows 16 + 4t .. (r[2], r[3]).
__device__ __forceinline__ void load_columns(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
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
  __shared__ __align__(8) uint64_t s_rawfull[2][kRawStages], s_rawempty[2][kRawStages];
  __shared__ __align__(8) uint64_t s_qfull, s_kfull[kStages], s_kempty[kStages],
      s_vfull[kStages], s_vempty[kStages], s_sfull[2][2], s_pfull[2][2], s_odone[2][2];
  __shared__ uint32_t s_tmem, s_amax[2];
  __shared__ int s_item[5];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // The CTAs with the most keys start first, so that the last ones to end are short (the heads of
  // one block of rows next to each other: they read the same slots).
  const int kvh = blockIdx.x % p.hkv, rank = blockIdx.x / p.hkv;

  // ---- the block of 256 packed rows that is rank'th by its tiles of keys, requests in order
  // among equals. A request's blocks see ever more keys, so how many of them have t tiles or
  // more is a formula, and t a bisection over its sum (lane l has requests l, l + 32, ..).
  if (warp == 0) {
    struct Req {
      int from, n, len, blocks;
    };
    auto request = [&](int r) {
      Req q{0, 0, 0, 0};
      if (r < p.num_reqs) {
        q.from = p.cu_seqlens_q[r];
        q.n = p.cu_seqlens_q[r + 1] - q.from;
        q.len = p.cache_seqlens[r];
        if (q.n > 0)
          q.blocks = static_cast<int>(
              (static_cast<int64_t>(q.n) * p.group + 2 * kRows - 1) / (2 * kRows));
      }
      return q;
    };
    // blocks of a request with at least t tiles of keys
    auto with_tiles = [&](const Req& q, int t) -> int {
      const int64_t len = min(static_cast<int64_t>(max(q.len, 0)), p.max_seqlen);
      const int64_t behind = static_cast<int64_t>(kKeys) * (t - 1) - (len - q.n);
      if (t == 0 || behind <= 0) return q.blocks;
      // the block's last packed row is at position `behind` at least
      const int64_t rows = behind * p.group + 1;
      if (static_cast<int64_t>(q.n) * p.group < rows) return 0;
      return q.blocks - static_cast<int>((rows + 2 * kRows - 1) / (2 * kRows) - 1);
    };
    const Req first = request(lane);
    auto count = [&](int t) {
      int c = with_tiles(first, t);
      for (int r = lane + 32; r < p.num_reqs; r += 32) c += with_tiles(request(r), t);
      return __reduce_add_sync(0xffffffffu, c);
    };
    int most = first.len;
    for (int r = lane + 32; r < p.num_reqs; r += 32) most = max(most, p.cache_seqlens[r]);
    most = __reduce_max_sync(0xffffffffu, most);
    if (static_cast<int64_t>(most) > p.max_seqlen) most = static_cast<int>(p.max_seqlen);
    int lo = 0, hi = max(most, 0) / kKeys + 2;  // count(lo) > rank >= count(hi)
    int at_hi = 0;
    const bool found = count(0) > rank;
    while (found && hi - lo > 1) {
      const int mid = (lo + hi) >> 1, c = count(mid);
      if (c > rank) {
        lo = mid;
      } else {
        hi = mid;
        at_hi = c;
      }
    }
    int left = rank - at_hi;  // among those with exactly lo tiles
    bool taken = !found;
    for (int base = 0; base < p.num_reqs && !taken; base += 32) {
      const Req q = base ? request(base + lane) : first;
      const int mine = with_tiles(q, lo) - with_tiles(q, lo + 1);
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, left < incl);
      if (hit) {
        taken = true;
        if (lane == __ffs(hit) - 1) {
          s_item[0] = base + lane;
          s_item[1] = q.blocks - with_tiles(q, lo) + left - (incl - mine);
          s_item[2] = q.from;
          s_item[3] = q.n;
          s_item[4] = q.len;
        }
      }
      left -= __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      if (!found) s_item[0] = -1;
      s_amax[0] = s_amax[1] = 0;
    }
  } else if (warp == 1 && lane == 0) {
    mbar_init(&s_qfull, 2 * kRows);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s_kfull[i], kWidenThreads);
      mbar_init(&s_vfull[i], kWidenThreads);
      mbar_init(&s_kempty[i], 2);
      mbar_init(&s_vempty[i], 2);
    }
    for (int g = 0; g < 2; ++g) {
      for (int i = 0; i < kRawStages; ++i) {
        mbar_init(&s_rawfull[g][i], 33);  // the copies of 32 lanes, the mask of keys
        mbar_init(&s_rawempty[g][i], kWidenWarps);
      }
      for (int e = 0; e < 2; ++e) {  // even and odd key tiles: a warp may be one tile ahead
        mbar_init(&s_sfull[g][e], 1);
        mbar_init(&s_pfull[g][e], kRows);
        mbar_init(&s_odone[g][e], 1);
      }
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  const int req = s_item[0];
  if (req < 0) return;
  const int64_t q_begin = s_item[2], n = s_item[3];
  int64_t kv_len = s_item[4];
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
    const int64_t last = from + kRows < packed ? from + kRows : packed;
    int64_t see = from < packed ? before + (last - 1) / p.group + 1 : 0;
    if (see > kv_len) see = kv_len;
    tiles[g] = see > 0 ? static_cast<int>((see + kKeys - 1) / kKeys) : 0;
  }
  const int ntiles = max(tiles[0], tiles[1]);
  const uint32_t smem0 = smem_u32(smem);
  // TMEM, all 512 columns from 0 on: two score tiles for each tile of rows, 64 columns each,
  // then the outputs, D each
  auto score_at = [](int g, int i) { return static_cast<uint32_t>((2 * g + (i & 1)) * kKeys); };
  auto out_at = [](int g) { return static_cast<uint32_t>(4 * kKeys + g * D); };

  if (warp >= kSoftWarps + kWidenWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (warp == kSoftWarps + kWidenWarps) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_u32(&s_tmem)),
                   "r"(512));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (warp < kSoftWarps + kWidenWarps + 2) {
      // ---- products. The whole warp walks the tiles, so that addresses stay uniform; one lane
      // issues.
      fence_before();
      asm volatile("bar.sync 1, %0;" ::"n"(32 * (kSoftWarps + 2)) : "memory");
      fence_after();
      const int g = __shfl_sync(0xffffffffu, warp - (kSoftWarps + kWidenWarps), 0);
      const int mine = __shfl_sync(0xffffffffu, tiles[g], 0);
      const int all = __shfl_sync(0xffffffffu, ntiles, 0);
      const uint32_t qd = operand(smem0 + S::q + g * S::kQ), kd = operand(smem0 + S::k),
                     vd = operand(smem0 + S::v);
      auto here = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.error_flag)) != 0;
      };
      // the ring position of the next K and V tile
      int kst = 0, vst = 0;
      uint32_t kph = 0, vph = 0;
      auto scores = [&](int i) {
        if (!here(&s_kfull[kst], kph)) return false;
        fence_after();
        if (elect_one()) {
          if (i < mine) {
            const uint32_t b = kd + kst * (S::kK >> 4), d = score_at(g, i);
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
              umma(d, qd + (s >> 2) * (kRows * 128 >> 4) + 2 * (s & 3),
                   b + (s >> 2) * (kKeys * 128 >> 4) + 2 * (s & 3), f16_shape(kKeys), s > 0);
            umma_commit(&s_sfull[g][i & 1]);
            umma_commit(&s_kempty[kst]);
          } else {
            mbar_arrive(&s_kempty[kst]);  // not this tile of rows' any more
          }
        }
        __syncwarp();
        if (++kst == kStages) {
          kst = 0;
          kph ^= 1;
        }
        return true;
      };
      bool ok = here(&s_qfull, 0);
      fence_after();
      for (int i = 0; i < 2 && i < all && ok; ++i) ok = scores(i);
      for (int i = 0; i < all && ok; ++i) {
        ok = here(&s_vfull[vst], vph);
        if (ok && i < mine) ok = here(&s_pfull[g][i & 1], (i >> 1) & 1);
        if (!ok) break;
        fence_after();
        if (elect_one()) {
          if (i < mine) {
            const uint32_t b = vd + vst * (S::kV >> 4), a = score_at(g, i);
#pragma unroll
            for (int s = 0; s < kKeys / 16; ++s)
              umma_tmem(out_at(g), a + 8 * s, b + 2 * s, f16_shape(D), i > 0 || s > 0);
            umma_commit(&s_odone[g][i & 1]);
            umma_commit(&s_vempty[vst]);
          } else {
            mbar_arrive(&s_vempty[vst]);
          }
        }
        __syncwarp();
        if (++vst == kStages) {
          vst = 0;
          vph ^= 1;
        }
        if (i + 2 < all) ok = scores(i + 2);
      }
    }
    else {
      // ---- copies: warp 14 of K, warp 15 of V. Lane k has keys k and k + 32 of the tile; their
      // pages are fetched one tile before.
      const bool is_v = warp == kSoftWarps + kWidenWarps + 3;
      const uint8_t* const base = (is_v ? p.v : p.k) + kvh * D;
      const float* const scales = (is_v ? p.vs : p.ks) + kvh;
      uint64_t* const full = s_rawfull[is_v], * const empty = s_rawempty[is_v];
      const uint32_t raw = smem0 + (is_v ? S::raw_v : S::raw_k);
      const uint32_t raw_bytes = is_v ? S::kRawV : S::kRawK;
      const uint32_t rsc = smem0 + S::raw_scales + (is_v ? kKeys * 4 : 0);
      const bool pow2 = (p.page_size & (p.page_size - 1)) == 0;
      const int pshift = __ffs(p.page_size) - 1;
      const int32_t* const pages = p.page_table + req * p.pt_stride;
      const uint32_t stride = static_cast<uint32_t>(p.slot_stride);
      const int len = static_cast<int>(kv_len);
      int page[2] = {0, 0};
      auto fetch_pages = [&](int i) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = i * kKeys + 32 * e + lane;
          if (i < ntiles && key < len) page[e] = pages[pow2 ? key >> pshift : key / p.page_size];
        }
      };
      constexpr bool kEven = 32 % CHUNKS == 0;
      const bool paged = pow2 && p.page_size >= 16 && static_cast<uint64_t>(stride) * 16 < (1u << 31);
      const uint64_t lane_src = static_cast<uint64_t>(lane / CHUNKS) * stride + 16 * (lane % CHUNKS);
      constexpr int kRowK = D < 64 ? D : 64;
      const uint32_t lane_k = raw_k_offset<D>(lane / CHUNKS, lane % CHUNKS);
      uint32_t lane_v[2] = {0, 0};
      if (kEven) {
        lane_v[0] = q8_tile_offset<D>(lane / CHUNKS, lane % CHUNKS);
        lane_v[1] = q8_tile_offset<D>(lane / CHUNKS + 32 / CHUNKS, lane % CHUNKS);
      }
      const uint8_t* row = base;
      fetch_pages(0);
      int rs = 0;
      uint32_t phase = 0;
      for (int i = 0; i < ntiles; ++i) {
        int slot[2];
        uint32_t mask[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = i * kKeys + 32 * e + lane;
          const int off = pow2 ? (key & (p.page_size - 1)) : key % p.page_size;
          const int64_t s = static_cast<int64_t>(page[e]) * p.page_size + off;
          const bool there = key < len, ok = there && s >= 0 && s < p.num_slots;
          if (there && !ok && p.error_flag) atomicOr(p.error_flag, LSB_DEVERR_SLOT);
          slot[e] = ok ? static_cast<int>(s) : -1;
          mask[e] = __ballot_sync(0xffffffffu, ok);
        }
        fetch_pages(i + 1);
        if (!__all_sync(0xffffffffu, mbar_wait(&empty[rs], phase ^ 1, p.error_flag))) break;
        const uint32_t dst = raw + rs * raw_bytes;
        if (kEven && paged && (mask[0] & mask[1]) == 0xffffffffu) {
          // whole pages of at least 16 tokens: rows of one page are a stride apart, so a copy's
          // address is a sum instead of a slot handed round, 1700 -> 700 cycles a tile
#pragma unroll
          for (int j = 0; j < 2 * CHUNKS; ++j) {
            constexpr int kStep = kEven ? 32 / CHUNKS : 1;  // rows per copy of the warp
            const int r = j * kStep, in16 = r & 15;
            if (in16 == 0) {
              const uint32_t first = __shfl_sync(0xffffffffu, slot[r >> 5], r & 31);
              row = base + lane_src + static_cast<uint64_t>(first) * stride;
            }
            copy16(dst + (is_v ? lane_v[j & 1] + (j >> 1) * 1024 : lane_k + j * kStep * kRowK),
                   row + static_cast<uint32_t>(in16) * stride, true);
          }
        } else
#pragma unroll
        for (int j = 0; j < 2 * CHUNKS; ++j) {  // 16-byte chunk j * 32 + lane of the tile
          const int idx = j * 32 + lane, r = idx / CHUNKS, c = idx - r * CHUNKS;
          const int at = __shfl_sync(0xffffffffu, slot[j >= CHUNKS], r & 31);
          const uint8_t* src =
              base + static_cast<uint64_t>(static_cast<uint32_t>(max(at, 0))) * stride + 16 * c;
          copy16(dst + (is_v ? q8_tile_offset<D>(r, c) : raw_k_offset<D>(r, c)), src, at >= 0);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
          copy4(rsc + (rs * 2 * kKeys + 32 * e + lane) * 4,
                scales + static_cast<uint64_t>(static_cast<uint32_t>(max(slot[e], 0)) >>
                                               p.block_shift) * p.hkv,
                slot[e] >= 0);
        copies_arrive(&full[rs]);
        if (lane == 0) {
          if (is_v)
            *reinterpret_cast<uint2*>(smem + S::valid + rs * 8) = make_uint2(mask[0], mask[1]);
          mbar_arrive(&full[rs]);
        }
        if (++rs == kRawStages) {
          rs = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp >= kSoftWarps) {
    // ---- codes to f16 tiles. Nothing here waits for another warp but at the rings.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWidenRegs));
    const int wt = tid - 32 * kSoftWarps, ww = warp - kSoftWarps;
    constexpr int KLOADS = kKeys * CHUNKS / kWidenThreads;  // 16 codes a thread each
    constexpr int VLOADS = 2 * CHUNKS / kWidenWarps;        // 32 keys x 16 dims a warp each
    const int t4 = lane & 3, g8 = lane >> 2;
    int st = 0, rs = 0;
    uint32_t ph = 0, rph = 0;
    for (int i = 0; i < ntiles; ++i) {
      bool ok = mbar_wait(&s_rawfull[0][rs], rph, p.error_flag) &&
                mbar_wait(&s_kempty[st], ph ^ 1, p.error_flag);
      if (!__all_sync(0xffffffffu, ok)) break;
      {
        uint8_t* const kt = smem + S::k + st * S::kK;
        const uint8_t* const src = smem + S::raw_k + rs * S::kRawK + 16 * wt;
        uint4 w[KLOADS];
#pragma unroll
        for (int j = 0; j < KLOADS; ++j)
          w[j] = *reinterpret_cast<const uint4*>(src + j * 16 * kWidenThreads);
        float ks = 0.f;
        if (wt < kKeys)
          ks = *reinterpret_cast<const float*>(smem + S::raw_scales + (rs * 2 * kKeys + wt) * 4);
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_rawempty[0][rs]);
        // thread's 16 codes j: in the first slab four threads a key, so the 16-byte stores of 8
        // threads (two keys, every other chunk) fall in different banks
        constexpr int kFirst = kKeys * (CHUNKS < 4 ? CHUNKS : 4) / kWidenThreads;
        constexpr int kPer0 = CHUNKS < 4 ? CHUNKS : 4, kPer1 = CHUNKS > 4 ? CHUNKS - 4 : 1;
#pragma unroll
        for (int j = 0; j < KLOADS; ++j) {
          const int per = j < kFirst ? kPer0 : kPer1, at = (j < kFirst ? j : j - kFirst) * kWidenThreads + wt;
          const int key = at / per, cc = 2 * (at - key * per);
          uint8_t* const slab = kt + (j < kFirst ? 0 : kKeys * 128);
          uint4 h[2];
          q8_decode4<INT8>(w[j].x, h[0].x, h[0].y);
          q8_decode4<INT8>(w[j].y, h[0].z, h[0].w);
          q8_decode4<INT8>(w[j].z, h[1].x, h[1].y);
          q8_decode4<INT8>(w[j].w, h[1].z, h[1].w);
          *reinterpret_cast<uint4*>(slab + swizzled(key, cc)) = h[0];
          *reinterpret_cast<uint4*>(slab + swizzled(key, cc + 1)) = h[1];
        }
        fence_operands();
        mbar_arrive(&s_kfull[st]);
        ok = mbar_wait(&s_rawfull[1][rs], rph, p.error_flag) &&
             mbar_wait(&s_vempty[st], ph ^ 1, p.error_flag);
        if (!__all_sync(0xffffffffu, ok)) break;
        // Keys that some row of the CTA must not see although others do: a NaN code would reach
        // it through 0 * NaN, so it becomes 0 and the key's scale NaN (which only rows that see
        // the key take in)
        const bool diagonal =
            !INT8 && (i + 1) * static_cast<int64_t>(kKeys) > before + row0 / p.group + 1;
        const uint32_t vsrc = smem0 + S::raw_v + rs * S::kRawV;
        // this warp's units: keys 32 half .., dims 16 (2j + ww / 2) ..
        const int half = ww & 1;
        uint32_t r[VLOADS][4];
#pragma unroll
        for (int j = 0; j < VLOADS; ++j)
          load_columns(r[j], vsrc + q8_tile_offset<D>(32 * half + lane, 2 * j + (ww >> 1)));
        if (diagonal) {
#pragma unroll
          for (int j = 0; j < VLOADS; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) r[j][e] &= ~nan_bytes<INT8>(r[j][e]);
        }
        uint8_t* const vt = smem + S::v + st * S::kV + (ww >> 1) * 16 * 128 + 8 * (t4 & 1);
#pragma unroll
        for (int hi = 0; hi < 2; ++hi) {  // keys 32 half + 16 hi + 4 t4 .., dims g8 and g8 + 8 of 16
          uint8_t* const at = vt + swizzled(g8, 4 * half + 2 * hi + (t4 >> 1));
#pragma unroll
          for (int j = 0; j < VLOADS; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint2 h;
              q8_decode4<INT8>(r[j][2 * hi + e], h.x, h.y);
              *reinterpret_cast<uint2*>(at + (32 * j + 8 * e) * 128) = h;
            }
        }
        if (wt < kKeys) {
          const float vs = *reinterpret_cast<const float*>(smem + S::raw_scales +
                                                           (rs * 2 * kKeys + kKeys + wt) * 4);
          const uint32_t valid =
              *reinterpret_cast<const uint32_t*>(smem + S::valid + rs * 8 + (wt >> 5) * 4);
          const float held = fmaxf(vs, 7.888609e-31f);  // 2^-100: less counts as that
          float lv = vs != vs ? vs : log2_fast(held), iv = 1.f / held;
          if (!((valid >> lane) & 1)) {
            ks = iv = 0.f;
            lv = -INFINITY;
          } else if (diagonal) {
            uint32_t bad = 0;
            for (int c = 0; c < CHUNKS; ++c) {
              const uint4 w = *reinterpret_cast<const uint4*>(smem + S::raw_v + rs * S::kRawV +
                                                              q8_tile_offset<D>(wt, c));
              bad |= nan_bytes<INT8>(w.x) | nan_bytes<INT8>(w.y) | nan_bytes<INT8>(w.z) |
                     nan_bytes<INT8>(w.w);
            }
            if (bad) lv = __uint_as_float(kNanBits);
          }
          ks *= p.scale_log2;
          reinterpret_cast<KeyScales*>(smem + S::scales)[st * kKeys + wt] = {ks, lv, iv, 0.f};
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_rawempty[1][rs]);
        fence_operands();
        mbar_arrive(&s_vfull[st]);
      }
      if (++st == kStages) {
        st = 0;
        ph ^= 1;
      }
      if (++rs == kRawStages) {
        rs = 0;
        rph ^= 1;
      }
    }
  } else {
    // ---- softmax: a thread per row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    const int g = warp >> 2;  // tile of rows
    const int trow = tid & (kRows - 1);
    const int64_t prow = row0 + g * kRows + trow;  // packed row
    const int64_t pos = prow < packed ? prow / p.group : 0;
    const int head = kvh * p.group + (prow < packed ? static_cast<int>(prow - pos * p.group) : 0);
    const int64_t qrow = q_begin + pos;
    const bool mine = prow < packed && qrow < p.rows;
    // the row's query as f16: as it is while the tile's largest finite element is from 2^-2 to
    // 2^15 (bf16's 8 bits then stay exact to 2^-15 of it at least), else scaled to [2^7, 2^8)
    float back = 1.f;
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
      if (lane == 0 && amax) atomicMax(&s_amax[g], amax);
      asm volatile("bar.sync %0, %1;" ::"r"(2 + g), "n"(kRows) : "memory");
      amax = s_amax[g];
      const int ex = max(static_cast<int>(amax >> 23), 16);
      float up = 1.f;
      if (amax != 0 && (ex < 125 || ex > 141)) {
        up = __uint_as_float(static_cast<uint32_t>(254 + 7 - ex) << 23);
        back = __uint_as_float(static_cast<uint32_t>(ex - 7) << 23);
      }
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
      mbar_arrive(&s_qfull);
    }
    asm volatile("bar.sync 1, %0;" ::"n"(32 * (kSoftWarps + 2)) : "memory");
    fence_after();
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t o_at = lanes + out_at(g);
    const int64_t limit = mine ? before + pos : -1;  // last key this row sees
    const bool four = p.block_shift >= 2;            // four neighbouring keys have one scale
    float m = kLow, sum = 0.f;
    bool ok = true;
    for (int i = 0; i < tiles[g]; ++i) {
      const int st = i % kStages;
      ok = __all_sync(0xffffffffu,
                      mbar_wait(&s_vfull[st], (i / kStages) & 1, p.error_flag) &&
                          mbar_wait(&s_sfull[g][i & 1], (i >> 1) & 1, p.error_flag));
      if (!ok) break;
      fence_after();
      const uint32_t s_at = lanes + score_at(g, i);
      float x[kKeys];
#pragma unroll
      for (int c = 0; c < kKeys; c += 16) tmem_load16(s_at + c, x + c);
      tmem_load_wait();
      const KeyScales* const sc = reinterpret_cast<const KeyScales*>(smem + S::scales) + st * kKeys;
      if (back != 1.f) {
#pragma unroll
        for (int k = 0; k < kKeys; ++k) x[k] *= back;
      }
      if (four) {
#pragma unroll
        for (int k = 0; k < kKeys; k += 4) {
          const float2 f = *reinterpret_cast<const float2*>(&sc[k]);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[k + e] = fmaf(x[k + e], f.x, f.y);
        }
      } else {
#pragma unroll
        for (int k = 0; k < kKeys; ++k) {
          const float2 f = *reinterpret_cast<const float2*>(&sc[k]);
          x[k] = fmaf(x[k], f.x, f.y);
        }
      }
      const int64_t sees = limit - static_cast<int64_t>(i) * kKeys;  // last visible key in the tile
      if (sees < kKeys - 1) {
#pragma unroll
        for (int k = 0; k < kKeys; ++k)
          if (k > sees) x[k] = -INFINITY;
      }
      float tops[4] = {m, m, m, m};
#pragma unroll
      for (int k = 0; k < kKeys; k += 2) tops[(k >> 1) & 3] = max3(tops[(k >> 1) & 3], x[k], x[k + 1]);
      const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
      const bool grows = top > m + kGrowth;
      if (__any_sync(0xffffffffu, grows)) {
        const float f = grows ? exp2_fast(m - top) : 1.f;
        if (grows) m = top;
        sum *= f;
        if (i > 0) {  // O, once the product before is in
          ok = __all_sync(0xffffffffu, mbar_wait(&s_odone[g][(i - 1) & 1], ((i - 1) >> 1) & 1,
                                                 p.error_flag));
          if (!ok) break;
          fence_after();
#pragma unroll
          for (int c = 0; c < D; c += 16) {
            float o[16];
            tmem_load16(o_at + c, o);
            tmem_load_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] *= f;
            tmem_store16(o_at + c, o);
          }
        }
      }
      const float shift = kWeightBits - m;
      float part[2] = {0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kKeys; c += 32) {  // 32 keys: 16 columns of P
        float w[16];
#pragma unroll
        for (int k = c; k < c + 32; k += 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[k + e] = exp2_fast(x[k + e] + shift);
          if (four) {
            part[(k >> 2) & 1] =
                fmaf((x[k] + x[k + 1]) + (x[k + 2] + x[k + 3]), sc[k].iv, part[(k >> 2) & 1]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) part[e & 1] = fmaf(x[k + e], sc[k + e].iv, part[e & 1]);
          }
          w[(k - c) / 2] = __uint_as_float(pack_f16(x[k], x[k + 1]));
          w[(k - c) / 2 + 1] = __uint_as_float(pack_f16(x[k + 2], x[k + 3]));
        }
        tmem_store16(s_at + c / 2, w);
      }
      sum += part[0] + part[1];
      tmem_store_wait();
      fence_before();
      mbar_arrive(&s_pfull[g][i & 1]);
    }
    // ---- output
    if (ok && tiles[g] > 0) {
      const int last = tiles[g] - 1;
      ok = __all_sync(0xffffffffu,
                      mbar_wait(&s_odone[g][last & 1], (last >> 1) & 1, p.error_flag));
    }
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
    fence_before();
  }
  __syncthreads();
  if (warp == kSoftWarps + kWidenWarps) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s_tmem), "r"(512));
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
  LSB_REQUIRE(blocks * p.hkv < (int64_t(1) << 31), "paged_attention_q8: grid too large");
  kernel<<<static_cast<unsigned>(blocks * p.hkv), kThreads, Smem<D>::total, stream>>>(p);
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
