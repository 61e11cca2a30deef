// Causal attention of prompts over the 8-bit paged KV cache (q8.cuh) on the 5th-generation
// tensor cores.
//
// An item is one KV head of one request and 256 of its packed query rows (row = position * group +
// head in the group, so grouped heads share the keys), as two tiles of 128; its keys are walked in
// tiles of 64 up to the last row's causal limit. A CTA per SM takes item after item, each warp at
// its own pace, so that one item's first tiles are under way while the one before ends:
//   warps 18-19 copy the codes of K and V, the scales and the queries into shared memory by tensor
//               copies (boxes of up to 64 slots of a page, single slots where pages are smaller)
//               and find the next item;
//   warps 8-11  widen K to bf16, 12-15 V to f16 and transposed, both K-major with a 128-byte
//               swizzle;
//   warps 16-17 issue the tcgen05 products, a warp per tile of rows: S = Q K^T two key tiles
//               ahead into TMEM, and O += P V^T with P from TMEM, where it replaces its own S;
//   warps 0-7   a thread per row: softmax of S, P back to TMEM as f16.
//
// u = S * k_scale + log2(v_scale) in the log2 domain, w = exp2(u - m) is softmax weight times
// value scale at once, and the row's sum takes w / v_scale: the value scales cost no
// instruction, and the largest contribution is near 1 whatever the scales. Codes of both types are
// exact in bf16 and f16; q is taken as it is; w is rounded to f16 (2^-11); all sums are fp32. O is
// rescaled only when a row's maximum grew by more than 2^8.
//
// Bound: the softmax warps' instructions and latencies. Per key tile and CTA the products need
// 1024 cycles of the tensor core (the first is fed 96 KB of shared memory, 768 cycles, for its
// 512), the exponentials 1024 of their unit (16 a clock and SM); measured 2560, of which a softmax
// warp takes 620 for reading S and the maximum, 220 for the check of growth, 1350 for exponentials
// and P (two warps share the unit), 370 for waits and votes. Code size matters: five roles share
// the SM's instruction cache, and with unrolled paths of 115 KB half of all stalls were fetches;
// short loops, short waits, one copy of the search and divisions by multiplication (70 KB) took
// 8256 tokens of prompts (16 heads of 128) from 152 to 97 us, 512-token chunks over 2048 to 8704
// keys (32 on 8 heads of 128, int8) from 307 to 272 us; now 92 us (420 TFLOP/s) and 269 us (638).
// A CTA per item instead took 129 us for the prompts: 15 thousand cycles to begin an item, 5
// thousand to end it. An item's keys are not split over CTAs: calls of few items leave SMs idle
// (one request of 16000 keys, 16 heads of 128: 262 us for 32 rows, 328 us for 256).
#include <cuda.h>
#include <cudaTypedefs.h>

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
constexpr int kWidenWarps = 4;  // for K, and as many for V
constexpr int kWidenThreads = 32 * kWidenWarps;
constexpr int kIssueWarp = kSoftWarps + 2 * kWidenWarps;  // two, then two that copy
constexpr int kCopyWarp = kIssueWarp + 2;
constexpr int kThreads = 32 * (kIssueWarp + 4);  // whole warpgroups
// Registers per thread of the warpgroups: softmax (two), K, V, issue and copies. They share the
// 5 * 96 per thread of the launch.
constexpr int kSoftRegs = 128, kWidenKRegs = 64, kWidenVRegs = 72, kIssueRegs = 88;
constexpr int kBoxMin = 4;  // slots that a box of codes has at least
constexpr uint32_t kWaitCycles = 3800000000u;  // about 2 s
constexpr float kLow = -3.402823466e38f;  // no finite score is below
constexpr float kGrowth = 8.f;      // rescale O when a maximum grew by more (log2)
constexpr float kFar = 1048576.f;   // maxima whose rounding counts in a weight
constexpr float kWeightBits = 6.f;  // weights are scaled by 2^6: at most 2^14 before a rescale

// A key's scales: the factor of its scores, log2 and inverse of its value scale; and lv for rows
// that see the whole tile and read one key's scales for a group of keys: NaN if a key nearby has a
// NaN code that its own lv stands for.
struct alignas(16) KeyScales {
  float ks, lv, iv, whole;
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
  static constexpr int kRaw = kKeys * D;                 // codes of a tile as they are
  static constexpr int raw_k = v + kStages * kV;
  static constexpr int raw_v = raw_k + kRawStages * kRaw;
  static constexpr int scales = raw_v + kRawStages * kRaw;
  static constexpr int raw_scales = scales + kStages * kKeys * 16;  // K's, then V's
  static constexpr int valid = raw_scales + kRawStages * kKeys * 8;
  static constexpr int total = valid + kRawStages * 16;
};

// Where the copies put 16-byte chunk c of row r of a tile of codes: rows of D bytes, swizzled by
// as much (96 bytes: not at all).
template <int D>
__device__ __forceinline__ int raw_offset(int r, int c) {
  return D == 96 ? r * 96 + 16 * c : q8_tile_offset<D>(r, c);
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
__device__ __forceinline__ void tmem_store8(uint32_t addr, const float* f) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(f);
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
               "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t addr, float* f) {
  uint32_t* r = reinterpret_cast<uint32_t*>(f);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_load_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
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

__device__ __forceinline__ float inverse_fast(float x) {
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// Is a byte of the four words such a code?
template <bool INT8>
__device__ __forceinline__ bool any_nan(const uint4& u) {
  if (INT8) return false;
  auto sum = [](uint32_t w) { return (w & 0x7f7f7f7fu) + 0x01010101u; };
  return ((sum(u.x) | sum(u.y) | sum(u.z) | sum(u.w)) & 0x80808080u) != 0;
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

// Tensor-core instruction descriptors: f16 or bf16 operands, fp32 accumulator, 128 rows, n
// columns.
__host__ __device__ constexpr uint32_t f16_shape(int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kRows >> 4) << 24);
}
__host__ __device__ constexpr uint32_t bf16_shape(int n) {
  return f16_shape(n) | (1u << 7) | (1u << 10);
}

// Two fp32 at once.
__device__ __forceinline__ void fma2(float& a, float& b, float f, float c) {  // a, b = a, b * f + c
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %2};\n\t"
      "mov.b64 z, {%3, %3};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(f), "f"(c));
}
__device__ __forceinline__ void add2(float& a, float& b, float c, float d) {  // a, b += c, d
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}

// Codes 0, 1 (`lo`) and 2, 3 (`hi`) of a word as bf16 pairs, exactly. int8: the low 7 bits under
// the exponent of 128, less 128 or (bit 7 set) 256. e4m3: sign, exponent and mantissa moved to
// their places are the value times 2^-120 (subnormal codes as subnormal numbers); NaN codes
// would come out as +-480, see nan_bytes.
template <bool INT8>
__device__ __forceinline__ void decode4_bf16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  auto pair = [](uint32_t x) -> uint32_t {
    __nv_bfloat162 r;
    if (INT8) {
      const uint32_t a = x & 0xff7fff7fu, b = x & 0x43804380u;
      r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                  *reinterpret_cast<const __nv_bfloat162*>(&b));
    } else {
      const uint32_t a = (x & 0x80008000u) | ((x >> 4) & 0x07f007f0u);
      const uint32_t up = 0x7b807b80u;  // 2^120
      r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                  *reinterpret_cast<const __nv_bfloat162*>(&up));
    }
    return *reinterpret_cast<const uint32_t*>(&r);
  };
  lo = pair(INT8 ? __byte_perm(w, 0x43434343u, 0x4140) : __byte_perm(w, 0, 0x1404));
  hi = pair(INT8 ? __byte_perm(w, 0x43434343u, 0x4342) : __byte_perm(w, 0, 0x3424));
}

// Four rows of a tensor, from element x on, next to each other in shared memory (a row that the
// tensor does not have is zeros).
__device__ __forceinline__ void gather4(uint32_t dst, const CUtensorMap* map, int x, int r0, int r1,
                                        int r2, int r3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(map), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(smem_u32(bar))
      : "memory");
}

// A box of a tensor.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// Asks for the index of a CTA that has not been started yet, to do its work here: 16 bytes at
// `answer`, counted by `bar`.
__device__ __forceinline__ void ask_next(void* answer, uint64_t* bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], "
      "[%1];" ::"r"(smem_u32(answer)),
      "r"(smem_u32(bar))
      : "memory");
}
// The answer: that CTA's blockIdx.x, or -1 when none is left.
__device__ __forceinline__ int next_of(const void* answer) {
  int x;
  asm volatile(
      "{\n\t.reg .b128 a;\n\t.reg .pred p;\n\t.reg .b32 y, z, w;\n\t"
      "ld.shared.b128 a, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\t"
      "mov.b32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, w}, a;\n\t}"
      : "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  return x;
}

// 256 packed query rows of a KV head, as the search leaves them: request, KV head, block of rows,
// the request's first row, rows, rows that the call has, and keys.
struct Item {
  int req, kvh, block, from, n, live, len, unused;
};
// What the roles need of it.
struct Work {
  int64_t before;      // the row at position j sees keys 0 .. before + j
  uint32_t row0, packed;
  int len, tiles[2], ntiles;  // tiles of keys for each tile of rows, and the larger
};

// The codes of K and V (rows are slots): to gather rows from, and in boxes of `box` slots where
// whole boxes lie in a page (0: nowhere). q, of a tile's positions and a group's heads at a time,
// where a tile's rows are whole positions.
struct Maps {
  CUtensorMap k, v, k_box, v_box, q;
  int box;
  bool q_tiled;
  uint32_t num_pages;
  // n / d = n * mul >> shift for n below 2^31
  struct Divisor {
    uint32_t mul;
    int shift;
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
      return static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> shift);
    }
  } page, group;
};

// With 2^s >= d: mul = ceil(2^(31 + s) / d) is below 2^32 and exceeds the quotient by less than
// 1, so n * mul exceeds n / d * 2^(31 + s) by less than 2^31 <= 2^(31 + s) / d: never as far as
// the next whole number.
Maps::Divisor divisor(uint32_t d) {
  int s = 0;
  while ((uint64_t(1) << s) < d) ++s;
  return {static_cast<uint32_t>(((uint64_t(1) << (31 + s)) + d - 1) / d), 31 + s};
}

// One row's softmax over the scores of a tile of keys, in short loops. S * ks + lv with ks >= 0
// grows with S, so the largest of G keys with one scale is that of the largest S: one product
// instead of G before the maximum.
template <int G>
__device__ __forceinline__ float largest_score(uint32_t s_at, const KeyScales* sc, float top) {
#pragma unroll 1
  for (int c = 0; c < kKeys; c += 32) {
    float x[32];
    tmem_load32(s_at + c, x);
    tmem_load_wait();
#pragma unroll
    for (int k = 0; k < 32; k += G) {
      const float2 f = *reinterpret_cast<const float2*>(&sc[c + k]);
      float a = fmaxf(x[k], x[k + 1]), b = fmaxf(x[k + 2], x[k + 3]);
#pragma unroll
      for (int e = 4; e < G; e += 4) {
        a = max3(a, x[k + e], x[k + e + 1]);
        b = max3(b, x[k + e + 2], x[k + e + 3]);
      }
      top = fmaxf(top, fmaf(fmaxf(a, b), f.x, f.y));
    }
  }
  return top;
}
// The weights exp2(S * ks + lv + kWeightBits - m) of the tile to TMEM, in the place of its scores;
// returns their sum, each less its value scale.
template <int G>
__device__ __forceinline__ float store_weights(uint32_t s_at, const KeyScales* sc, float m) {
  const float shift = kWeightBits - m;
  float sum = 0.f;
#pragma unroll 1
  for (int c = 0; c < kKeys; c += 32) {
    float x[32], w[16];
    tmem_load32(s_at + c, x);
    tmem_load_wait();
#pragma unroll
    for (int k = 0; k < 32; k += G) {
      const float4 f = *reinterpret_cast<const float4*>(&sc[c + k]);
      const float add = f.w + shift;
      float t[2] = {0.f, 0.f};
#pragma unroll
      for (int e = k; e < k + G; e += 2) {
        fma2(x[e], x[e + 1], f.x, add);
        x[e] = exp2_fast(x[e]);
        x[e + 1] = exp2_fast(x[e + 1]);
        add2(t[0], t[1], x[e], x[e + 1]);
        w[e / 2] = __uint_as_float(pack_f16(x[e], x[e + 1]));
      }
      sum = fmaf(t[0] + t[1], f.z, sum);
    }
    tmem_store16(s_at + c / 2, w);
  }
  return sum;
}
// The same two where keys have scales of their own, or lie past the last one that the row sees.
// Or where the maximum is so large that rounding counts: here scores are rounded as it was before
// they are taken from it, and `shift` is rounded down, so that no weight exceeds 2^14.
__device__ __forceinline__ float largest_score(uint32_t s_at, const KeyScales* sc, float top,
                                               int sees) {
#pragma unroll 1
  for (int c = 0; c < kKeys; c += 16) {
    float x[16];
    tmem_load16(s_at + c, x);
    tmem_load_wait();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float2 f = *reinterpret_cast<const float2*>(&sc[c + k]);
      x[k] = c + k > sees ? -INFINITY : fmaf(x[k], f.x, f.y);
    }
#pragma unroll
    for (int k = 0; k < 16; k += 2) top = max3(top, x[k], x[k + 1]);
  }
  return top;
}
__device__ __forceinline__ float store_weights(uint32_t s_at, const KeyScales* sc, float m,
                                               int sees) {
  const float shift = __fsub_rd(kWeightBits, m);
  float sum = 0.f;
#pragma unroll 1
  for (int c = 0; c < kKeys; c += 16) {
    float x[16];
    float w[8];
    tmem_load16(s_at + c, x);
    tmem_load_wait();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float4 f = *reinterpret_cast<const float4*>(&sc[c + k]);
      x[k] = exp2_fast(c + k > sees ? -INFINITY : fmaf(x[k], f.x, f.y) + shift);
      sum = fmaf(x[k], f.z, sum);
    }
#pragma unroll
    for (int k = 0; k < 16; k += 2) w[k / 2] = __uint_as_float(pack_f16(x[k], x[k + 1]));
    tmem_store8(s_at + c / 2, w);
  }
  return sum;
}

template <int D, bool INT8>
__global__ void __launch_bounds__(kThreads, 1)
    q8_prefill_kernel(const __grid_constant__ Q8PrefillParams p,
                      const __grid_constant__ Maps maps) {
  using S = Smem<D>;
  constexpr int CHUNKS = D / 16;  // 16-byte chunks of codes per row
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t s_rawfull[2][kRawStages], s_rawempty[2][kRawStages];
  __shared__ __align__(8) uint64_t s_qfull[2], s_qempty[2], s_kfull[kStages], s_kempty[kStages],
      s_vfull[kStages], s_vempty[kStages], s_sfull[2][2], s_pfull[2][2], s_odone[2][2],
      s_itemfull[2], s_itemempty[2], s_answered, s_drained[2];
  __shared__ __align__(16) Item s_item[2];
  __shared__ __align__(16) uint4 s_answer;
  __shared__ uint32_t s_tmem;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (warp == 0 && lane == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s_kfull[i], kWidenThreads);
      mbar_init(&s_vfull[i], kWidenThreads);
      mbar_init(&s_kempty[i], 2);
      mbar_init(&s_vempty[i], 2);
    }
    mbar_init(&s_answered, 1);
    for (int g = 0; g < 2; ++g) {
      for (int i = 0; i < kRawStages; ++i) {
        mbar_init(&s_rawfull[g][i], g ? 33 : 1);  // V: the scales that 32 lanes copy, too
        mbar_init(&s_rawempty[g][i], kWidenWarps);
      }
      for (int e = 0; e < 2; ++e) {  // even and odd key tiles: a warp may be one tile ahead
        mbar_init(&s_sfull[g][e], 1);
        mbar_init(&s_pfull[g][e], kRows);
        mbar_init(&s_odone[g][e], 1);
      }
      mbar_init(&s_qfull[g], 1);
      mbar_init(&s_qempty[g], 1);
      mbar_init(&s_drained[g], 1);
      mbar_init(&s_itemfull[g], 1);
      mbar_init(&s_itemempty[g], kThreads / 32 - 1);  // every warp but the one that searches
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&s_tmem)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t smem0 = smem_u32(smem);
  // TMEM, all 512 columns from 0 on: two score tiles for each tile of rows, 64 columns each,
  // then the outputs, D each
  auto score_at = [](int g, uint32_t i) {
    return static_cast<uint32_t>((2 * g + (i & 1)) * kKeys);
  };
  auto out_at = [](int g) { return static_cast<uint32_t>(4 * kKeys + g * D); };
  // Bounded waits, short as code; each role reports its own that ran out.
  auto done_waiting = [](uint64_t* bar, uint32_t parity) {
    const uint32_t addr = smem_u32(bar);
    bool yes = mbar_try_wait(addr, parity);
    if (!yes) {
      const uint32_t from = clock();
      do {
        yes = mbar_try_wait(addr, parity);
      } while (!yes && static_cast<uint32_t>(clock()) - from < kWaitCycles);
    }
    return yes;
  };
  auto here = [&](uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, done_waiting(bar, parity)) != 0;
  };
  bool ok = true;
  auto work_of = [&](const Item& it) {
    Work w;
    const int64_t len = min(static_cast<int64_t>(max(it.len, 0)), p.max_seqlen);
    const uint32_t group = p.group;
    w.len = static_cast<int>(len);
    w.before = len - it.n;
    w.packed = it.live * group;
    w.row0 = it.block * 2 * kRows;
#pragma unroll
    for (int g = 0; g < 2; ++g) {  // up to its last row's limit
      const uint32_t from = w.row0 + g * kRows, last = min(from + kRows, w.packed);
      const int64_t see =
          from < w.packed ? min(len, w.before + maps.group(last - 1) + 1) : 0;
      w.tiles[g] = see > 0 ? static_cast<int>((see + kKeys - 1) / kKeys) : 0;
    }
    w.ntiles = max(w.tiles[0], w.tiles[1]);
    return w;
  };
  // The turn'th item of this CTA, for all roles but the one that finds it: false at the end.
  auto next_item = [&](uint32_t turn, Item& it) {
    ok = here(&s_itemfull[turn & 1], (turn >> 1) & 1);
    if (!ok) return false;
    it = s_item[turn & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&s_itemempty[turn & 1]);
    return it.req >= 0;
  };
  // The work of CTA `index`: KV head index % hkv (the heads of one block of rows next to each
  // other, as they read the same slots) of the block of 256 packed rows that is index / hkv'th by
  // its tiles of keys, the most first, so that the last ones to end are short. Requests in order
  // among equals. A request's blocks see ever more keys, so how many of them have t tiles or more
  // is a formula, and t a bisection over its sum (lane l has requests l, l + 32, ..).
  int last_hi = -1, last_count = 0;
  auto find = [&](int index, Item* item) {
    const int kvh = index % p.hkv, rank = index / p.hkv;
    if (last_hi == 0 && rank >= last_count) return;  // (there are last_count blocks in all)
    struct Req {
      int from, n, live, len, blocks;
      int64_t before;
    };
    auto request = [&](int r) {
      Req q{0, 0, 0, 0, 0, 0};
      if (r < p.num_reqs) {
        q.from = p.cu_seqlens_q[r];
        q.n = p.cu_seqlens_q[r + 1] - q.from;
        q.len = p.cache_seqlens[r];
        q.before = min(static_cast<int64_t>(max(q.len, 0)), p.max_seqlen) - q.n;
        if (q.n > 0 && q.from >= 0 && q.from < p.rows) {
          q.live = static_cast<int>(min(static_cast<int64_t>(q.n), p.rows - q.from));
          q.blocks = (q.live * p.group + 2 * kRows - 1) / (2 * kRows);
        }
      }
      return q;
    };
    // blocks of a request with at least t tiles of keys: those whose last packed row is at
    // position `behind` at least
    auto with_tiles = [&](const Req& q, int t) -> int {
      const int64_t behind = static_cast<int64_t>(kKeys) * (t - 1) - q.before;
      if (t == 0 || behind <= 0) return q.blocks;
      if (behind >= q.live) return 0;
      return q.blocks - (static_cast<int>(behind) * p.group) / (2 * kRows);
    };
    const Req first = request(lane);
    auto count = [&](int t) {
      int c = 0;
      Req q = first;
      for (int r = lane;;) {
        c += with_tiles(q, t);
        if ((r += 32) >= p.num_reqs) break;
        q = request(r);
      }
      return __reduce_add_sync(0xffffffffu, c);
    };
    // count(lo) > rank >= count(hi); lo stays -1 if there are not so many blocks. As a rule a CTA's
    // ranks grow, so that the last one's hi holds still, and its lo is not far below; nothing
    // promises the order, so a lower rank than that hi's begins anew.
    int lo = -1, hi = last_hi, at_hi = last_count, step = 1;
    if (rank < at_hi) {
      hi = -1;
      at_hi = 0;
    }
    if (hi < 0) {
      int most = first.len;
      for (int r = lane + 32; r < p.num_reqs; r += 32) most = max(most, p.cache_seqlens[r]);
      most = __reduce_max_sync(0xffffffffu, most);
      if (static_cast<int64_t>(most) > p.max_seqlen) most = static_cast<int>(p.max_seqlen);
      step = hi = max(most, 0) / kKeys + 2;
    }
    while (hi > lo + 1) {
      const int mid = lo >= 0 ? (lo + hi) >> 1 : max(hi - step, 0), c = count(mid);
      if (c > rank) {
        lo = mid;
      } else {
        hi = mid;
        at_hi = c;
        step <<= 1;
      }
    }
    last_hi = hi;
    last_count = at_hi;
    int left = rank - at_hi;  // among those with exactly lo tiles
    bool taken = lo < 0;
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
          item->req = base + lane;
          item->kvh = kvh;
          item->block = q.blocks - with_tiles(q, lo) + left - (incl - mine);
          item->from = q.from;
          item->n = q.n;
          item->live = q.live;
          item->len = q.len;
        }
      }
      left -= __shfl_sync(0xffffffffu, incl, 31);
    }
  };
  Item it;

  if (warp >= kIssueWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (warp < kCopyWarp) {
      // ---- products. The whole warp walks the tiles, so that addresses stay uniform; one lane
      // issues.
      const int g = __shfl_sync(0xffffffffu, warp - kIssueWarp, 0);
      const uint32_t qd = operand(smem0 + S::q + g * S::kQ), kd = operand(smem0 + S::k),
                     vd = operand(smem0 + S::v);
      // the ring position of the next K and V tile
      int kst = 0, vst = 0;
      uint32_t kph = 0, vph = 0, done = 0;  // tiles of this tile of rows before this item
      for (uint32_t turn = 0; ok && next_item(turn, it); ++turn) {
        const Work w = work_of(it);
        const int mine = __shfl_sync(0xffffffffu, g ? w.tiles[1] : w.tiles[0], 0);
        const int all = __shfl_sync(0xffffffffu, w.ntiles, 0);
        auto scores = [&](int i) {
          if (!here(&s_kfull[kst], kph)) return false;
          fence_after();
          if (elect_one()) {
            if (i < mine) {
              const uint32_t b = kd + kst * (S::kK >> 4), d = score_at(g, done + i);
#pragma unroll
              for (int s = 0; s < D / 16; ++s)
                umma(d, qd + (s >> 2) * (kRows * 128 >> 4) + 2 * (s & 3),
                     b + (s >> 2) * (kKeys * 128 >> 4) + 2 * (s & 3), bf16_shape(kKeys), s > 0);
              umma_commit(&s_sfull[g][(done + i) & 1]);
              umma_commit(&s_kempty[kst]);
              if (i == mine - 1) umma_commit(&s_qempty[g]);
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
        ok = here(&s_qfull[g], turn & 1);
        fence_after();
        if (ok && mine == 0 && elect_one()) mbar_arrive(&s_qempty[g]);
        __syncwarp();
        for (int i = -2; i < all && ok; ++i) {
          if (i >= 0) {
            const uint32_t at = done + i;
            ok = here(&s_vfull[vst], vph);
            if (ok && i < mine) ok = here(&s_pfull[g][at & 1], (at >> 1) & 1);
            if (!ok) break;
            fence_after();
            if (elect_one()) {
              if (i < mine) {
                const uint32_t b = vd + vst * (S::kV >> 4), a = score_at(g, at);
#pragma unroll
                for (int s = 0; s < kKeys / 16; ++s)
                  umma_tmem(out_at(g), a + 8 * s, b + 2 * s, f16_shape(D), i > 0 || s > 0);
                umma_commit(&s_odone[g][at & 1]);
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
          }
          if (i + 2 < all) ok = scores(i + 2);
        }
        done += mine;
      }
      if (!ok) {  // no product may outlive the CTA
        if (elect_one()) umma_commit(&s_drained[g]);
        __syncwarp();
        done_waiting(&s_drained[g], 0);
      }
    } else {
      // ---- copies: one warp of K and the first tile of Q, one of V, the scales and the second.
      // The first also finds the items.
      const bool is_v = warp == kCopyWarp + 1;
      uint64_t* const full = s_rawfull[is_v], * const empty = s_rawempty[is_v];
      const uint32_t raw = smem0 + (is_v ? S::raw_v : S::raw_k);
      const CUtensorMap* const map = is_v ? &maps.v : &maps.k;
      const CUtensorMap* const box_map = is_v ? &maps.v_box : &maps.k_box;
      const int box = maps.box, boxes = box > 0 ? kKeys / box : 1;
      const int box_shift = box > 0 ? __ffs(box / kBoxMin) - 1 : 0;
      int rs = 0;
      uint32_t phase = 0;
      uint32_t asked = 0, answers = 0, filled = 0;  // (filled: tiles of codes)
      auto ask = [&] {
        if (lane == 0) {
          mbar_expect_tx(&s_answered, 16);
          ask_next(&s_answer, &s_answered);
        }
        ++asked;
        __syncwarp();
      };
      auto answer = [&](int& index) {
        const bool fine = here(&s_answered, answers & 1);
        ++answers;
        if (fine) index = next_of(&s_answer);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        return fine;
      };
      // Finds the turn'th item, asks for the one behind it. False on a timeout.
      auto search = [&](uint32_t turn) {
        bool fine = here(&s_itemempty[turn & 1], ((turn >> 1) & 1) ^ 1);
        int index = blockIdx.x;  // of the CTA whose work is next
        if (fine && turn > 0) fine = answer(index);
        Item* const item = &s_item[turn & 1];
        if (lane == 0) item->req = -1;
        __syncwarp();
        // A CTA without work is called off here, needing no start, and the next one asked for.
        bool found = false;
        while (fine && index >= 0) {
          find(index, item);
          __syncwarp();
          found = item->req >= 0;
          if (found) break;
          ask();
          fine = answer(index);
        }
        if (lane == 0) {
          if (found && item->len > p.max_seqlen && p.error_flag)
            atomicOr(p.error_flag, LSB_DEVERR_SEQLEN);
          mbar_arrive(&s_itemfull[turn & 1]);
        }
        __syncwarp();
        if (found) ask();
        return fine;
      };
      Work w{};
      const int32_t* pages = p.page_table;
      const uint32_t page_size = p.page_size, num_slots = static_cast<uint32_t>(p.num_slots);
      // the slot of a key, num_slots where there is none
      auto slot_of = [&](int key, uint32_t page) {
        const uint32_t s = page * page_size + key - maps.page(key) * page_size;
        const bool there = key < w.len, in = there && page < maps.num_pages && s < num_slots;
        if (there && !in && p.error_flag) atomicOr(p.error_flag, LSB_DEVERR_SLOT);
        return in ? s : num_slots;
      };
      auto page_of = [&](int key) -> uint32_t {
        return key < w.len ? pages[maps.page(key)] : 0;
      };
      // Boxes, 32 at a time: lane l has the first slot of box l of these, and the page of box l of
      // the next.
      uint32_t box_slot = num_slots, next_page = 0;
      uint32_t turn = 0, found = 0;  // items begun, and (K's warp) looked for
      for (int i = 0;; ++i) {
        // the next item, once the rings are full of this one's tiles
        if (!is_v && found == turn && (i == w.ntiles || i == kStages + kRawStages)) {
          ok = search(found);
          if (!ok) break;
          ++found;
        }
        if (i == w.ntiles) {
          if (is_v) {
            if (!next_item(turn, it)) break;
          } else {
            it = s_item[turn & 1];
            if (it.req < 0) break;
          }
          w = work_of(it);
          // the tile of queries
          ok = here(&s_qempty[is_v], (turn & 1) ^ 1);
          if (!ok) break;
          const uint32_t group = p.group, qt = smem0 + S::q + is_v * S::kQ;
          const uint32_t first = w.row0 + (is_v ? kRows : 0);  // its first packed row
          if (maps.q_tiled) {  // (positions past the request's take its place: rows nobody reads)
            if (lane == 0) {
              mbar_expect_tx(&s_qfull[is_v], S::kQ);
#pragma unroll
              for (int c = 0; c < S::kSlabs; ++c)
                load_box(qt + c * (kRows * 128), &maps.q, 64 * c, it.kvh * p.group,
                         it.from + static_cast<int>(maps.group(first)), &s_qfull[is_v]);
            }
          } else {
            constexpr int ROW = D / 8;
#pragma unroll 1
            for (int i = lane; i < kRows * ROW; i += 32) {
              const int r = i / ROW, chunk = i - r * ROW;
              const uint32_t j = maps.group(first + r), h = first + r - j * group;
              const bool there = j < static_cast<uint32_t>(it.live);
              const bf16* const src =
                  p.q + (there ? (it.from + static_cast<int64_t>(j)) * p.q_stride +
                                     (static_cast<int64_t>(it.kvh) * group + h) * D + 8 * chunk
                               : 0);
              copy16(qt + (chunk >> 3) * (kRows * 128) + swizzled(r, chunk & 7), src, there);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_operands();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_qfull[is_v]);
          }
          pages = p.page_table + it.req * p.pt_stride;
          if (box > 0) next_page = page_of(lane * box);
          ++turn;
          i = -1;
          continue;
        }
        bool whole = box > 0 && (i + 1) * kKeys <= w.len;
        const int at = i * kKeys / kBoxMin >> box_shift;  // the tile's first box
        if (whole) {
          if ((at & 31) == 0) {
            box_slot = slot_of((at + lane) * box, next_page);
            next_page = page_of((at + 32 + lane) * box);
          }
          const uint32_t first = __shfl_sync(0xffffffffu, box_slot, at + (lane & (boxes - 1)));
          whole = __all_sync(0xffffffffu, first + box <= num_slots);
        }
        ok = here(&empty[rs], phase ^ 1);
        if (!ok) break;
        const uint32_t dst = raw + rs * S::kRaw;
        const uint32_t rsc = smem0 + S::raw_scales + (rs * 2 * kKeys + lane) * 4;
        uint32_t mask[2] = {0xffffffffu, 0xffffffffu};
        int shift = 0;  // of a key to its place among the scales
        uint32_t slot[2];
        if (whole && (!is_v || p.block_shift >= 2)) {
          if (is_v) {  // a scale for each block: K's from lanes 0-15, V's from lanes 16-31
            shift = min(p.block_shift, 6);
            const int key = (lane & 15) << shift;
            const uint32_t s =
                __shfl_sync(0xffffffffu, box_slot, at + (key / kBoxMin >> box_shift)) +
                (key & (box - 1));
            if (key < kKeys)
              copy4(rsc + (lane & 16 ? (kKeys - 16) * 4 : 0),
                    (lane & 16 ? p.vs : p.ks) +
                        static_cast<uint64_t>(s >> p.block_shift) * p.hkv + it.kvh,
                    true);
          }
        } else {
#pragma unroll 1
          for (int e = 0; e < 2; ++e) {
            const int key = i * kKeys + 32 * e + lane;
            const uint32_t s = slot_of(key, page_of(key));
            const bool in = s < num_slots;
            const uint32_t m = __ballot_sync(0xffffffffu, in);
            if (e) {
              slot[1] = s;
              mask[1] = m;
            } else {
              slot[0] = s;
              mask[0] = m;
            }
            if (is_v) {
              const uint64_t of =
                  in ? static_cast<uint64_t>(s >> p.block_shift) * p.hkv + it.kvh : 0;
              copy4(rsc + 128 * e, p.ks + of, in);
              copy4(rsc + 128 * e + kKeys * 4, p.vs + of, in);
            }
          }
        }
        if (is_v) copies_arrive(&full[rs]);
        if (lane == 0) {
          if (is_v)
            *reinterpret_cast<uint4*>(smem + S::valid + rs * 16) =
                make_uint4(mask[0], mask[1], shift, 0);
          mbar_expect_tx(&full[rs], S::kRaw);
        }
        const uint32_t first = __shfl_sync(0xffffffffu, box_slot, at + (lane & (boxes - 1)));
        if (whole) {
          if (lane < boxes)
            load_box(dst + lane * (box * D), box_map, it.kvh * D, first, &full[rs]);
        } else {  // keys 4 * lane .. a lane
          int r[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int lo = __shfl_sync(0xffffffffu, slot[0], (4 * lane + e) & 31);
            const int hi = __shfl_sync(0xffffffffu, slot[1], (4 * lane + e) & 31);
            r[e] = lane < 8 ? lo : hi;
          }
          if (lane < 16)
            gather4(dst + lane * (4 * D), map, it.kvh * D, r[0], r[1], r[2], r[3], &full[rs]);
        }
        ++filled;
        if (++rs == kRawStages) {
          rs = 0;
          phase ^= 1;
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (!ok) {  // nor may a copy or an answer
#pragma unroll 1
        for (uint32_t s = 0; s < kRawStages && s < filled; ++s)
          done_waiting(&full[s], ((filled - 1 - s) / kRawStages) & 1);
        if (turn > 0) done_waiting(&s_qfull[is_v], (turn - 1) & 1);
        if (asked > answers) done_waiting(&s_answered, answers & 1);
      }
    }
  } else if (warp >= kSoftWarps + kWidenWarps) {
    // ---- V: 32 keys x 16 dims a warp at a time, transposed
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWidenVRegs));
    const int wt = tid - 32 * (kSoftWarps + kWidenWarps), ww = wt >> 5;
    constexpr int LOADS = 2 * CHUNKS / kWidenWarps;
    const int t4 = lane & 3, g8 = lane >> 2;
    int st = 0, rs = 0;
    uint32_t ph = 0, rph = 0;
    for (uint32_t turn = 0; ok && next_item(turn, it); ++turn) {
      const Work w = work_of(it);
      for (int i = 0; i < w.ntiles; ++i) {
        ok = here(&s_rawfull[1][rs], rph) && here(&s_vempty[st], ph ^ 1);
        if (!ok) break;
        // Keys that some row of the CTA must not see although others do: a NaN code would reach
        // it through 0 * NaN, so it becomes 0 and the key's scale NaN (which only rows that see
        // the key take in; those that see the whole tile by `whole`)
        const bool diagonal = !INT8 && (i + 1) * static_cast<int64_t>(kKeys) >
                                           w.before + maps.group(w.row0) + 1;
        const uint32_t src = smem0 + S::raw_v + rs * S::kRaw;
        // this warp's units: keys 32 half .., dims 16 (2j + ww / 2) ..
        const int half = ww & 1;
        uint8_t* const vt = smem + S::v + st * S::kV + (ww >> 1) * 16 * 128 + 8 * (t4 & 1);
        // keys 32 half + 16 hi + 4 t4 .., dims g8 and g8 + 8 of 16
        uint8_t* const at[2] = {vt + swizzled(g8, 4 * half + (t4 >> 1)),
                                vt + swizzled(g8, 4 * half + 2 + (t4 >> 1))};
#pragma unroll 1
        for (int j = 0; j < LOADS; ++j) {
          uint32_t r[4];
          load_columns(r, src + raw_offset<D>(32 * half + lane, 2 * j + (ww >> 1)));
          if (diagonal) {
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] &= ~nan_bytes<INT8>(r[e]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint2 h;
            q8_decode4<INT8>(r[e], h.x, h.y);
            *reinterpret_cast<uint2*>(at[e >> 1] + (32 * j + 8 * (e & 1)) * 128) = h;
          }
        }
        if (wt < kKeys) {
          const uint4 valid_of = *reinterpret_cast<const uint4*>(smem + S::valid + rs * 16);
          const float* const rsc = reinterpret_cast<const float*>(smem + S::raw_scales) +
                                   rs * 2 * kKeys + (wt >> valid_of.z);
          const float vs = rsc[kKeys];
          const uint32_t valid = wt < 32 ? valid_of.x : valid_of.y;
          const float held = fmaxf(vs, 7.888609e-31f);  // 2^-100: less counts as that
          float ks = rsc[0] * p.scale_log2, lv = vs != vs ? vs : log2_fast(held),
                iv = inverse_fast(held);
          if (!((valid >> lane) & 1)) {
            ks = iv = 0.f;
            lv = -INFINITY;
          }
          float whole = lv;
          if (diagonal) {  // (keys that there are not have codes of zero)
            bool bad = false;
#pragma unroll 1
            for (int c = 0; c < CHUNKS; ++c)
              bad |= any_nan<INT8>(*reinterpret_cast<const uint4*>(
                  smem + S::raw_v + rs * S::kRaw + raw_offset<D>(wt, c)));
            if (bad) lv = __uint_as_float(kNanBits);
            if (__any_sync(0xffffffffu, bad)) whole = __uint_as_float(kNanBits);
          }
          reinterpret_cast<KeyScales*>(smem + S::scales)[st * kKeys + wt] = {ks, lv, iv, whole};
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_rawempty[1][rs]);
        fence_operands();
        mbar_arrive(&s_vfull[st]);
        if (++st == kStages) {
          st = 0;
          ph ^= 1;
        }
        if (++rs == kRawStages) {
          rs = 0;
          rph ^= 1;
        }
      }
    }
  } else if (warp >= kSoftWarps) {
    // ---- K: 16 codes of a key a thread at a time
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWidenKRegs));
    const int wt = tid - 32 * kSoftWarps;
    constexpr int LOADS = kKeys * CHUNKS / kWidenThreads;
    // Unit j of a thread: in the first slab of 64 dims four threads a key, so that the 16-byte
    // stores of 8 threads (two keys, every other chunk) fall in different banks.
    constexpr int kPer0 = CHUNKS < 4 ? CHUNKS : 4, kPer1 = CHUNKS > 4 ? CHUNKS - 4 : 1;
    constexpr int kFirst = kKeys * kPer0 / kWidenThreads;
    int st = 0, rs = 0;
    uint32_t ph = 0, rph = 0;
    for (uint32_t turn = 0; ok && next_item(turn, it); ++turn) {
      const int ntiles = work_of(it).ntiles;
      for (int i = 0; i < ntiles; ++i) {
        ok = here(&s_rawfull[0][rs], rph) && here(&s_kempty[st], ph ^ 1);
        if (!ok) break;
        const uint8_t* const src = smem + S::raw_k + rs * S::kRaw;
        uint8_t* const kt = smem + S::k + st * S::kK;
#pragma unroll 1
        for (int j = 0; j < LOADS; ++j) {
          const bool second = j >= kFirst;
          const int n = (second ? j - kFirst : j) * kWidenThreads + wt;
          const int per = second ? kPer1 : kPer0;
          const int key = n / per, c = n - key * per;
          const uint4 u = *reinterpret_cast<const uint4*>(src + raw_offset<D>(key, c + 4 * second));
          uint8_t* const slab = kt + second * (kKeys * 128);
          uint4 h[2];
          decode4_bf16<INT8>(u.x, h[0].x, h[0].y);
          decode4_bf16<INT8>(u.y, h[0].z, h[0].w);
          decode4_bf16<INT8>(u.z, h[1].x, h[1].y);
          decode4_bf16<INT8>(u.w, h[1].z, h[1].w);
          if (any_nan<INT8>(u)) h[0].x = 0x7fff7fffu;  // one NaN makes the key's score NaN
          *reinterpret_cast<uint4*>(slab + swizzled(key, 2 * c)) = h[0];
          *reinterpret_cast<uint4*>(slab + swizzled(key, 2 * c + 1)) = h[1];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_rawempty[0][rs]);
        fence_operands();
        mbar_arrive(&s_kfull[st]);
        if (++st == kStages) {
          st = 0;
          ph ^= 1;
        }
        if (++rs == kRawStages) {
          rs = 0;
          rph ^= 1;
        }
      }
    }
  } else {
    // ---- softmax: a thread per row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    const int g = warp >> 2;  // tile of rows
    const int trow = tid & (kRows - 1);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t o_at = lanes + out_at(g);
    // Neighbouring keys with one scale (in pools of whole blocks, where they exist together; a
    // negative factor would turn the order of their scores around). 8 prompts of 1000 tokens in
    // blocks of 4: 81 us, a key at a time 104.
    const bool ordered = p.scale_log2 >= 0.f;
    const bool four = ordered && p.block_shift >= 2 && p.num_slots % 4 == 0;
    const bool sixteen = ordered && p.block_shift >= 4 && p.num_slots % 16 == 0;
    uint32_t done = 0;         // tiles of this tile of rows before this item
    uint32_t st = 0, ph = 0;  // the ring position of the next V tile
    auto advance = [&] {
      if (++st == kStages) {
        st = 0;
        ph ^= 1;
      }
    };
    for (uint32_t turn = 0; ok && next_item(turn, it); ++turn) {
      const Work w0 = work_of(it);
      const uint32_t prow = w0.row0 + g * kRows + trow;  // packed row
      const uint32_t pos = maps.group(prow);
      const bool mine = prow < w0.packed;
      const int tiles = g ? w0.tiles[1] : w0.tiles[0];
      // last key this row sees (a row of zeros behind the last one takes what comes), and that
      // every row of the warp sees
      const int limit = mine ? static_cast<int>(max(w0.before + pos, int64_t(-1))) : w0.len;
      const int common = __reduce_min_sync(0xffffffffu, limit);
      float m = kLow, sum = 0.f;
      bool far = false;  // some row's m in the warp is
      for (int i = 0; i < tiles; ++i) {
        const uint32_t at = done + i;
        // The scores first: they are issued after V of two tiles before is in (or of the whole item
        // before), so that stage's last use lies behind it and its parity stands for this tile. A
        // tile of rows that skipped an item's keys would otherwise test the barrier phases early,
        // when the parity of the one before the last reads as done.
        ok = __all_sync(0xffffffffu, done_waiting(&s_sfull[g][at & 1], (at >> 1) & 1) &&
                                         done_waiting(&s_vfull[st], ph));
        if (!ok) break;
        fence_after();
        const uint32_t s_at = lanes + score_at(g, at);
        const KeyScales* const sc =
            reinterpret_cast<const KeyScales*>(smem + S::scales) + st * kKeys;
        advance();
        const int sees = limit - i * kKeys;  // last visible key of the tile
        const bool full = common - i * kKeys >= kKeys - 1;
        const float top = full && sixteen ? largest_score<16>(s_at, sc, m)
                          : full && four  ? largest_score<4>(s_at, sc, m)
                                          : largest_score(s_at, sc, m, sees);
        const bool grows = top > m + kGrowth;
        if (__any_sync(0xffffffffu, grows)) {
          const float f = grows ? exp2_fast(m - top) : 1.f;
          if (grows) m = top;
          far = __any_sync(0xffffffffu, fabsf(m) >= kFar && m != kLow);
          sum *= f;
          if (i > 0) {  // O, once the product before is in
            ok = here(&s_odone[g][(at - 1) & 1], ((at - 1) >> 1) & 1);
            if (!ok) break;
            fence_after();
#pragma unroll 1
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
        sum += full && !far && sixteen ? store_weights<16>(s_at, sc, m)
               : full && !far && four  ? store_weights<4>(s_at, sc, m)
                                       : store_weights(s_at, sc, m, sees);
        tmem_store_wait();
        fence_before();
        mbar_arrive(&s_pfull[g][at & 1]);
      }
      done += tiles;
      for (int i = tiles; i < w0.ntiles; ++i) advance();
      // ---- output
      if (ok && tiles > 0) ok = here(&s_odone[g][(done - 1) & 1], ((done - 1) >> 1) & 1);
      if (ok) {
        fence_after();
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        bf16* const dst = p.out + (it.from + static_cast<int64_t>(pos)) * p.out_stride +
                          (static_cast<int64_t>(it.kvh) * p.group + prow - pos * p.group) * D;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          float o[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0.f;
          if (tiles > 0) {
            tmem_load16(o_at + c, o);
            tmem_load_wait();
          }
          if (mine) {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = sum == 0.f ? 0.f : o[e] * inv;
            const bf16x8 lo = pack8(o), hi = pack8(o + 8);
            *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(&lo);
            *reinterpret_cast<uint4*>(dst + c + 8) = *reinterpret_cast<const uint4*>(&hi);
          }
        }
      }
    }
    fence_before();
  }
  if (!ok && lane == 0 && p.error_flag) atomicOr(p.error_flag, LSB_DEVERR_TIMEOUT);
  __syncthreads();
  if (warp == kIssueWarp) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s_tmem), "r"(512));
  }
}

// A tensor of `dims` elements, innermost first, and boxes of it.
int tensor_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* ptr,
               const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
               CUtensorMapSwizzle swizzle) {
  static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  if (!encode) return fail(LSB_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint32_t elem[3] = {1, 1, 1};
  const CUresult r = encode(map, type, rank, const_cast<void*>(ptr), dims, strides, box, elem,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(LSB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
  return LSB_OK;
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
  LSB_REQUIRE(blocks * p.hkv < (int64_t(1) << 31) && blocks * 2 * kRows < (int64_t(1) << 31),
              "paged_attention_q8: too many rows");
  Maps maps{};
  constexpr CUtensorMapSwizzle kCodes = D == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                        : D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                        : D == 32 ? CU_TENSOR_MAP_SWIZZLE_32B
                                                  : CU_TENSOR_MAP_SWIZZLE_NONE;
  maps.num_pages = static_cast<uint32_t>((p.num_slots - 1) / p.page_size + 1);
  maps.page = divisor(p.page_size);
  maps.group = divisor(p.group);
  maps.box = kKeys;
  while (maps.box > 0 && p.page_size % maps.box) maps.box = maps.box > kBoxMin ? maps.box / 2 : 0;
  const cuuint64_t slots[2] = {static_cast<cuuint64_t>(p.hkv) * D,
                               static_cast<cuuint64_t>(p.num_slots)};
  const cuuint64_t slot_bytes[1] = {static_cast<cuuint64_t>(p.slot_stride)};
  const cuuint32_t one[2] = {D, 1}, box[2] = {D, static_cast<cuuint32_t>(maps.box)};
  auto codes_map = [&](CUtensorMap* map, const uint8_t* codes, const cuuint32_t* shape) {
    return tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, slots, slot_bytes, shape,
                      kCodes);
  };
  int rc = codes_map(&maps.k, p.k, one);
  if (!rc) rc = codes_map(&maps.v, p.v, one);
  if (!rc && maps.box > 0) rc = codes_map(&maps.k_box, p.k, box);
  if (!rc && maps.box > 0) rc = codes_map(&maps.v_box, p.v, box);
  maps.q_tiled = kRows % p.group == 0;
  if (!rc && maps.q_tiled) {
    const cuuint64_t heads[3] = {D, static_cast<cuuint64_t>(p.hkv) * p.group,
                                 static_cast<cuuint64_t>(p.rows)};
    const cuuint64_t strides[2] = {2 * D, 2 * static_cast<cuuint64_t>(p.q_stride)};
    const cuuint32_t tile[3] = {64, static_cast<cuuint32_t>(p.group),
                                static_cast<cuuint32_t>(kRows / p.group)};
    rc = tensor_map(&maps.q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, p.q, heads, strides, tile,
                    CU_TENSOR_MAP_SWIZZLE_128B);
  }
  if (rc) return rc;
  kernel<<<static_cast<unsigned>(blocks * p.hkv), kThreads, Smem<D>::total, stream>>>(p, maps);
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
