// Appending to the 8-bit paged KV cache: the neox rotation of the q and k heads of a fused
// QKV projection, and the k and v heads quantised into their slots under one scale per block
// of slots and KV head (q8.cuh).
//
// Per touched block and head, K and V apart: amax over the call's tokens, the scale the
// larger of the block's own (nothing when the call starts at the block's first slot) and the
// one amax needs; a scale that grows re-expresses the block's earlier codes. Values are
// quantised from the fp32 rotation, not from its bf16 rounding: one rounding instead of two.
//
// Eight lanes own one head of one token, 8 + 8 elements each (dims 8c.. and half + 8c.., the
// two sides of the rotation), so loads are 16 bytes and the amax of a head is three shuffles.
// With blocks of one token a warp takes four (token, head) items; with larger blocks a warp
// takes one head of one run (the call's adjacent tokens of one block), its four lane groups a
// quarter of the tokens each, up to 16 tokens held in registers between the amax and the
// rounding.
#include "q8.cuh"

namespace lsb {
namespace {

struct Q8StoreParams {
  const bf16* q;  // nullptr: nothing to rotate into q_out
  int64_t q_stride;
  bf16* q_out;
  int64_t q_out_stride;
  const bf16 *k, *v;  // first k / v head of row 0
  int64_t k_stride, v_stride;
  const int32_t* positions;
  const float* cos_sin;  // nullptr: no rotation
  int64_t max_pos;
  uint8_t *k_cache, *v_cache;
  int64_t slot_stride, num_slots;
  float *k_scale, *v_scale;
  int block_shift;
  const int32_t* out_loc;
  int64_t tokens;
  int hq, hkv;
  int tile;            // tokens whose runs one warp takes (blocks of several tokens)
  int64_t kv_blocks;   // CTAs of the grid that store; the rest rotate q
  int* error_flag;
};

constexpr int kStoreWarps = 8;

__device__ __forceinline__ bf16x8 load8(const bf16* p) {
  bf16x8 v;
  *reinterpret_cast<uint4*>(&v) = *reinterpret_cast<const uint4*>(p);
  return v;
}

__device__ __forceinline__ int checked_position(const Q8StoreParams& p, int64_t t) {
  const int pos = p.positions[t];
  if (pos >= 0 && pos < p.max_pos) return pos;
  if (p.error_flag) atomicOr(p.error_flag, LSB_DEVERR_POSITION);
  return 0;
}

// Rotates the pairs (x[i], x[8 + i]), dims 8c + i and half + 8c + i, by row `cs` of the table.
template <int D>
__device__ __forceinline__ void rotate8(float* x, const float* cs, int c) {
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    const float4 cc = *reinterpret_cast<const float4*>(cs + 8 * c + i);
    const float4 ss = *reinterpret_cast<const float4*>(cs + D / 2 + 8 * c + i);
    rope_rotate(x[i], x[8 + i], cc.x, ss.x, x[i], x[8 + i]);
    rope_rotate(x[i + 1], x[9 + i], cc.y, ss.y, x[i + 1], x[9 + i]);
    rope_rotate(x[i + 2], x[10 + i], cc.z, ss.z, x[i + 2], x[10 + i]);
    rope_rotate(x[i + 3], x[11 + i], cc.w, ss.w, x[i + 3], x[11 + i]);
  }
}

// The 16 elements of lane c of head hh (k heads, then v heads) of token t, k heads rotated.
template <int D>
__device__ __forceinline__ void load_head(const Q8StoreParams& p, int64_t t, int hh, int c,
                                          float* x) {
  const bool is_v = hh >= p.hkv;
  const bf16* src = is_v ? p.v + t * p.v_stride + static_cast<int64_t>(hh - p.hkv) * D
                         : p.k + t * p.k_stride + static_cast<int64_t>(hh) * D;
  unpack8(load8(src + 8 * c), x);
  unpack8(load8(src + D / 2 + 8 * c), x + 8);
  if (!is_v && p.cos_sin)
    rotate8<D>(x, p.cos_sin + static_cast<int64_t>(checked_position(p, t)) * D, c);
}

__device__ __forceinline__ uint32_t amax16(const float* x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  return m;
}

template <int D, bool INT8>
__device__ __forceinline__ void store_codes(uint8_t* row, int c, const float* x, float inv) {
  uint2 lo, hi;
  lo.x = q8_encode4<INT8>(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
  lo.y = q8_encode4<INT8>(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
  hi.x = q8_encode4<INT8>(x[8] * inv, x[9] * inv, x[10] * inv, x[11] * inv);
  hi.y = q8_encode4<INT8>(x[12] * inv, x[13] * inv, x[14] * inv, x[15] * inv);
  *reinterpret_cast<uint2*>(row + 8 * c) = lo;
  *reinterpret_cast<uint2*>(row + D / 2 + 8 * c) = hi;
}

// A slot the call may write: not the padding slot 0, within the pool.
__device__ __forceinline__ bool writable(const Q8StoreParams& p, int64_t loc) {
  return loc > 0 && loc < p.num_slots;
}

template <int D, bool INT8>
__global__ void __launch_bounds__(32 * kStoreWarps) q8_store_kernel(Q8StoreParams p) {
  constexpr int kLanes = D / 16;  // lanes of eight that hold a head
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int grp = lane >> 3, c = lane & 7;
  const bool on = c < kLanes;
  const int heads = 2 * p.hkv;

  if (blockIdx.x >= p.kv_blocks) {  // q: one thread per 8 + 8 elements
    const int64_t i =
        (static_cast<int64_t>(blockIdx.x) - p.kv_blocks) * (32 * kStoreWarps) + threadIdx.x;
    const int64_t row_items = static_cast<int64_t>(p.hq) * kLanes;
    const int64_t t = i / row_items;
    if (t >= p.tokens) return;
    const int r = static_cast<int>(i - t * row_items);
    const int h = r / kLanes, qc = r - h * kLanes;
    const bf16* src = p.q + t * p.q_stride + static_cast<int64_t>(h) * D;
    float x[16];
    unpack8(load8(src + 8 * qc), x);
    unpack8(load8(src + D / 2 + 8 * qc), x + 8);
    rotate8<D>(x, p.cos_sin + static_cast<int64_t>(checked_position(p, t)) * D, qc);
    bf16* dst = p.q_out + t * p.q_out_stride + static_cast<int64_t>(h) * D;
    const bf16x8 lo = pack8(x), hi = pack8(x + 8);
    *reinterpret_cast<uint4*>(dst + 8 * qc) = *reinterpret_cast<const uint4*>(&lo);
    *reinterpret_cast<uint4*>(dst + D / 2 + 8 * qc) = *reinterpret_cast<const uint4*>(&hi);
    return;
  }

  const int64_t item = static_cast<int64_t>(blockIdx.x) * kStoreWarps + warp;
  if (p.block_shift == 0) {  // one token per block: a lane group per (token, head)
    const int64_t gi = item * 4 + grp;
    const int64_t t = gi / heads;
    const int hh = static_cast<int>(gi - t * heads);
    int64_t loc = 0;
    if (t < p.tokens) {
      loc = p.out_loc[t];
      if (loc != 0 && !writable(p, loc)) {
        if (c == 0 && p.error_flag) atomicOr(p.error_flag, LSB_DEVERR_SLOT);
        loc = 0;
      }
    }
    const bool live = on && loc != 0;
    float x[16];
    uint32_t amax = 0;
    if (live) {
      load_head<D>(p, t, hh, c, x);
      amax = amax16(x);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!live) return;
    const bool is_v = hh >= p.hkv;
    const int kh = is_v ? hh - p.hkv : hh;
    const uint32_t sb = q8_scale_bits<INT8>(amax);
    uint8_t* row = (is_v ? p.v_cache : p.k_cache) + loc * p.slot_stride + kh * D;
    store_codes<D, INT8>(row, c, x, q8_inverse(sb));
    if (c == 0) (is_v ? p.v_scale : p.k_scale)[loc * p.hkv + kh] = __uint_as_float(sb);
    return;
  }

  // several tokens per block: the runs that start among this warp's `tile` tokens
  const int64_t tile = item / heads;
  const int hh = static_cast<int>(item - tile * heads);
  const int64_t t0 = tile * p.tile;
  if (t0 >= p.tokens) return;
  const bool is_v = hh >= p.hkv;
  const int kh = is_v ? hh - p.hkv : hh;
  uint8_t* const cache = (is_v ? p.v_cache : p.k_cache) + static_cast<int64_t>(kh) * D;
  float* const scales = (is_v ? p.v_scale : p.k_scale) + kh;
  bool starts = false;
  {
    const int64_t t = t0 + lane;
    if (lane < p.tile && t < p.tokens) {
      const int64_t loc = p.out_loc[t];
      if (writable(p, loc)) {
        const int64_t before = t > 0 ? p.out_loc[t - 1] : 0;
        starts = !(writable(p, before) && (before >> p.block_shift) == (loc >> p.block_shift));
      } else if (loc != 0 && p.error_flag) {
        atomicOr(p.error_flag, LSB_DEVERR_SLOT);
      }
    }
  }
  for (uint32_t todo = __ballot_sync(0xffffffffu, starts); todo; todo &= todo - 1) {
    const int64_t t = t0 + __ffs(todo) - 1;
    const int64_t block = static_cast<int64_t>(p.out_loc[t]) >> p.block_shift;
    // the run's length and the first slot it writes
    int64_t n = 0;
    uint32_t first = ~0u;
    for (;;) {
      const int64_t tt = t + n + lane;
      const int64_t loc = tt < p.tokens ? p.out_loc[tt] : 0;
      const bool same = writable(p, loc) && (loc >> p.block_shift) == block;
      const uint32_t other = ~__ballot_sync(0xffffffffu, same);
      const int more = other ? __ffs(other) - 1 : 32;
      const uint32_t off = static_cast<uint32_t>(loc - (block << p.block_shift));
      first = min(first, __reduce_min_sync(0xffffffffu, lane < more ? off : ~0u));
      n += more;
      if (more < 32) break;
    }
    float x[4][16];
    auto load = [&](int64_t base) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (on && base + 4 * j + grp < n) load_head<D>(p, t + base + 4 * j + grp, hh, c, x[j]);
    };
    const uint32_t old =
        first > 0 ? __float_as_uint(scales[block * p.hkv]) & 0x7fffffffu : 0u;
    uint32_t amax = 0;
    for (int64_t base = 0; base < n; base += 16) {
      load(base);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (on && base + 4 * j + grp < n) amax = max(amax, amax16(x[j]));
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    const uint32_t sb = max(old, q8_scale_bits<INT8>(amax));
    const float inv = q8_inverse(sb);
    for (int64_t base = 0; base < n; base += 16) {
      if (n > 16) load(base);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t i = base + 4 * j + grp;
        if (on && i < n)
          store_codes<D, INT8>(cache + static_cast<int64_t>(p.out_loc[t + i]) * p.slot_stride, c,
                               x[j], inv);
      }
    }
    if (sb > old) {
      if (lane == 0) scales[block * p.hkv] = __uint_as_float(sb);
      if (old != 0 && sb < kInfBits) {  // the block's earlier tokens, in the new scale
        const float ratio = __fdiv_rn(__uint_as_float(old), __uint_as_float(sb));
        for (uint32_t r = grp; r < first; r += 4) {
          uint8_t* row = cache + ((block << p.block_shift) + r) * p.slot_stride + 16 * c;
          if (!on) continue;
          uint4 w = *reinterpret_cast<const uint4*>(row);
          uint32_t* ws = &w.x;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 f = q8_decode4f<INT8>(ws[i]);
            ws[i] = q8_encode4<INT8>(f.x * ratio, f.y * ratio, f.z * ratio, f.w * ratio);
          }
          *reinterpret_cast<uint4*>(row) = w;
        }
      }
    }
  }
}

int launch_store(Q8StoreParams& p, int head_dim, int code, cudaStream_t stream,
                 const char* what) {
  const int heads = 2 * p.hkv;
  int64_t warps;
  p.tile = 1;
  if (p.block_shift == 0) {
    warps = (p.tokens * heads + 3) / 4;
  } else {
    // a warp per (token, head) while those fit the GPU about twice over (single-token calls:
    // every token starts a run); prompts give each warp up to 16 tokens, of which one or two
    // start a run
    while (p.tile < 16 && (p.tokens / p.tile) * heads > 16384) p.tile <<= 1;
    warps = (p.tokens + p.tile - 1) / p.tile * heads;
  }
  p.kv_blocks = (warps + kStoreWarps - 1) / kStoreWarps;
  const int64_t q_items = p.q ? p.tokens * p.hq * (head_dim / 16) : 0;
  const int64_t blocks = p.kv_blocks + (q_items + 32 * kStoreWarps - 1) / (32 * kStoreWarps);
  LSB_REQUIRE(blocks < (int64_t(1) << 31), "%s: too many tokens", what);
  p.error_flag = lsb_device_error_flag();
  auto launch = [&](auto kernel) {
    kernel<<<static_cast<unsigned>(blocks), 32 * kStoreWarps, 0, stream>>>(p);
    return check_launch(what);
  };
#define LSB_Q8_STORE(DIM) \
  case DIM: return code == LSB_Q8_INT8 ? launch(q8_store_kernel<DIM, true>) \
                                       : launch(q8_store_kernel<DIM, false>);
  switch (head_dim) {
    LSB_Q8_STORE(32)
    LSB_Q8_STORE(64)
    LSB_Q8_STORE(96)
    LSB_Q8_STORE(128)
  }
#undef LSB_Q8_STORE
  return fail(LSB_ERR_UNSUPPORTED, "%s: head_dim %d", what, head_dim);
}

int check_cache(const char* what, const void* k_cache, const void* v_cache, int64_t slot_stride,
                int64_t num_slots, const float* k_scale, const float* v_scale, int32_t block,
                int32_t code, const int32_t* out_loc, int32_t hkv, int32_t head_dim) {
  LSB_REQUIRE(k_cache && v_cache && k_scale && v_scale && out_loc, "%s: null pointer", what);
  LSB_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128,
              "%s: head_dim %d unsupported (32, 64, 96, 128)", what, head_dim);
  LSB_REQUIRE(hkv > 0, "%s: bad heads", what);
  LSB_REQUIRE(code == LSB_Q8_E4M3 || code == LSB_Q8_INT8, "%s: unknown code type %d", what, code);
  LSB_REQUIRE(block >= 1 && block <= 128 && (block & (block - 1)) == 0,
              "%s: block of %d tokens (a power of two up to 128)", what, block);
  LSB_REQUIRE(slot_stride >= (int64_t)hkv * head_dim && slot_stride % 16 == 0 &&
                  aligned(k_cache, 16) && aligned(v_cache, 16),
              "%s: cache rows must be 16-byte aligned", what);
  LSB_REQUIRE(aligned(k_scale, 4) && aligned(v_scale, 4), "%s: misaligned scales", what);
  LSB_REQUIRE(num_slots > 0 && num_slots < (int64_t(1) << 31), "%s: bad slot count", what);
  return LSB_OK;
}

int shift_of(int32_t block) {
  int s = 0;
  while ((1 << s) < block) ++s;
  return s;
}

}  // namespace
}  // namespace lsb

using namespace lsb;

extern "C" int lsb_rope_store_kv_q8(const void* qkv, int64_t qkv_stride, void* q_out,
                                    int64_t q_out_stride, const int32_t* positions,
                                    const float* cos_sin, int64_t max_pos, void* k_cache,
                                    void* v_cache, int64_t slot_stride, int64_t num_slots,
                                    float* k_scale, float* v_scale, int32_t block, int32_t code,
                                    const int32_t* out_loc, int64_t tokens, int32_t hq,
                                    int32_t hkv, int32_t head_dim, void* stream) {
  const char* what = "lsb_rope_store_kv_q8";
  LSB_REQUIRE(qkv && q_out && positions && cos_sin, "%s: null pointer", what);
  if (int rc = check_cache(what, k_cache, v_cache, slot_stride, num_slots, k_scale, v_scale,
                           block, code, out_loc, hkv, head_dim))
    return rc;
  LSB_REQUIRE(hq > 0 && hq % hkv == 0, "%s: bad heads %d/%d", what, hq, hkv);
  LSB_REQUIRE(qkv_stride >= (int64_t)(hq + 2 * hkv) * head_dim && qkv_stride % 8 == 0 &&
                  q_out_stride >= (int64_t)hq * head_dim && q_out_stride % 8 == 0,
              "%s: strides must be multiples of 8 elements and hold a row", what);
  LSB_REQUIRE(aligned(qkv, 16) && aligned(q_out, 16) && aligned(cos_sin, 16),
              "%s: tensors must be 16-byte aligned", what);
  LSB_REQUIRE(max_pos > 0, "%s: empty cos/sin table", what);
  if (tokens <= 0) return LSB_OK;
  Q8StoreParams p{};
  p.q = static_cast<const bf16*>(qkv);
  p.q_stride = p.k_stride = p.v_stride = qkv_stride;
  p.q_out = static_cast<bf16*>(q_out);
  p.q_out_stride = q_out_stride;
  p.k = p.q + static_cast<int64_t>(hq) * head_dim;
  p.v = p.k + static_cast<int64_t>(hkv) * head_dim;
  p.positions = positions;
  p.cos_sin = cos_sin;
  p.max_pos = max_pos;
  p.k_cache = static_cast<uint8_t*>(k_cache);
  p.v_cache = static_cast<uint8_t*>(v_cache);
  p.slot_stride = slot_stride;
  p.num_slots = num_slots;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_shift = shift_of(block);
  p.out_loc = out_loc;
  p.tokens = tokens;
  p.hq = hq;
  p.hkv = hkv;
  return launch_store(p, head_dim, code, as_stream(stream), what);
}

extern "C" int lsb_store_kv_q8(void* k_cache, void* v_cache, int64_t slot_stride,
                               int64_t num_slots, float* k_scale, float* v_scale, int32_t block,
                               int32_t code, const void* k, int64_t k_stride, const void* v,
                               int64_t v_stride, const int32_t* out_loc, int64_t tokens,
                               int32_t hkv, int32_t head_dim, void* stream) {
  const char* what = "lsb_store_kv_q8";
  LSB_REQUIRE(k && v, "%s: null pointer", what);
  if (int rc = check_cache(what, k_cache, v_cache, slot_stride, num_slots, k_scale, v_scale,
                           block, code, out_loc, hkv, head_dim))
    return rc;
  LSB_REQUIRE(k_stride >= (int64_t)hkv * head_dim && v_stride >= (int64_t)hkv * head_dim &&
                  k_stride % 8 == 0 && v_stride % 8 == 0 && aligned(k, 16) && aligned(v, 16),
              "%s: k and v rows must be 16-byte aligned", what);
  if (tokens <= 0) return LSB_OK;
  Q8StoreParams p{};
  p.k = static_cast<const bf16*>(k);
  p.v = static_cast<const bf16*>(v);
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.k_cache = static_cast<uint8_t*>(k_cache);
  p.v_cache = static_cast<uint8_t*>(v_cache);
  p.slot_stride = slot_stride;
  p.num_slots = num_slots;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_shift = shift_of(block);
  p.out_loc = out_loc;
  p.tokens = tokens;
  p.hkv = hkv;
  return launch_store(p, head_dim, code, as_stream(stream), what);
}
