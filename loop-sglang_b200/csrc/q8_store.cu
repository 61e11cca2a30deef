// Appending to the 8-bit paged KV cache: the neox rotation of the q and k heads of a fused
// QKV projection, and the k and v heads quantised into their slots under one scale per block
// of slots and KV head (q8.cuh).
//
// Per touched block and head, K and V apart: amax over the call's tokens, the scale the
// larger of the block's own (nothing when the call starts at the block's first slot, which
// then takes its scale whatever was there) and the one amax needs; a scale that grows
// re-expresses the block's earlier codes. Values are
// quantised from the fp32 rotation, not from its bf16 rounding: one rounding instead of two.
//
// D / 16 lanes (8 at 96 dims) own one head of a token, 8 + 8 elements each (dims 8c.. and
// half + 8c.., the two sides of the rotation), so loads are 16 bytes and a head's amax is three
// shuffles. A warp takes up to 16 tokens of a few heads of one kind (q, k or v): the runs
// (adjacent tokens of one block) that start among its tokens, as many whole runs at a time as
// it holds, so single tokens of many requests and the blocks of a prompt take the same
// path. A head's elements stay in registers between the amax and the rounding, and the next
// head's loads are issued before that.
//
// Bound: HBM; 178 MB for 8256 tokens of 16 + 32 heads of 128 take 26.8 us at the copy rate, the
// kernel 40 us (4.4 TB/s), held back by the latency of its 12 warps per SM (168 registers: a
// head of 16 tokens as fp32 and the next one's loads; 16 warps, with more spills, took 46 us).
// Calls of one token per request are a chain of four dependent loads behind a launch: 2.9 us for
// one token, 3.7 us for 143, 4.4 us for 265.
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
  int tile;  // tokens whose runs one warp takes (at most 16)
  int per;   // heads of one warp
  int* error_flag;
};

constexpr int kStoreWarps = 4;
constexpr int kMostTokens = 16;  // tokens that a warp holds at once in large calls

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

// max(m, |a|, |b|), NaN if one of them is.
__device__ __forceinline__ float amax3(float m, float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
  return d;
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

// lanes of a token's head, and tokens side by side
template <int D>
constexpr int kHeadLanes = D == 96 ? 8 : D / 16;
template <int D>
constexpr int kAbreast = 32 / kHeadLanes<D>;

// J tokens a lane; CTAs per SM by their registers. One token a lane spills nothing, two (16 tokens
// of 64 dims) 12 bytes a thread, four (of 96 and 128 dims) 72 to 80.
template <int D, bool INT8, int J>
__global__ void __launch_bounds__(32 * kStoreWarps, J == 1 ? 5 : J == 2 ? 4 : 3)
    q8_store_kernel(Q8StoreParams p) {
  constexpr int GL = kHeadLanes<D>, GR = kAbreast<D>, kChunk = GR * J;
  const uint32_t all = 0xffffffffu;
  const int lane = threadIdx.x & 31, grp = lane / GL, c = lane % GL;
  const bool on = c < D / 16;

  // this warp's tokens and heads
  const uint32_t item = blockIdx.x * kStoreWarps + (threadIdx.x >> 5);
  const uint32_t kv_groups = (p.hkv + p.per - 1) / p.per, q_groups = (p.hq + p.per - 1) / p.per;
  const uint32_t groups = 2 * kv_groups + (p.q ? q_groups : 0);
  const int64_t t0 = static_cast<int64_t>(item / groups) * p.tile;
  if (t0 >= p.tokens) return;
  uint32_t part = item % groups;
  const int kind = part < kv_groups ? 1 : part < 2 * kv_groups ? 2 : 0;  // q, k, v
  part -= kind == 1 ? 0 : kind == 2 ? kv_groups : 2 * kv_groups;
  const int h0 = part * p.per, h1 = min(h0 + p.per, kind ? p.hkv : p.hq);
  const bf16* const src = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
  const int64_t stride = kind == 0 ? p.q_stride : kind == 1 ? p.k_stride : p.v_stride;
  const bool turns = kind != 2 && p.cos_sin;
  const int ahead = static_cast<int>(min(static_cast<int64_t>(32), p.tokens - t0));

  // a head's elements of the n tokens from `t` on: token GR * j + grp in raw[j], whose bit of
  // `has` says that it counts. Lanes without one load another's: no branch keeps the loads apart.
  uint4 raw[J][2];
  float x[J][16];
  int pos[J];
  uint32_t has;
  const int cc = on ? c : 0;
  auto fetch = [&](int64_t t, int n, int h) {
    const bf16* at = src + t * stride + static_cast<int64_t>(h) * D + 8 * cc;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const bf16* const row = at + min(j * GR + grp, n - 1) * stride;
      raw[j][0] = *reinterpret_cast<const uint4*>(row);
      raw[j][1] = *reinterpret_cast<const uint4*>(row + D / 2);
    }
  };
  auto fetch_positions = [&](int64_t t, int n) {
    if (!turns) return;
#pragma unroll
    for (int j = 0; j < J; ++j) pos[j] = p.positions[t + min(j * GR + grp, n - 1)];
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (pos[j] < 0 || pos[j] >= p.max_pos) {
        if (((has >> j) & 1) && p.error_flag) atomicOr(p.error_flag, LSB_DEVERR_POSITION);
        pos[j] = 0;
      }
  };
  auto turn = [&] {  // raw to x
#pragma unroll
    for (int j = 0; j < J; ++j) {
      unpack8(*reinterpret_cast<const bf16x8*>(&raw[j][0]), x[j]);
      unpack8(*reinterpret_cast<const bf16x8*>(&raw[j][1]), x[j] + 8);
    }
    if (turns) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        rotate8<D>(x[j], p.cos_sin + static_cast<int64_t>(pos[j]) * D, cc);
    }
  };
  auto largest = [&](int j) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) m = amax3(m, x[j][i], x[j][i + 1]);
    return (has >> j) & 1 ? __float_as_uint(m) : 0u;
  };

  if (kind == 0) {
    const int n = min(p.tile, ahead);
    has = 0;
#pragma unroll
    for (int j = 0; j < J; ++j) has |= static_cast<uint32_t>(on && j * GR + grp < n) << j;
    fetch(t0, n, h0);
    fetch_positions(t0, n);
    for (int h = h0; h < h1; ++h) {
      turn();
      if (h + 1 < h1) fetch(t0, n, h + 1);
      bf16* const dst = p.q_out + (t0 + grp) * p.q_out_stride + static_cast<int64_t>(h) * D + 8 * c;
#pragma unroll
      for (int j = 0; j < J; ++j)
        if ((has >> j) & 1) {
          const bf16x8 lo = pack8(x[j]), hi = pack8(x[j] + 8);
          bf16* const row = dst + j * GR * p.q_out_stride;
          *reinterpret_cast<uint4*>(row) = *reinterpret_cast<const uint4*>(&lo);
          *reinterpret_cast<uint4*>(row + D / 2) = *reinterpret_cast<const uint4*>(&hi);
        }
    }
    return;
  }

  uint8_t* const cache = kind == 1 ? p.k_cache : p.v_cache;
  float* const scales = kind == 1 ? p.k_scale : p.v_scale;
  // Lane l looks at token t0 - 1 + l: which tokens are stored, and which of them continue the
  // block of the one before.
  int64_t loc = 0;
  if ((lane > 0 || t0 > 0) && lane - 1 < ahead) loc = p.out_loc[t0 - 1 + lane];
  const bool ok = writable(p, loc);
  if (!ok && loc != 0 && lane > 0 && lane <= p.tile && p.error_flag)
    atomicOr(p.error_flag, LSB_DEVERR_SLOT);
  const int slot = ok ? static_cast<int>(loc) : 0, block = slot >> p.block_shift;
  const int prev_slot = __shfl_up_sync(all, slot, 1);
  const bool goes_on = ok && lane > 0 && prev_slot != 0 && p.block_shift > 0 &&
                       (prev_slot >> p.block_shift) == block;
  const uint32_t stored = __ballot_sync(all, ok), cont = __ballot_sync(all, goes_on);
  const uint32_t starts = stored & ~cont & ~1u;  // (a run that lane 0 starts is not this warp's)
  // does token t0 + 31 go on with lane 31's block?
  bool beyond = false;
  if ((stored >> 31) && p.block_shift > 0 && t0 + 31 < p.tokens) {
    const int64_t next = p.out_loc[t0 + 31];
    beyond = writable(p, next) &&
             (next >> p.block_shift) == (__shfl_sync(all, slot, 31) >> p.block_shift);
  }
  // bit e: the tokens before lane e end with a whole run
  const uint64_t ends = (static_cast<uint64_t>(!beyond) << 32) | static_cast<uint32_t>(~cont);

  // the earlier rows of a block, in a scale larger by 1 / ratio
  auto reexpress = [&](int64_t blk, int h, int first, float ratio) {
    if (!on) return;
    for (int r = grp; r < first; r += GR) {
      uint4* const row = reinterpret_cast<uint4*>(
          cache + ((blk << p.block_shift) + r) * p.slot_stride + h * D + 16 * c);
      uint4 w = *row;
      uint32_t* const ws = &w.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 f = q8_decode4f<INT8>(ws[i]);
        ws[i] = q8_encode4<INT8>(f.x * ratio, f.y * ratio, f.z * ratio, f.w * ratio);
      }
      *row = w;
    }
  };

  const uint32_t mine = (2u << p.tile) - 2;  // lanes 1 .. tile
  // the last whole run that starts there ends before lane `limit`
  const int limit = __ffsll(static_cast<long long>(ends >> (p.tile + 1)));
  const int stop = limit ? limit + p.tile : 33;
  for (uint32_t todo = starts & mine; todo;) {
    const int s = __ffs(todo) - 1;
    const int most = min(s + kChunk, stop);  // 33: no end in sight
    const uint64_t fit = ends & ((uint64_t(1) << (most + 1)) - 1) & ~((uint64_t(2) << s) - 1);
    if (fit) {
      // ---- whole runs, tokens of lanes s .. e - 1
      const int e = 63 - __clzll(static_cast<long long>(fit));
      const int64_t t = t0 - 1 + s;
      todo &= e >= 32 ? 0u : ~((1u << e) - 1);
      has = 0;
      int at[J];  // the slots of this lane's tokens
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int l = s + j * GR + grp;
        at[j] = __shfl_sync(all, slot, l & 31);
        has |= static_cast<uint32_t>(on && l < e && at[j] != 0) << j;
      }
      fetch(t, e - s, h0);
      // lane l has token l's run: where it starts, its block, the first slot that it writes
      const int l = s + min(lane, e - s - 1);
      const uint32_t before = starts & (l >= 31 ? all : (2u << l) - 1);
      const int run = 31 - __clz(before);
      const bool single =
          (before >> s) == 1 && 31 - __clz(starts & (e >= 32 ? all : (1u << e) - 1)) == s;
      const bool one_run = __all_sync(all, single);
      const int blk = __shfl_sync(all, block, run);
      int first = __shfl_sync(all, slot, l);
      first = first ? first - (blk << p.block_shift) : 1 << p.block_shift;
      // (the smallest of the run: its tokens need not be in the order of their slots)
      // the run's last token
      const int last = __ffsll(static_cast<long long>(ends >> (l + 1))) + l - s - 1;
      auto over_run = [&](uint32_t v, auto op) {
#pragma unroll
        for (int o = 1; o < kChunk; o <<= 1) {
          const uint32_t u = __shfl_up_sync(all, v, o);
          if (lane < kChunk && s + lane - o >= run) v = op(v, u);
        }
        return __shfl_sync(all, v, min(last, e - s - 1));
      };
      if (one_run)
        first = __reduce_min_sync(all, first);
      else if (p.block_shift > 0)
        first = over_run(first, [](uint32_t a, uint32_t b) { return min(a, b); });
      else
        first = 0;
      float* const scale = scales + static_cast<int64_t>(blk) * p.hkv;
      uint32_t old = first > 0 ? __float_as_uint(scale[h0]) & 0x7fffffffu : 0u;
      fetch_positions(t, e - s);
      for (int h = h0; h < h1; ++h) {
        turn();
        const uint32_t held = old;
        if (h + 1 < h1) {
          fetch(t, e - s, h + 1);
          old = first > 0 ? __float_as_uint(scale[h + 1]) & 0x7fffffffu : 0u;
        }
        uint32_t amax = 0;
        if (one_run) {
#pragma unroll
          for (int j = 0; j < J; ++j)
            amax = max(amax, largest(j));
          amax = __reduce_max_sync(all, amax);
        } else {
          uint32_t mx = 0;  // token l's to lane l
#pragma unroll
          for (int j = 0; j < J; ++j) {
            uint32_t m = largest(j);
#pragma unroll
            for (int o = 1; o < GL; o <<= 1) m = max(m, __shfl_xor_sync(all, m, o));
            m = __shfl_sync(all, m, (lane % GR) * GL);
            if (lane / GR == j) mx = m;
          }
          amax = p.block_shift == 0
                     ? mx
                     : over_run(mx, [](uint32_t a, uint32_t b) { return max(a, b); });
        }
        const uint32_t sb = max(held, q8_scale_bits<INT8>(amax));
        const float inv = q8_inverse(sb);
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const float f = one_run ? inv : __shfl_sync(all, inv, j * GR + grp);
          if ((has >> j) & 1)
            store_codes<D, INT8>(cache + static_cast<int64_t>(at[j]) * p.slot_stride + h * D, c,
                                 x[j], f);
        }
        // (a block begun here takes its scale even where that is 0: what is there was another's)
        const bool leads = lane < e - s && s + lane == run, grows = leads && sb > held;
        if (grows || (leads && first == 0)) scale[h] = __uint_as_float(sb);
        for (uint32_t more = __ballot_sync(all, grows && held != 0 && sb < kInfBits); more;
             more &= more - 1) {
          const int w = __ffs(more) - 1;
          const float ratio = __fdiv_rn(__uint_as_float(held), __uint_as_float(sb));
          reexpress(__shfl_sync(all, blk, w), h, __shfl_sync(all, first, w),
                    __shfl_sync(all, ratio, w));
        }
      }
    } else {
      // ---- one run of more tokens than that: its elements are read twice
      const int64_t t = t0 - 1 + s;
      const int64_t blk = __shfl_sync(all, block, s);
      int64_t n = 0;
      uint32_t first = ~0u;
      for (;;) {
        const int64_t tt = t + n + lane;
        const int64_t at = tt < p.tokens ? p.out_loc[tt] : 0;
        const bool same = writable(p, at) && (at >> p.block_shift) == blk;
        const uint32_t other = ~__ballot_sync(all, same);
        const int more = other ? __ffs(other) - 1 : 32;
        const uint32_t off = static_cast<uint32_t>(at - (blk << p.block_shift));
        first = min(first, __reduce_min_sync(all, lane < more ? off : ~0u));
        n += more;
        if (more < 32) break;
      }
      todo &= s + n >= 32 ? 0u : ~((1u << (s + n)) - 1);
      auto part_of = [&](int64_t base, int h) {
        has = 0;
#pragma unroll
        for (int j = 0; j < J; ++j)
          has |= static_cast<uint32_t>(on && base + j * GR + grp < n) << j;
        const int here = static_cast<int>(min(static_cast<int64_t>(kChunk), n - base));
        fetch(t + base, here, h);
        fetch_positions(t + base, here);
        turn();
      };
      for (int h = h0; h < h1; ++h) {
        float* const scale = scales + blk * p.hkv + h;
        const uint32_t held = first > 0 ? __float_as_uint(*scale) & 0x7fffffffu : 0u;
        uint32_t amax = 0;
        for (int64_t base = 0; base < n; base += kChunk) {
          part_of(base, h);
#pragma unroll
          for (int j = 0; j < J; ++j)
            amax = max(amax, largest(j));
        }
        amax = __reduce_max_sync(all, amax);
        const uint32_t sb = max(held, q8_scale_bits<INT8>(amax));
        const float inv = q8_inverse(sb);
        for (int64_t base = 0; base < n; base += kChunk) {
          part_of(base, h);
#pragma unroll
          for (int j = 0; j < J; ++j)
            if ((has >> j) & 1)
              store_codes<D, INT8>(
                  cache + static_cast<int64_t>(p.out_loc[t + base + j * GR + grp]) * p.slot_stride +
                      h * D,
                  c, x[j], inv);
        }
        if (lane == 0 && (sb > held || first == 0)) *scale = __uint_as_float(sb);
        if (sb > held && held != 0 && sb < kInfBits)
          reexpress(blk, h, first, __fdiv_rn(__uint_as_float(held), __uint_as_float(sb)));
      }
    }
  }
}

int launch_store(Q8StoreParams& p, int head_dim, int code, cudaStream_t stream,
                 const char* what) {
  // Few tokens: a warp per 4 of them (128 dims) and head, for the shortest way through. From 2^21
  // elements on 16 tokens, whose runs are then mostly whole blocks (16 + 32 heads of 128, blocks of
  // 16, 4 and 16 tokens a warp: 256 tokens 6.6 and 6.3 us, 400 tokens 7.9 and 6.7, 1600 tokens 16.7
  // and 10.7; 55 + 110 heads of 96: 64 tokens 6.4 and 6.3, 128 tokens 7.8 and 6.7; 8 + 16 heads of
  // 64: 1000 tokens 5.0 and 5.4, 1600 tokens 5.8 and 5.5; one-token blocks: 128 tokens 3.3 and 4.3,
  // 256 tokens 4.3 and 4.6, 400 tokens 5.4 and 4.8). When four heads a warp still
  // make 4736 warps, four heads, so that a head's loads run under the work on the one before: that
  // is the GPU full 2.7 times over at 128 and 96 dims (1776 warps at a time), twice at 64 (2368),
  // 1.6 times at 32 (2960). Measured at 128 dims (8256 tokens, 16 + 32 heads): 4 heads 40 us,
  // 1 head 56 us, 8 heads, 3100 warps, 56 us.
  const int64_t heads = 2 * p.hkv + (p.q ? p.hq : 0);
  auto warps_of = [&](int tile, int per) {
    const int64_t groups = 2 * ((p.hkv + per - 1) / per) + (p.q ? (p.hq + per - 1) / per : 0);
    return (p.tokens + tile - 1) / tile * groups;
  };
  const bool large = p.tokens * heads * head_dim >= int64_t(1) << 21;
  const int abreast = head_dim == 64 ? 8 : head_dim == 32 ? 16 : 4;
  p.tile = large ? kMostTokens : abreast;
  p.per = large && warps_of(kMostTokens, 4) >= 4736 ? 4 : 1;
  const int64_t blocks = (warps_of(p.tile, p.per) + kStoreWarps - 1) / kStoreWarps;
  LSB_REQUIRE(blocks < (int64_t(1) << 29), "%s: too many tokens", what);
  p.error_flag = lsb_device_error_flag();
  auto launch = [&](auto kernel) {
    kernel<<<static_cast<unsigned>(blocks), 32 * kStoreWarps, 0, stream>>>(p);
    return check_launch(what);
  };
#define LSB_Q8_STORE(DIM) \
  case DIM: \
    if (large) { \
      constexpr int kMost = kMostTokens / kAbreast<DIM>; \
      return code == LSB_Q8_INT8 ? launch(q8_store_kernel<DIM, true, kMost>) \
                                 : launch(q8_store_kernel<DIM, false, kMost>); \
    } \
    return code == LSB_Q8_INT8 ? launch(q8_store_kernel<DIM, true, 1>) \
                               : launch(q8_store_kernel<DIM, false, 1>);
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
  if (tokens <= 0) return LSB_OK;
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
  if (tokens <= 0) return LSB_OK;
  LSB_REQUIRE(k && v, "%s: null pointer", what);
  if (int rc = check_cache(what, k_cache, v_cache, slot_stride, num_slots, k_scale, v_scale,
                           block, code, out_loc, hkv, head_dim))
    return rc;
  LSB_REQUIRE(k_stride >= (int64_t)hkv * head_dim && v_stride >= (int64_t)hkv * head_dim &&
                  k_stride % 8 == 0 && v_stride % 8 == 0 && aligned(k, 16) && aligned(v, 16),
              "%s: k and v rows must be 16-byte aligned", what);
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
