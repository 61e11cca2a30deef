// Causal attention over the 8-bit paged KV cache (q8.cuh), one query row per work item: the
// decode form, and the general form of every call.
//
// Bound: HBM (two codes per key and dim). The work is the flat sequence of (head group, row,
// tile of 16 keys); every team of warps takes an equal contiguous share of it, whatever the
// rows' lengths, so all SMs end together and a row is cut only where a share ends. A team's
// warps hold one KV head each and walk the same keys, so a slot's heads are read together.
// Warps never wait for each other: each keeps its own ring of tiles in shared memory, filled
// by its own 16-byte cp.async copies (any page size, any head count; keys past the context
// or outside the pool are zero-filled and masked), and waits only for its own copy groups.
//
// Per tile: S = q . codes on the tensor cores with the KV head's query heads (up to 8) as the
// rows and f16 operands: codes are exact in f16, q is scaled by a power of two to stay exact
// too. The keys' scales multiply S in fp32. The softmax weight and the value scale go into the
// second product together, w = exp2(s - m) * v_scale, with the running maximum m taken over
// s + exponent(v_scale): the largest contribution has weight 1 to 2, so w fits f16 for any
// scales (its rounding, 2^-12 of each weight, is below the bf16 output's). The sum of
// exp2(s - m) stays in fp32. O^T = V^T w takes V as the left operand (16 dims x 16 keys), so
// the query heads fill its 8 columns and a lane ends with 16 neighbouring dims of one head.
// Which keys a lane's fragments hold is free (sums over keys commute); the order is chosen so
// that no shared-memory read has bank conflicts at 96 and 128 dims.
#include <cuda_fp16.h>

#include "q8.cuh"

namespace lsb {
namespace {

constexpr int kTile = 16;         // keys per tile
constexpr int kWarps = 16;        // per CTA, one CTA per SM
constexpr int kMaxRows = 2048;    // query rows per launch (their table is in shared memory)
constexpr int kMinShare = 4;      // tiles per team at least
constexpr float kNegBig = -1e30f;
constexpr float kLog2e = 1.4426950408889634f;

struct Q8AttentionParams {
  bf16* out;
  int64_t out_stride;
  const bf16* q;
  int64_t q_stride;
  const uint8_t *k, *v;
  int64_t slot_stride, num_slots;
  const float *ks, *vs;
  int block_shift;
  const int32_t* page_table;
  int64_t pt_stride;
  const int32_t *cache_seqlens, *cu_seqlens_q;
  int num_reqs;
  int64_t row0;  // first row of this launch
  int rows;      // its rows, at most kMaxRows
  int hq, hkv, group, chunks;  // query heads per KV head; chunks of 8 of them
  int page_size;
  int64_t max_seqlen;
  float scale_log2;
  int hg, nhg, teams_per_cta, stages;
  // workspace
  int64_t* share_out;  // tiles per team
  int32_t* prefix_out;  // [rows + 1] tiles before each row
  float* part_o;
  float* part_ml;
  int* error_flag;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

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

__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// D[16x8] += A[16x16] . B[16x8], f16 in, fp32 accumulate.
__device__ __forceinline__ void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The tile's key that column n of S's column tile j holds: lane (g, t) of the second product
// then needs keys t, 4 + (t+2)%4, 8 + t and 12 + (t+2)%4 (i = 0..3 below).
__device__ __forceinline__ int key_of(int j, int n) {
  return 8 * j + ((n & 1) ? 4 + (((n >> 1) + 2) & 3) : (n >> 1));
}
__device__ __forceinline__ int key_at(int t, int i) {
  return 8 * (i >> 1) + ((i & 1) ? 4 + ((t + 2) & 3) : t);
}
// Where a key's scale lies, so that lane t reads its four keys' as one float4.
__device__ __forceinline__ int scale_at(int key) {
  const int r = key & 3, odd = (key >> 2) & 1;
  return (odd ? ((r + 2) & 3) : r) * 4 + (key >> 3) * 2 + odd;
}

// Byte offset of 16-byte chunk c of row r in a K or V tile.
template <int D>
__device__ __forceinline__ int k_offset(int r, int c) {
  if (D == 128) return r * D + ((c ^ (((r >> 2) & 1) << 2)) << 4);
  if (D == 64) return (r ^ ((r >> 2) & 1)) * D + (c << 4);
  return r * D + (c << 4);
}
template <int D>
__device__ __forceinline__ int v_offset(int r, int c) {
  if (D == 128) return r * D + ((c ^ ((r & 3) << 1)) << 4);
  if (D == 64) return r * D + ((c ^ (((r >> 1) & 1) << 1)) << 4);
  return r * D + (c << 4);
}

template <int D>
__host__ __device__ constexpr int stage_bytes() {
  return 2 * kTile * D + 2 * kTile * 4 + 16;  // K, V, their scales, the mask of valid keys
}

struct Unit {  // a place in the sequence
  int hgroup, row, tile;
};

template <int D, bool INT8, int STAGES>
__global__ void __launch_bounds__(kWarps * 32, 1) q8_attention_kernel(Q8AttentionParams p) {
  constexpr int KSTEPS = D / 16;
  constexpr int W = D % 64 == 0 ? 16 : 8;  // bytes per K read of a lane
  constexpr int KREADS = D / (4 * W);
  constexpr int DPT = D / 8;               // dims per lane of the output
  constexpr int CHUNKS = D / 16;           // 16-byte chunks per row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_scan[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int32_t* const s_prefix = reinterpret_cast<int32_t*>(smem + kWarps * STAGES * stage_bytes<D>());
  int32_t* const s_len = s_prefix + p.rows + 1;
  int32_t* const s_req = s_len + p.rows;

  // ---- every row's request, keys and place in the sequence (the same in every CTA)
  constexpr int kPerThread = kMaxRows / (kWarps * 32);
  {
    int tiles[kPerThread], sum = 0;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      const int i = tid * kPerThread + j;
      tiles[j] = 0;
      if (i < p.rows) {
        const int64_t r = p.row0 + i;
        int req = -1;
        if (r < p.num_reqs && p.cu_seqlens_q[r] == r && p.cu_seqlens_q[r + 1] == r + 1) {
          req = static_cast<int>(r);
        } else if (r < p.cu_seqlens_q[p.num_reqs]) {
          int lo = 0, hi = p.num_reqs;  // cu[lo] <= r < cu[hi]
          while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.cu_seqlens_q[mid] <= r) lo = mid; else hi = mid;
          }
          req = lo;
        }
        int64_t len = -1;  // a row behind the last request: left as it is
        if (req >= 0) {
          int64_t kv = p.cache_seqlens[req];
          if (kv > p.max_seqlen) {
            if (p.error_flag) atomicOr(p.error_flag, LSB_DEVERR_SEQLEN);
            kv = p.max_seqlen;
          }
          const int64_t after = p.cu_seqlens_q[req + 1] - r - 1;  // the request's later rows
          len = kv - after;
          if (len < 0) len = 0;
        }
        s_len[i] = static_cast<int32_t>(len);
        s_req[i] = req;
        tiles[j] = len > 0 ? static_cast<int>((len + kTile - 1) / kTile) : 0;
        sum += tiles[j];
      }
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    int base = incl - sum;
    for (int w = 0; w < warp; ++w) base += s_scan[w];
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      const int i = tid * kPerThread + j;
      if (i <= p.rows) s_prefix[i] = base;
      base += tiles[j];
    }
    if (p.rows == kMaxRows && tid == kWarps * 32 - 1) s_prefix[kMaxRows] = base;
    __syncthreads();
  }
  const int row_tiles = s_prefix[p.rows];
  const int64_t total = static_cast<int64_t>(row_tiles) * p.nhg;
  const int teams = p.teams_per_cta * gridDim.x;
  int64_t share = (total + teams - 1) / teams;
  if (share < kMinShare) share = kMinShare;
  if (blockIdx.x == 0) {
    for (int i = tid; i <= p.rows; i += kWarps * 32) p.prefix_out[i] = s_prefix[i];
    if (tid == 0) *p.share_out = share;
  }
  for (int i = blockIdx.x; i < p.rows; i += gridDim.x)  // rows that see no key
    if (s_len[i] == 0)
      for (int e = tid; e < p.hq * D / 4; e += kWarps * 32)
        *reinterpret_cast<uint2*>(p.out + (p.row0 + i) * p.out_stride + 4 * e) = make_uint2(0, 0);

  // ---- this warp's share
  const int team_in_cta = warp / p.hg, wt = warp - team_in_cta * p.hg;
  if (team_in_cta >= p.teams_per_cta) return;
  // neighbouring shares go to different SMs first
  const int team = team_in_cta * gridDim.x + blockIdx.x;
  const int64_t u0 = team * share;
  int64_t count64 = total - u0;
  if (count64 > share) count64 = share;
  if (count64 <= 0) return;
  const int count = static_cast<int>(count64);

  Unit first;
  first.hgroup = static_cast<int>(u0 / row_tiles);
  {
    const int at = static_cast<int>(u0 - static_cast<int64_t>(first.hgroup) * row_tiles);
    int lo = 0, hi = p.rows;  // the row with prefix[row] <= at < prefix[row + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_prefix[mid] <= at) lo = mid; else hi = mid;
    }
    first.row = lo;
    first.tile = at - s_prefix[lo];
  }
  auto advance = [&](Unit& u) {
    if (++u.tile < s_prefix[u.row + 1] - s_prefix[u.row]) return;
    u.tile = 0;
    do {
      if (++u.row == p.rows) {
        u.row = 0;
        ++u.hgroup;
      }
    } while (s_prefix[u.row + 1] == s_prefix[u.row]);
  };

  uint8_t* const ring = smem + warp * STAGES * stage_bytes<D>();
  const uint32_t ring_addr = smem_addr(ring);
  const int vheads = p.hkv * p.chunks;
  const bool pow2 = (p.page_size & (p.page_size - 1)) == 0;
  const int pshift = __ffs(p.page_size) - 1;
  const int g = lane >> 2, t = lane & 3;

  // ---- producer: the page of this lane's key (lanes 16.. repeat 0..15) is fetched one tile
  // before its copies are issued
  Unit pu = first;
  int produced = 0;
  int page = 0;
  auto fetch_page = [&]() {  // for unit pu
    const int key = pu.tile * kTile + (lane & 15);
    if (produced < count && key < s_len[pu.row])
      page = p.page_table[s_req[pu.row] * p.pt_stride +
                          (pow2 ? (key >> pshift) : key / p.page_size)];
  };
  auto issue = [&](int stage) {  // unit pu's copies, then on to the next unit
    if (produced < count) {
      const int vh = pu.hgroup * p.hg + wt;
      if (vh < vheads) {
        const int kvh = vh / p.chunks;
        const int key = pu.tile * kTile + (lane & 15);
        const int off = pow2 ? (key & (p.page_size - 1)) : key % p.page_size;
        const int64_t slot64 = static_cast<int64_t>(page) * p.page_size + off;
        const bool in = key < s_len[pu.row];
        const bool valid = in && slot64 >= 0 && slot64 < p.num_slots;
        if (in && !valid && p.error_flag) atomicOr(p.error_flag, LSB_DEVERR_SLOT);
        const int slot = valid ? static_cast<int>(slot64) : 0;
        const uint32_t mask = __ballot_sync(0xffffffffu, valid) & 0xffffu;
        const uint32_t st = ring_addr + stage * stage_bytes<D>();
        const uint8_t* kb = p.k + kvh * D;
        const uint8_t* vb = p.v + kvh * D;
#pragma unroll
        for (int i = 0; i < (kTile * CHUNKS + 31) / 32; ++i) {
          const int idx = i * 32 + lane;
          const int r = idx / CHUNKS, c = idx - r * CHUNKS;
          const int s = __shfl_sync(0xffffffffu, slot, r);
          if (kTile * CHUNKS % 32 != 0 && r >= kTile) continue;
          const bool ok = (mask >> r) & 1;
          const int64_t o = s * p.slot_stride + (c << 4);
          copy16(st + k_offset<D>(r, c), kb + o, ok);
          copy16(st + kTile * D + v_offset<D>(r, c), vb + o, ok);
        }
        const float* sc = (lane < 16 ? p.ks : p.vs) +
                          static_cast<int64_t>(slot >> p.block_shift) * p.hkv + kvh;
        copy4(st + 2 * kTile * D + ((lane & 16) + scale_at(lane & 15)) * 4, sc, valid);
        if (lane == 0)
          *reinterpret_cast<uint32_t*>(ring + stage * stage_bytes<D>() + 2 * kTile * D +
                                       2 * kTile * 4) = mask;
      }
      ++produced;
      if (produced < count) advance(pu);
    }
    copy_commit();
  };

  fetch_page();
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    issue(s);
    fetch_page();
  }

  // ---- consumer
  uint32_t qf[KSTEPS][2];
  float acc[KSTEPS][4];
  float m = kNegBig, l = 0.f, qscale = 0.f;
  Unit u = first;
  int heads_here = 0;  // query heads of this warp's chunk
  int head0 = 0;
  bool from_start = false;
  for (int i = 0; i < count; ++i) {
    copy_wait<STAGES - 2>();
    __syncwarp();
    const int stage = i % STAGES;
    issue((i + STAGES - 1) % STAGES);
    fetch_page();
    const int vh = u.hgroup * p.hg + wt;
    const int ntiles = s_prefix[u.row + 1] - s_prefix[u.row];
    if (vh < vheads) {
      if (i == 0 || u.tile == 0) {  // a new row: its query heads, scaled to f16
        from_start = u.tile == 0;
        const int kvh = vh / p.chunks, chunk = vh - kvh * p.chunks;
        head0 = kvh * p.group + chunk * 8;
        heads_here = min(8, p.group - chunk * 8);
        m = kNegBig;
        l = 0.f;
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) acc[s][0] = acc[s][1] = acc[s][2] = acc[s][3] = 0.f;
        bf16x8 raw[KREADS][W / 8];
        uint32_t amax = 0;
        const bool real = g < heads_here;
        const bf16* qrow = p.q + (p.row0 + u.row) * p.q_stride +
                           static_cast<int64_t>(head0 + (real ? g : 0)) * D;
#pragma unroll
        for (int rd = 0; rd < KREADS; ++rd)
#pragma unroll
          for (int h = 0; h < W / 8; ++h) {
            *reinterpret_cast<uint4*>(&raw[rd][h]) =
                *reinterpret_cast<const uint4*>(qrow + (t + 4 * rd) * W + 8 * h);
            float f[8];
            unpack8(raw[rd][h], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(f[e]) & 0x7fffffffu);
          }
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // largest element to [2^7, 2^8): bf16's 8 bits stay exact down to 2^-22 of it
        int ex = static_cast<int>(amax >> 23);
        if (amax == 0 || amax >= kInfBits) ex = 127 + 7;
        ex = max(ex, 16);
        const float up = __uint_as_float(static_cast<uint32_t>(254 + 7 - ex) << 23);
        qscale = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(ex - 7) << 23);
        const float mul = real ? up : 0.f;
#pragma unroll
        for (int rd = 0; rd < KREADS; ++rd)
#pragma unroll
          for (int h = 0; h < W / 8; ++h) {
            float f[8];
            unpack8(raw[rd][h], f);
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const int s = rd * (W / 4) + 2 * h + w;
              qf[s][0] = real ? pack_f16(f[4 * w] * mul, f[4 * w + 1] * mul) : 0u;
              qf[s][1] = real ? pack_f16(f[4 * w + 2] * mul, f[4 * w + 3] * mul) : 0u;
            }
          }
      }
      const uint8_t* const st = ring + stage * stage_bytes<D>();
      // S = q . K codes
      float s[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
        const int r = key_of(j, g);
#pragma unroll
        for (int rd = 0; rd < KREADS; ++rd) {
          uint32_t w[W / 4];
          const int byte = (t + 4 * rd) * W;
          const uint8_t* src = st + k_offset<D>(r, byte >> 4) + (byte & 15);
          if (W == 16) {
            const uint4 x = *reinterpret_cast<const uint4*>(src);
            w[0] = x.x; w[1] = x.y; w[W / 4 - 2] = x.z; w[W / 4 - 1] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(src);
            w[0] = x.x; w[1] = x.y;
          }
#pragma unroll
          for (int e = 0; e < W / 4; ++e) {
            uint32_t b0, b1;
            q8_decode4<INT8>(w[e], b0, b1);
            const int ks = rd * (W / 4) + e;
            mma_f16(s[j], qf[ks][0], 0u, qf[ks][1], 0u, b0, b1);
          }
        }
      }
      const float4 ks4 = *reinterpret_cast<const float4*>(st + 2 * kTile * D + 16 * t);
      const float4 vs4 =
          *reinterpret_cast<const float4*>(st + 2 * kTile * D + kTile * 4 + 16 * t);
      const uint32_t mask =
          *reinterpret_cast<const uint32_t*>(st + 2 * kTile * D + 2 * kTile * 4);
      const float ksv[4] = {ks4.x, ks4.y, ks4.z, ks4.w};
      const float vsv[4] = {vs4.x, vs4.y, vs4.z, vs4.w};
      float x[4], top = m;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool live = (mask >> key_at(t, e)) & 1;
        x[e] = live ? s[e >> 1][e & 1] * (ksv[e] * qscale) : kNegBig;
        // the value scale's exponent, as fp32 (below 2^-100 a scale counts as 2^-100)
        const float ve = fmaxf(__uint_as_float(0x4b000000u | (__float_as_uint(vsv[e]) >> 23)) -
                                   (8388608.f + 127.f),
                               -100.f);
        top = fmaxf(top, live ? x[e] + ve : kNegBig);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (__any_sync(0xffffffffu, top > m)) {
        const float c = ex2(m - top);
        const float c0 = __shfl_sync(0xffffffffu, c, 8 * t);
        const float c1 = __shfl_sync(0xffffffffu, c, 8 * t + 4);
        l *= c;
#pragma unroll
        for (int e = 0; e < KSTEPS; ++e) {
          acc[e][0] *= c0;
          acc[e][1] *= c1;
          acc[e][2] *= c0;
          acc[e][3] *= c1;
        }
        m = top;
      }
      float wgt[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool live = (mask >> key_at(t, e)) & 1;
        const float pe = live ? ex2(x[e] - m) : 0.f;
        l += pe;
        wgt[e] = live ? pe * vsv[e] : 0.f;
      }
      const uint32_t b0 = pack_f16(wgt[0], wgt[1]), b1 = pack_f16(wgt[2], wgt[3]);
      // O^T += V^T w
      uint32_t vw[4][DPT / 4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint8_t* vt = st + kTile * D;
        const int r = key_at(t, e), byte = DPT * g;
        if (DPT == 16) {
          const uint4 y = *reinterpret_cast<const uint4*>(vt + v_offset<D>(r, g));
          vw[e][0] = y.x; vw[e][1 % (DPT / 4)] = y.y; vw[e][2 % (DPT / 4)] = y.z;
          vw[e][3 % (DPT / 4)] = y.w;
        } else if (DPT == 8) {
          const uint2 y =
              *reinterpret_cast<const uint2*>(vt + v_offset<D>(r, byte >> 4) + (byte & 15));
          vw[e][0] = y.x; vw[e][1 % (DPT / 4)] = y.y;
        } else {
#pragma unroll
          for (int w = 0; w < DPT / 4; ++w)
            vw[e][w] = *reinterpret_cast<const uint32_t*>(vt + r * D + byte + 4 * w);
        }
      }
#pragma unroll
      for (int w = 0; w < DPT / 4; ++w) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // dims 4w + 2h and 4w + 2h + 1 of the lane's DPT
          const uint32_t sel = h ? 0x7362 : 0x5140;
          uint32_t a0, a1, a2, a3;
          q8_decode4<INT8>(__byte_perm(vw[0][w], vw[1][w], sel), a0, a1);
          q8_decode4<INT8>(__byte_perm(vw[2][w], vw[3][w], sel), a2, a3);
          mma_f16(acc[2 * w + h], a0, a1, a2, a3, b0, b1);
        }
      }
      if (u.tile == ntiles - 1 || i == count - 1) {  // the row, or this team's part of it, ends
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const bool whole = from_start && u.tile == ntiles - 1;
        const int gm = min(8, p.group);
        const int64_t part =
            ((static_cast<int64_t>(team) * 2 + (from_start ? 1 : 0)) * p.hg + wt) * gm;
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int h = 2 * t + hh;
          const float lh = __shfl_sync(0xffffffffu, l, 8 * t + 4 * hh);
          const float mh = __shfl_sync(0xffffffffu, m, 8 * t + 4 * hh);
          if (h >= heads_here) continue;
          if (whole) {
            const float inv = lh == 0.f ? 0.f : 1.f / lh;
            bf16* dst = p.out + (p.row0 + u.row) * p.out_stride +
                        static_cast<int64_t>(head0 + h) * D + DPT * g;
#pragma unroll
            for (int w = 0; w < DPT / 4; ++w) {
              bf162 o2[2];
              o2[0] = __floats2bfloat162_rn(acc[2 * w][hh] * inv, acc[2 * w][2 + hh] * inv);
              o2[1] =
                  __floats2bfloat162_rn(acc[2 * w + 1][hh] * inv, acc[2 * w + 1][2 + hh] * inv);
              *reinterpret_cast<uint2*>(dst + 4 * w) = *reinterpret_cast<const uint2*>(o2);
            }
          } else {
            float* dst = p.part_o + (part + h) * D + DPT * g;
#pragma unroll
            for (int w = 0; w < DPT / 4; ++w)
              *reinterpret_cast<float4*>(dst + 4 * w) =
                  make_float4(acc[2 * w][hh], acc[2 * w][2 + hh], acc[2 * w + 1][hh],
                              acc[2 * w + 1][2 + hh]);
            if (g == 0)
              *reinterpret_cast<float2*>(p.part_ml + (part + h) * 2) = make_float2(mh, lh);
          }
        }
      }
    }
    if (i + 1 < count) advance(u);
  }
  copy_wait<0>();
}

// Rows cut between teams: their parts merged in team order, one warp per row and query head.
template <int D>
__global__ void __launch_bounds__(128) q8_attention_merge_kernel(Q8AttentionParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int row = static_cast<int>(item / p.hq);
  if (row >= p.rows) return;
  const int head = static_cast<int>(item - static_cast<int64_t>(row) * p.hq);
  const int32_t begin = p.prefix_out[row], end = p.prefix_out[row + 1];
  if (begin == end) return;
  const int64_t share = *p.share_out;
  const int kvh = head / p.group, hg_in = head - kvh * p.group;
  const int vh = kvh * p.chunks + (hg_in >> 3), h = hg_in & 7;
  const int hgroup = vh / p.hg, wt = vh - hgroup * p.hg;
  const int64_t base = static_cast<int64_t>(hgroup) * p.prefix_out[p.rows];
  const int c0 = static_cast<int>((base + begin) / share);
  const int c1 = static_cast<int>((base + end - 1) / share);
  if (c0 == c1) return;
  const int gm = min(8, p.group);
  auto index = [&](int c) -> int64_t {
    return ((static_cast<int64_t>(c) * 2 + (c == c0 ? 1 : 0)) * p.hg + wt) * gm + h;
  };
  float top = kNegBig;
  for (int c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, p.part_ml[index(c) * 2]);
  top = warp_max(top);
  float sum = 0.f, o[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) o[e] = 0.f;
  for (int c = c0; c <= c1; ++c) {
    const int64_t at = index(c);
    const float f = ex2(p.part_ml[at * 2] - top);
    sum += f * p.part_ml[at * 2 + 1];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) o[e] += f * p.part_o[at * D + e * 32 + lane];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  bf16* dst = p.out + (p.row0 + row) * p.out_stride + static_cast<int64_t>(head) * D;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) dst[e * 32 + lane] = __float2bfloat16_rn(o[e] * inv);
}

int sm_count() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return 148;
  }
  if (!cached[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      return 148;
    }
    cached[dev] = n;
  }
  return cached[dev];
}

// How the (KV head, chunk of 8 query heads) pairs are spread over warps.
struct TeamShape {
  int chunks, hg, nhg, teams_per_cta;
};

TeamShape team_shape(int hq, int hkv) {
  TeamShape s;
  const int group = hq / hkv;
  s.chunks = (group + 7) / 8;
  const int vheads = hkv * s.chunks;
  s.nhg = (vheads + kWarps - 1) / kWarps;
  s.hg = (vheads + s.nhg - 1) / s.nhg;
  s.teams_per_cta = kWarps / s.hg;
  return s;
}

int64_t parts_bytes(const TeamShape& s, int hq, int hkv, int d) {
  const int gm = hq / hkv < 8 ? hq / hkv : 8;
  return static_cast<int64_t>(sm_count()) * s.teams_per_cta * 2 * s.hg * gm * (d + 2) * 4;
}

constexpr int64_t kHeaderBytes = 16 + (kMaxRows + 4) * 4;  // the share, the rows' prefix

template <int D, bool INT8, int STAGES>
int launch_one(Q8AttentionParams& p, cudaStream_t stream) {
  auto kernel = q8_attention_kernel<D, INT8, STAGES>;
  const int smem = kWarps * STAGES * stage_bytes<D>() + (3 * p.rows + 1) * 4;
  LSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kWarps * STAGES * stage_bytes<D>() + (3 * kMaxRows + 1) * 4));
  const int ctas = sm_count();
  kernel<<<ctas, kWarps * 32, smem, stream>>>(p);
  if (int rc = check_launch("lsb_paged_attention_q8")) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((static_cast<int64_t>(p.rows) * p.hq + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  LSB_CUDA(cudaLaunchKernelEx(&cfg, q8_attention_merge_kernel<D>, p));
  return check_launch("lsb_paged_attention_q8 (merge)");
}

template <bool INT8>
int launch_dim(Q8AttentionParams& p, int head_dim, cudaStream_t stream) {
  switch (head_dim) {  // rings of about 200 KB per SM
    case 32: return launch_one<32, INT8, 8>(p, stream);
    case 64: return launch_one<64, INT8, 5>(p, stream);
    case 96: return launch_one<96, INT8, 3>(p, stream);
    case 128: return launch_one<128, INT8, 3>(p, stream);
  }
  return fail(LSB_ERR_UNSUPPORTED, "lsb_paged_attention_q8: head_dim %d", head_dim);
}

}  // namespace
}  // namespace lsb

using namespace lsb;

extern "C" int64_t lsb_paged_attention_q8_workspace_size(int64_t rows, int32_t hq, int32_t hkv,
                                                         int32_t head_dim) {
  if (rows <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || head_dim <= 0) return 0;
  return kHeaderBytes + parts_bytes(team_shape(hq, hkv), hq, hkv, head_dim);
}

extern "C" int lsb_paged_attention_q8(
    void* out, int64_t out_stride, const void* q, int64_t q_stride, const void* k_cache,
    const void* v_cache, int64_t slot_stride, int64_t num_slots, const float* k_scale,
    const float* v_scale, int32_t block, int32_t code, const int32_t* page_table,
    int64_t pt_stride, const int32_t* cache_seqlens, const int32_t* cu_seqlens_q,
    int64_t num_reqs, int64_t rows, int32_t hq, int32_t hkv, int32_t head_dim, int32_t page_size,
    int64_t max_seqlen, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "lsb_paged_attention_q8";
  LSB_REQUIRE(out && q && k_cache && v_cache && k_scale && v_scale && page_table &&
                  cache_seqlens && cu_seqlens_q,
              "%s: null pointer", what);
  LSB_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128,
              "%s: head_dim %d unsupported (32, 64, 96, 128)", what, head_dim);
  LSB_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0, "%s: bad heads %d/%d", what, hq, hkv);
  LSB_REQUIRE(code == LSB_Q8_E4M3 || code == LSB_Q8_INT8, "%s: unknown code type %d", what, code);
  LSB_REQUIRE(block >= 1 && block <= 128 && (block & (block - 1)) == 0,
              "%s: block of %d tokens (a power of two up to 128)", what, block);
  LSB_REQUIRE(page_size > 0 && page_size % block == 0,
              "%s: pages of %d tokens do not hold whole blocks of %d", what, page_size, block);
  LSB_REQUIRE(max_seqlen > 0 && max_seqlen < (int64_t(1) << 30) && num_reqs > 0 &&
                  num_reqs < (int64_t(1) << 30),
              "%s: bad sizes", what);
  LSB_REQUIRE(pt_stride > 0 && (max_seqlen + page_size - 1) / page_size <= pt_stride,
              "%s: max_seqlen %lld is beyond the page table's rows", what, (long long)max_seqlen);
  LSB_REQUIRE(num_slots > 0 && num_slots < (int64_t(1) << 31), "%s: bad slot count", what);
  LSB_REQUIRE(aligned(out, 16) && aligned(q, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) &&
                  aligned(k_scale, 4) && aligned(v_scale, 4),
              "%s: tensors must be 16-byte aligned", what);
  LSB_REQUIRE(q_stride % 8 == 0 && out_stride % 8 == 0 && slot_stride % 16 == 0,
              "%s: row strides must be multiples of 16 bytes", what);
  LSB_REQUIRE(q_stride >= (int64_t)hq * head_dim && out_stride >= (int64_t)hq * head_dim &&
                  slot_stride >= (int64_t)hkv * head_dim,
              "%s: strides too small", what);
  if (rows <= 0) return LSB_OK;
  const int64_t need = lsb_paged_attention_q8_workspace_size(rows, hq, hkv, head_dim);
  LSB_REQUIRE(workspace && workspace_bytes >= need && aligned(workspace, 16),
              "%s: workspace of %lld bytes needed", what, (long long)need);
  const TeamShape ts = team_shape(hq, hkv);
  Q8AttentionParams p{};
  p.out = static_cast<bf16*>(out);
  p.out_stride = out_stride;
  p.q = static_cast<const bf16*>(q);
  p.q_stride = q_stride;
  p.k = static_cast<const uint8_t*>(k_cache);
  p.v = static_cast<const uint8_t*>(v_cache);
  p.slot_stride = slot_stride;
  p.num_slots = num_slots;
  p.ks = k_scale;
  p.vs = v_scale;
  while ((1 << p.block_shift) < block) ++p.block_shift;
  p.page_table = page_table;
  p.pt_stride = pt_stride;
  p.cache_seqlens = cache_seqlens;
  p.cu_seqlens_q = cu_seqlens_q;
  p.num_reqs = static_cast<int>(num_reqs);
  p.hq = hq;
  p.hkv = hkv;
  p.group = hq / hkv;
  p.chunks = ts.chunks;
  p.page_size = page_size;
  p.max_seqlen = max_seqlen;
  p.scale_log2 = scale * kLog2e;
  p.hg = ts.hg;
  p.nhg = ts.nhg;
  p.teams_per_cta = ts.teams_per_cta;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.share_out = reinterpret_cast<int64_t*>(ws);
  p.prefix_out = reinterpret_cast<int32_t*>(ws + 16);
  p.part_o = reinterpret_cast<float*>(ws + kHeaderBytes);
  const int gm = p.group < 8 ? p.group : 8;
  p.part_ml = p.part_o +
              static_cast<int64_t>(sm_count()) * ts.teams_per_cta * 2 * ts.hg * gm * head_dim;
  p.error_flag = lsb_device_error_flag();
  // rows per launch: their table's size, and tile counts within 32 bits
  const int64_t tiles = (max_seqlen + kTile - 1) / kTile;
  int64_t per = ((int64_t(1) << 31) - 1) / tiles;
  if (per > kMaxRows) per = kMaxRows;
  for (int64_t r = 0; r < rows; r += per) {
    p.row0 = r;
    p.rows = static_cast<int>(rows - r < per ? rows - r : per);
    const int rc = code == LSB_Q8_INT8 ? launch_dim<true>(p, head_dim, as_stream(stream))
                                       : launch_dim<false>(p, head_dim, as_stream(stream));
    if (rc) return rc;
  }
  return LSB_OK;
}
