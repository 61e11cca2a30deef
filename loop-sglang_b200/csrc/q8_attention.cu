// Causal attention over the 8-bit paged KV cache (q8.cuh), one query row per work item: the
// decode form, and the general form of every call.
//
// Bound: HBM (two codes per key and dim). The work is the flat sequence of (row, tile of 32
// keys); every squad of warps takes an equal contiguous share of it, whatever the rows'
// lengths, so all SMs end together and a row is cut only where a share ends. A squad's warps
// hold one KV head each and walk the same keys at the same time, so a slot's heads are read
// together; a squad is one team of warps of a CTA, or as many as its heads need.
// A warp has a ring of tiles in shared memory to itself. A producer warp fills the rings of two
// of them with 16-byte cp.async copies (any page size, any head count; keys past the context
// or outside the pool are zero-filled and masked), so that working out addresses and issuing
// copies, 700 to 900 cycles a tile, is not in the way of the products (1100 cycles).
//
// What the copies leave time for is about 1400 instructions per tile and scheduler, so the
// products run on the tensor cores (m16n8k16 and k32), whose 8-bit float form is no gain here
// (it widens both operands again in every product):
//   S = codes . q with 16 keys as rows and the KV head's query heads (up to 8) as columns.
//   e4m3: the codes are widened to f16 (exact), q is scaled by a power of two to f16 (exact).
//   int8: the codes go in as they are; q is a 16-bit fixed-point number in two signed bytes
//   (off by 2^-16 of the head's largest element, so elements below 2^-8 of that keep fewer bits
//   than bf16's 8: what wide products of the codes as they are cost), one product for each, exact
//   in int32.
//   O^T = V^T w with 16 dims as rows: V's codes come transposed from shared memory and are
//   widened to f16; the weights are f16.
// The keys' scales multiply S in fp32. The softmax weight and the value scale go into the
// second product together, w = exp2(s - m) * v_scale, with the running maximum m taken over
// s + exponent(v_scale), one fp32 number: the largest contribution is 2^14 to 2^15 in f16, so
// weights keep their 11 bits down to 2^-28 of it for any scales. The sum of exp2(s - m) stays in
// fp32.
//
// Measured: 143 rows of 512 to 2304 keys, 16 heads of 128, e4m3: 133 us (0.96 of the copy rate);
// 265 rows over scattered one-token pages, int8: 177 us (0.88; a key's 64 bytes of scales are an
// access of their own); 55 heads of 96: 101 us (0.80: a tile has 3/4 of the bytes and 0.87 of the
// instructions of one of 128 dims, and waits twice as much for shared memory); 4 rows of 32 to 131
// thousand keys, 32 on 8 heads: 110 us (0.94); one row of 700 keys: 9.0 us, two launches and the
// loads of a few tiles in turn. More than 8 query heads to a KV head are read and widened once per
// 8: 64 rows of 2000 keys on 2 KV heads of 128 take 20 us with 16 heads, 27 with 32 (floor 10.1).
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "mbarrier.cuh"
#include "q8.cuh"
#include "q8_prefill.cuh"

namespace lsb {
namespace {

constexpr int kTile = 32;         // keys per tile
constexpr int kWarps = 8;         // consumer warps per CTA, one CTA per SM
constexpr int kFeeders = 4;       // producer warps, two consumers each
constexpr int kThreads = 32 * (kWarps + kFeeders);
constexpr int kMaxRows = 2048;    // query rows per launch (their table is in shared memory)
constexpr int kMinShare = 1;      // tiles per team at least
constexpr float kLow = -3.402823466e38f;  // no finite score is below
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kWeightBits = 14.f;  // weights are scaled by 2^14

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
  int hg, nhg, teams_per_cta, squads;
  // workspace
  int32_t* share_out;  // tiles per squad
  int32_t* prefix_out;  // [rows + 1] tiles before each row
  float* part_o;
  float* part_ml;
  int* error_flag;
};

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

// An arrival on `bar` once all earlier copies of this thread are in.
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
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

// D[16x8] += A[16x32] . B[32x8], int8 in, exact in int32.
__device__ __forceinline__ void mma_s8(int* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four 8-row x 16-byte matrices: lane (g, t) gets bytes 4t.. of row g of each.
__device__ __forceinline__ void load_rows(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 32 rows x 16 bytes, transposed: lane (g, t) gets column g (r[0]) and g + 8 (r[1]) of rows
// 4t.. 4t + 3, and the same of rows 16 + 4t.. (r[2], r[3]).
__device__ __forceinline__ void load_columns(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The 8 x 8 matrix of 16-bit elements whose row g lane (g, t) holds two of, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The row of the K tile that key k is stored at. Rows 8j + n are the rows of S that lanes
// (n, t) hold; transposed, lane (g, t) has the weights of rows 8j + 2t and 8j + 2t + 1. With
// key_of below those are keys 4t .. 4t + 3 (j = 0, 1) and 16 + 4t .. (j = 2, 3), the ones that
// a lane gets of a transposed V tile.
__device__ __forceinline__ int k_row(int k) {
  return (k & 16) | ((k & 2) << 2) | ((k >> 1) & 6) | (k & 1);
}
__device__ __forceinline__ int key_of(int j, int n) {
  return ((j & 2) << 3) | ((n & 6) << 1) | ((j & 1) << 1) | (n & 1);
}
// A key's scale lies at 4n + j, so that lane (n, t) reads its four as one float4.
__device__ __forceinline__ int scale_at(int k) {
  const int r = k_row(k);
  return ((r & 7) << 2) | (r >> 3);
}

// Chunk c's address in the row whose chunk 0 (at 96 dims: or any) is at row_addr.
template <int D>
__device__ __forceinline__ uint32_t chunk_of(uint32_t row_addr, int c) {
  return D == 96 ? row_addr + (c << 4) : row_addr ^ (c << 4);
}

template <int D>
__host__ __device__ constexpr int half_bytes() {  // the K or the V tile
  return kTile * q8_row_bytes<D>();
}
template <int D>
__host__ __device__ constexpr int stage_bytes() {
  // K, V, their scales, the mask of valid keys; whole 128-byte lines
  return (2 * half_bytes<D>() + 2 * kTile * 4 + 4 + 127) / 128 * 128;
}

// MHA: one query head per KV head (the odd columns of S are then never real).
template <int D, bool INT8, bool MHA, int STAGES>
__global__ void __launch_bounds__(kThreads, 1) q8_attention_kernel(Q8AttentionParams p) {
  constexpr int KSTEPS = D / 32;
  constexpr int COLS = MHA ? 1 : 2;  // query heads whose scores a lane holds
  constexpr int CHUNKS = D / 16;     // 16-byte chunks per row of codes
  constexpr int COPIES = kTile * CHUNKS / 32;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_scan[kThreads / 32];
  __shared__ __align__(8) uint64_t s_full[kWarps][STAGES], s_empty[kWarps][STAGES];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int32_t* const s_prefix = reinterpret_cast<int32_t*>(smem + kWarps * STAGES * stage_bytes<D>());
  int32_t* const s_len = s_prefix + p.rows + 1;
  int32_t* const s_req = s_len + p.rows;

  for (int i = tid; i < kWarps * STAGES; i += kThreads) {
    mbar_init(&s_full[0][0] + i, 33);  // the producer's lanes' copies, and its mask of keys
    mbar_init(&s_empty[0][0] + i, 1);
  }
  // The heads of consumer warp w: its team's of a squad, whose share of the tiles it walks.
  // Neighbouring shares go to different SMs first; a squad's teams are neighbours.
  struct Work {
    int squad, vh, kvh;
    bool idle;
  };
  const int vheads = p.hkv * p.chunks;
  auto work_of = [&](int w) {
    const int team_in_cta = w / p.hg;
    const int team = team_in_cta * gridDim.x + blockIdx.x;
    Work k;
    k.squad = team / p.nhg;
    k.vh = (team - k.squad * p.nhg) * p.hg + (w - team_in_cta * p.hg);
    k.kvh = k.vh / p.chunks;
    k.idle = team_in_cta >= p.teams_per_cta || k.squad >= p.squads || k.vh >= vheads;
    return k;
  };
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- every row's request, keys and place in the sequence (the same in every CTA)
  constexpr int kPerThread = (kMaxRows + kThreads - 1) / kThreads;
  const int per_thread = (p.rows + kThreads - 1) / kThreads;
  {
    int tiles[kPerThread], sum = 0;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      const int i = tid * per_thread + j;
      tiles[j] = 0;
      if (j < per_thread && i < p.rows) {
        const int64_t r = p.row0 + i;
        int req = -1;
        int64_t kv = 0, after = 0;  // the request's keys, its rows after this one
        // one row per request so far (decode): all that is needed in one round of loads
        const int64_t guess = r < p.num_reqs ? r : 0;
        const int at0 = p.cu_seqlens_q[guess], at1 = p.cu_seqlens_q[guess + 1];
        const int guessed = p.cache_seqlens[guess];
        if (guess == r && at0 == r && at1 == r + 1) {
          req = static_cast<int>(r);
          kv = guessed;
        } else if (r >= p.cu_seqlens_q[0] && r < p.cu_seqlens_q[p.num_reqs]) {
          int lo = 0, hi = p.num_reqs;  // cu[lo] <= r < cu[hi]
          while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.cu_seqlens_q[mid] <= r) lo = mid; else hi = mid;
          }
          req = lo;
          kv = p.cache_seqlens[req];
          after = max(p.cu_seqlens_q[req + 1] - r - 1, int64_t(0));
        }
        int64_t len = -1;  // a row of no request: left as it is
        if (req >= 0) {
          if (kv > p.max_seqlen) {
            if (p.error_flag) atomicOr(p.error_flag, LSB_DEVERR_SEQLEN);
            kv = p.max_seqlen;
          }
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
      const int i = tid * per_thread + j;
      if (j < per_thread && i < p.rows) {
        s_prefix[i] = base;
        base += tiles[j];
        if (i == p.rows - 1) s_prefix[p.rows] = base;
      }
    }
    __syncthreads();
  }
  allow_dependent_launch();  // the merge kernel's CTAs may wait beside this one
  const int row_tiles = s_prefix[p.rows];
  const int share = max((row_tiles + p.squads - 1) / p.squads, kMinShare);
  if (blockIdx.x == gridDim.x - 1) {  // (the CTA with the least to do)
    for (int i = tid; i <= p.rows; i += kThreads) p.prefix_out[i] = s_prefix[i];
    if (tid == 0) *p.share_out = share;
  }
  for (int i = blockIdx.x; i < p.rows; i += gridDim.x)  // rows that see no key
    if (s_len[i] == 0)
      for (int e = tid; e < p.hq * D / 4; e += kThreads)
        *reinterpret_cast<uint2*>(p.out + (p.row0 + i) * p.out_stride + 4 * e) = make_uint2(0, 0);

  // A place in the sequence: row, tile of the row. Rows without tiles are skipped.
  struct Place {
    int row, tile, tiles;
  };
  auto place_at = [&](int at) {
    int lo = 0, hi = p.rows;  // the row with prefix[row] <= at < prefix[row + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_prefix[mid] <= at) lo = mid; else hi = mid;
    }
    return Place{lo, at - s_prefix[lo], s_prefix[lo + 1] - s_prefix[lo]};
  };
  auto next_row = [&](Place& u) {
    u.tile = 0;
    do {
      ++u.row;
      u.tiles = s_prefix[u.row + 1] - s_prefix[u.row];
    } while (u.tiles == 0);
  };
  // a squad's share of the tiles
  auto share_of = [&](const Work& k) {
    const int64_t begin = static_cast<int64_t>(k.squad) * share;
    return k.idle || begin >= row_tiles ? 0 : min(share, row_tiles - static_cast<int>(begin));
  };

  if (warp >= kWarps) {
    // ---- producer of the rings of consumers w0 and w0 + 1: lane k has key k of the tile; its
    // page is fetched one tile before its copies are issued. Two heads of one team walk the
    // same tiles: their slots are worked out once.
    const int w0 = 2 * (warp - kWarps);
    const bool pow2 = (p.page_size & (p.page_size - 1)) == 0;
    const int pshift = __ffs(p.page_size) - 1;
    // copy i of a lane moves chunk copy_chunk / 16 of row copy_row(i) of both tiles (96 dims: six
    // chunks a row, so five lanes and a third share one: the chunk then differs by copy)
    const uint32_t stride = static_cast<uint32_t>(p.slot_stride), hkv = p.hkv;
    constexpr bool kEven = 32 % CHUNKS == 0;
    auto copy_row = [&](int i) { return (i * 32 + lane) / CHUNKS; };
    const uint32_t copy_chunk = kEven ? (lane % CHUNKS) << 4 : 0;
    uint32_t copy_k[COPIES], copy_v[COPIES];
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int r = copy_row(i), c = (i * 32 + lane) - r * CHUNKS;
      copy_k[i] = q8_tile_offset<D>(k_row(r), c);
      copy_v[i] = half_bytes<D>() + q8_tile_offset<D>(r, c);
    }
    struct Feed {
      Place at;
      int left, len, page;
      const int32_t* pages;
      int kvh;
    } feed[2];
    int stage = 0;  // both rings are filled in step: a tile each, or one of them is done
    uint32_t phase = 0;
    auto fetch_page = [&](Feed& f) {
      const int key = f.at.tile * kTile + lane;
      if (f.left > 0 && key < f.len)
        f.page = f.pages[pow2 ? (key >> pshift) : key / p.page_size];
    };
    auto enter_row = [&](Feed& f) {
      f.len = s_len[f.at.row];
      f.pages = p.page_table + s_req[f.at.row] * p.pt_stride;
    };
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const Work k = work_of(w0 + e);
      Feed& f = feed[e];
      f.left = share_of(k);
      f.kvh = k.kvh;
      f.page = 0;
      if (f.left > 0) {
        f.at = place_at(k.squad * share);
        enter_row(f);
        fetch_page(f);
      }
    }
    const bool paired = feed[0].left > 0 && feed[1].left > 0 &&
                        work_of(w0).squad == work_of(w0 + 1).squad;
    // the slot of this lane's key of f's tile (0 if there is none to read) and the mask of keys
    // that there are; then on to the next tile
    auto slot_of = [&](Feed& f, uint32_t& mask) {
      const int key = f.at.tile * kTile + lane;
      const int off = pow2 ? (key & (p.page_size - 1)) : key % p.page_size;
      const int64_t slot64 = static_cast<int64_t>(f.page) * p.page_size + off;
      const bool in = key < f.len;
      const bool valid = in && slot64 >= 0 && slot64 < p.num_slots;
      if (in && !valid && p.error_flag) atomicOr(p.error_flag, LSB_DEVERR_SLOT);
      mask = __ballot_sync(0xffffffffu, valid);
      if (--f.left > 0) {
        if (++f.at.tile == f.at.tiles) {
          next_row(f.at);
          enter_row(f);
        }
        fetch_page(f);
      }
      return valid ? static_cast<uint32_t>(slot64) : 0u;
    };
    // the tile of HEADS neighbouring KV heads from kvh on, into the rings of consumers w ..
    auto fill = [&](auto heads, int w, int kvh, int kvh_step, uint32_t slot, uint32_t mask) {
      constexpr int HEADS = decltype(heads)::value;
      uint32_t st[HEADS];
#pragma unroll
      for (int e = 0; e < HEADS; ++e) {
        if (!__all_sync(0xffffffffu,
                        mbar_wait(&s_empty[w + e][stage], phase ^ 1, p.error_flag)))
          return false;
        st[e] = smem_u32(smem + ((w + e) * STAGES + stage) * stage_bytes<D>());
      }
      const uint8_t* const kb = p.k + kvh * D + copy_chunk;
      const uint8_t* const vb = p.v + kvh * D + copy_chunk;
      const int step = kvh_step * D;
#pragma unroll
      for (int i = 0; i < COPIES; ++i) {
        const int r = copy_row(i);
        const uint64_t o = static_cast<uint64_t>(__shfl_sync(0xffffffffu, slot, r)) * stride +
                           (kEven ? 0 : (i * 32 + lane - r * CHUNKS) << 4);
        const bool ok = (mask >> r) & 1;
#pragma unroll
        for (int e = 0; e < HEADS; ++e) copy16(st[e] + copy_k[i], kb + o + e * step, ok);
#pragma unroll
        for (int e = 0; e < HEADS; ++e) copy16(st[e] + copy_v[i], vb + o + e * step, ok);
      }
      const uint64_t so = static_cast<uint64_t>(slot >> p.block_shift) * hkv + kvh;
      const uint32_t sd = 2 * half_bytes<D>() + 4 * scale_at(lane);
#pragma unroll
      for (int e = 0; e < HEADS; ++e) {
        copy4(st[e] + sd, p.ks + so + e * kvh_step, (mask >> lane) & 1);
        copy4(st[e] + sd + 4 * kTile, p.vs + so + e * kvh_step, (mask >> lane) & 1);
        copies_arrive(&s_full[w + e][stage]);
      }
      if (lane == 0) {
#pragma unroll
        for (int e = 0; e < HEADS; ++e) {
          *reinterpret_cast<uint32_t*>(smem + ((w + e) * STAGES + stage) * stage_bytes<D>() +
                                       2 * half_bytes<D>() + 2 * kTile * 4) = mask;
          mbar_arrive(&s_full[w + e][stage]);
        }
      }
      return true;
    };
    bool ok = true;
    while (ok && (feed[0].left > 0 || feed[1].left > 0)) {
      uint32_t mask;
      if (paired) {
        const uint32_t slot = slot_of(feed[0], mask);
        ok = fill(std::integral_constant<int, 2>{}, w0, feed[0].kvh, feed[1].kvh - feed[0].kvh,
                  slot, mask);
        feed[1].left = feed[0].left;
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (ok && feed[e].left > 0) {
            const uint32_t slot = slot_of(feed[e], mask);
            ok = fill(std::integral_constant<int, 1>{}, w0 + e, feed[e].kvh, 0, slot, mask);
          }
      }
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");  // no copy outlives the CTA, whoever gave up
    return;
  }

  // ---- consumer
  const Work work = work_of(warp);
  const int count = share_of(work);
  if (count == 0) return;
  const int g = lane >> 2, t = lane & 3;
  const int head0 = work.kvh * p.group + (work.vh - work.kvh * p.chunks) * 8;
  const int heads_here = min(8, (work.kvh + 1) * p.group - head0);  // query heads of this warp
  const uint8_t* const ring = smem + warp * STAGES * stage_bytes<D>();
  const uint32_t ring_addr = smem_u32(ring);
  // the query heads of a row, one row ahead: lane (g, t) has dims 16c + 4t .. of head g
  const bool real = g < heads_here;
  uint2 raw[CHUNKS];
  auto fetch_q = [&](int row) {
    const bf16* src =
        p.q + (p.row0 + row) * p.q_stride + static_cast<int64_t>(head0 + (real ? g : 0)) * D + 4 * t;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) raw[c] = *reinterpret_cast<const uint2*>(src + 16 * c);
  };
  Place u = place_at(work.squad * share);
  fetch_q(u.row);
  uint32_t qf[CHUNKS][2];  // of head g: f16 dims of chunk c, or the two bytes' dims
  float acc[CHUNKS][4];
  float m[COLS], l[COLS], qscale[COLS];  // of heads 2t and 2t + 1
  bool from_start = false;
  int stage = 0;
  uint32_t phase = 0;
  // K: rows 0-7, chunk 2s | rows 8-15, 2s | rows 0-7, 2s + 1 | rows 8-15, 2s + 1 per read
  const uint32_t k_lane = q8_tile_offset<D>(lane & 15, lane >> 4);
  const uint32_t k_lane2 = q8_tile_offset<D>(16 | (lane & 15), lane >> 4);
  const uint32_t v_lane = half_bytes<D>() + q8_tile_offset<D>(lane, 0);
  for (int i = 0; i < count; ++i) {
    if (i == 0 || u.tile == 0) {  // a new row: its query heads
      from_start = u.tile == 0;
#pragma unroll
      for (int s = 0; s < CHUNKS; ++s) acc[s][0] = acc[s][1] = acc[s][2] = acc[s][3] = 0.f;
      uint32_t amax = 0;
      auto wide = [&](const uint2& x, float* f) {
        const float2 a = __bfloat1622float2(*reinterpret_cast<const bf162*>(&x.x));
        const float2 b = __bfloat1622float2(*reinterpret_cast<const bf162*>(&x.y));
        f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
      };
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        float f[4];
        wide(raw[c], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) amax = max(amax, __float_as_uint(f[e]) & 0x7fffffffu);
      }
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      float up, down;
      if (INT8) {  // largest element to 32500
        const float a = fmaxf(__uint_as_float(amax), 1e-30f);
        up = __fdividef(32500.f, a);
        down = a * (1.f / 32500.f);
      } else {     // largest element to [2^7, 2^8): bf16's 8 bits stay exact to 2^-22 of it
        const int ex = amax == 0 ? 134 : max(static_cast<int>(amax >> 23), 16);
        up = __uint_as_float(static_cast<uint32_t>(254 + 7 - ex) << 23);
        down = __uint_as_float(static_cast<uint32_t>(ex - 7) << 23);
      }
      if (amax >= kInfBits) down = __uint_as_float(kNanBits);
      down *= p.scale_log2;
#pragma unroll
      for (int e = 0; e < COLS; ++e) {
        m[e] = kLow;
        l[e] = 0.f;
        qscale[e] = __shfl_sync(0xffffffffu, down, 8 * t + 4 * e);
      }
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        float f[4];
        wide(raw[c], f);
        uint32_t a, b;
        if (INT8) {
          int h[4], v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = __float2int_rn(f[e] * up);
            h[e] = (v[e] + 128) >> 8;
            v[e] -= h[e] * 256;
          }
          a = (h[0] & 0xff) | ((h[1] & 0xff) << 8) | ((h[2] & 0xff) << 16) | (h[3] << 24);
          b = (v[0] & 0xff) | ((v[1] & 0xff) << 8) | ((v[2] & 0xff) << 16) | (v[3] << 24);
        } else {
          a = pack_f16(f[0] * up, f[1] * up);
          b = pack_f16(f[2] * up, f[3] * up);
        }
        qf[c][0] = real ? a : 0u;
        qf[c][1] = real ? b : 0u;
      }
    }
    if (u.tile == u.tiles - 1 && i + 1 < count) {
      Place after = u;
      next_row(after);
      fetch_q(after.row);
    }
    if (!__all_sync(0xffffffffu, mbar_wait(&s_full[warp][stage], phase, p.error_flag))) return;
    const uint32_t st = ring_addr + stage * stage_bytes<D>();
    const uint8_t* const tail = ring + stage * stage_bytes<D>() + 2 * half_bytes<D>();
    const uint32_t mask = *reinterpret_cast<const uint32_t*>(tail + 2 * kTile * 4);
    float ks[4], vs[4], x[4][COLS];  // keys key_of(j, g)
    *reinterpret_cast<float4*>(ks) = *reinterpret_cast<const float4*>(tail + 16 * g);
    *reinterpret_cast<float4*>(vs) = *reinterpret_cast<const float4*>(tail + 128 + 16 * g);
    // S = K codes . q: rows 16 mt + g and 16 mt + 8 + g (keys key_of(2mt, g), (2mt + 1, g))
    if (INT8) {
      int hi[2][4], lo[2][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) hi[mt][e] = lo[mt][e] = 0;
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t k[4];
          load_rows(k, chunk_of<D>(st + (mt ? k_lane2 : k_lane), 2 * s));
          mma_s8(hi[mt], k, qf[2 * s][0], qf[2 * s + 1][0]);
          mma_s8(lo[mt], k, qf[2 * s][1], qf[2 * s + 1][1]);
        }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < COLS; ++e)
          x[j][e] = static_cast<float>(hi[j >> 1][(j & 1) * 2 + e] * 256 +
                                       lo[j >> 1][(j & 1) * 2 + e]);
    } else {
      float s0[2][4], s1[2][4];  // even and odd chunks apart: shorter chains of products
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s0[mt][e] = s1[mt][e] = 0.f;
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t k[4], a[8];
          load_rows(k, chunk_of<D>(st + (mt ? k_lane2 : k_lane), 2 * s));
#pragma unroll
          for (int e = 0; e < 4; ++e) q8_decode4<false>(k[e], a[2 * e], a[2 * e + 1]);
          mma_f16(s0[mt], a[0], a[2], a[1], a[3], qf[2 * s][0], qf[2 * s][1]);
          mma_f16(s1[mt], a[4], a[6], a[5], a[7], qf[2 * s + 1][0], qf[2 * s + 1][1]);
        }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < COLS; ++e)
          x[j][e] = s0[j >> 1][(j & 1) * 2 + e] + s1[j >> 1][(j & 1) * 2 + e];
    }
    uint32_t v[CHUNKS][4];  // V's fragments while the products run
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) load_columns(v[c], chunk_of<D>(st + v_lane, c));
    __syncwarp();
    if (lane == 0) mbar_arrive(&s_empty[warp][stage]);  // all of the tile is in registers
    float top[COLS];
#pragma unroll
    for (int e = 0; e < COLS; ++e) top[e] = m[e];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < COLS; ++e) x[j][e] *= ks[j] * qscale[e];
    if (mask != 0xffffffffu) {
      // keys past the context or outside the pool: nothing of them counts (their codes and
      // scales are zero-filled)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (!((mask >> key_of(j, g)) & 1))
#pragma unroll
          for (int e = 0; e < COLS; ++e) x[j][e] = -INFINITY;
    }
    float ve[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // the value scale's exponent, as fp32 (below 2^-100 a scale counts as 2^-100)
      ve[j] = fmaxf(__uint_as_float(0x4b000000u | (__float_as_uint(vs[j]) >> 23)) -
                        (8388608.f + 127.f),
                    -100.f);
#pragma unroll
      for (int e = 0; e < COLS; ++e) {
        x[j][e] += ve[j];
        top[e] = fmaxf(top[e], x[j][e]);
      }
    }
    bool grows = false;
#pragma unroll
    for (int e = 0; e < COLS; ++e) {
      top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 4));
      top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 8));
      top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 16));
      grows |= top[e] > m[e];
    }
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int e = 0; e < COLS; ++e) {
        const float f = ex2(m[e] - top[e]);
        l[e] *= f;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          acc[c][e] *= f;
          acc[c][2 + e] *= f;
        }
        m[e] = top[e];
      }
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float we[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < COLS; ++e) {
        // (in this order the weight stays below 2^15 however coarse the rounding of large scores)
        const float pe = ex2((x[j][e] - m[e]) + (kWeightBits - ve[j]));
        l[e] += pe;
        we[e] = pe * vs[j];
      }
      w[j] = transpose8(pack_f16(we[0], we[1]));
    }
    // O^T += V^T w: lane (g, t) has dims 16c + g (acc[c][0..1]) and 16c + 8 + g (acc[c][2..3])
    // of heads 2t and 2t + 1
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      uint32_t a[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) q8_decode4<INT8>(v[c][e], a[2 * e], a[2 * e + 1]);
      mma_f16(acc[c], a[0], a[2], a[1], a[3], w[0], w[1]);
      mma_f16(acc[c], a[4], a[6], a[5], a[7], w[2], w[3]);
    }
    if (u.tile == u.tiles - 1 || i == count - 1) {  // the row, or this team's part of it, ends
      const bool whole = from_start && u.tile == u.tiles - 1;
      const int gm = min(8, p.group);
      const int64_t part =
          ((static_cast<int64_t>(work.squad) * 2 + (from_start ? 1 : 0)) * vheads + work.vh) * gm;
      float inv[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < COLS; ++e) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 4);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 8);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 16);
        if (l[e] > 3e38f) l[e] = 3e38f;  // keys of a tiny value scale outweigh all others
        inv[e] = l[e] == 0.f ? 0.f : 1.f / l[e];
      }
      if (whole) {
        // even g stores dims g, g + 1 of head 2t, odd g those of head 2t + 1
        const int h = 2 * t + (g & 1);
        bf16* dst = p.out + (p.row0 + u.row) * p.out_stride +
                    static_cast<int64_t>(head0 + h) * D + (g & 6);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
          for (int up8 = 0; up8 < 2; ++up8) {
            const float a = acc[c][2 * up8] * inv[0], b = acc[c][2 * up8 + 1] * inv[1];
            const float got = __shfl_xor_sync(0xffffffffu, (g & 1) ? a : b, 4);
            const bf162 o2 = (g & 1) ? __floats2bfloat162_rn(got, b)
                                     : __floats2bfloat162_rn(a, got);
            if (h < heads_here) *reinterpret_cast<bf162*>(dst + 16 * c + 8 * up8) = o2;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < COLS; ++e) {
          const int h = 2 * t + e;
          if (h >= heads_here) continue;
          float* dst = p.part_o + (part + h) * D + g;
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) {
            dst[16 * c] = acc[c][e];
            dst[16 * c + 8] = acc[c][2 + e];
          }
          if (g == 0)
            *reinterpret_cast<float2*>(p.part_ml + (part + h) * 2) = make_float2(m[e], l[e]);
        }
      }
    }
    if (++stage == STAGES) {
      stage = 0;
      phase ^= 1;
    }
    if (i + 1 < count && ++u.tile == u.tiles) next_row(u);
  }
}

// Rows cut between squads: their parts merged in order. A warp takes a row and query head,
// or, with few rows (then of many parts), each of the CTA's four warps a quarter of its parts.
constexpr int kMergeWarps = 4;

template <int D, bool FEW_ROWS>
__global__ void __launch_bounds__(32 * kMergeWarps)
    q8_attention_merge_kernel(Q8AttentionParams p) {
  constexpr int STEP = FEW_ROWS ? kMergeWarps : 1;  // warps of one row and head
  __shared__ float s_o[STEP][D], s_ml[STEP][2];
  const int lane = threadIdx.x & 31, warp = FEW_ROWS ? threadIdx.x >> 5 : 0;
  const int item = FEW_ROWS ? blockIdx.x : blockIdx.x * kMergeWarps + (threadIdx.x >> 5);
  const int row = item / p.hq, head = item - row * p.hq;
  if (row >= p.rows) return;
  const int kvh = head / p.group, in_group = head - kvh * p.group;
  const int vh = kvh * p.chunks + (in_group >> 3), h = in_group & 7, vheads = p.hkv * p.chunks;
  const int gm = min(8, p.group);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int begin = p.prefix_out[row], end = p.prefix_out[row + 1], share = *p.share_out;
  if (begin == end) return;
  const int c0 = begin / share, c1 = (end - 1) / share;
  if (c0 == c1) return;
  auto index = [&](int c) -> int64_t {
    return ((static_cast<int64_t>(c) * 2 + (c == c0 ? 1 : 0)) * vheads + vh) * gm + h;
  };
  // this warp's parts c0 + warp, + STEP, ...: 32 at a time, a lane per part's maximum and
  // sum, then their outputs with eight loads in flight
  float top = kLow, sum = 0.f, o[D / 32];
#pragma unroll
  for (int e = 0; e < D / 32; ++e) o[e] = 0.f;
  for (int base = c0 + warp; base <= c1; base += 32 * STEP) {
    const int mine = base + lane * STEP;
    float2 ml = make_float2(kLow, 0.f);
    if (mine <= c1) ml = *reinterpret_cast<const float2*>(p.part_ml + index(mine) * 2);
    const float now = fmaxf(top, warp_max(ml.x)), f = ex2(ml.x - now), back = ex2(top - now);
    top = now;
    sum = sum * back + warp_sum(f * ml.y);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) o[e] *= back;
    const int n = min(32, (c1 - base) / STEP + 1);
    for (int k0 = 0; k0 < n; k0 += 8) {
      float part[8][D / 32];
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int e = 0; e < D / 32; ++e)
          part[k][e] = k0 + k < n
                           ? p.part_o[index(base + (k0 + k) * STEP) * D + e * 32 + lane]
                           : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, (k0 + k) & 31);
        if (k0 + k < n)
#pragma unroll
          for (int e = 0; e < D / 32; ++e) o[e] += fk * part[k][e];
      }
    }
  }
  if (!FEW_ROWS) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    bf16* dst = p.out + (p.row0 + row) * p.out_stride + static_cast<int64_t>(head) * D + lane;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) dst[e * 32] = __float2bfloat16_rn(o[e] * inv);
    return;
  }
  if (lane == 0) {
    s_ml[warp][0] = top;
    s_ml[warp][1] = sum;
  }
#pragma unroll
  for (int e = 0; e < D / 32; ++e) s_o[warp][e * 32 + lane] = o[e];
  __syncthreads();
  if (threadIdx.x >= D) return;
  float m = kLow;
#pragma unroll
  for (int w = 0; w < STEP; ++w) m = fmaxf(m, s_ml[w][0]);
  float all = 0.f, total = 0.f;
#pragma unroll
  for (int w = 0; w < STEP; ++w) {
    const float f = ex2(s_ml[w][0] - m);
    total += f * s_ml[w][1];
    all += f * s_o[w][threadIdx.x];
  }
  p.out[(p.row0 + row) * p.out_stride + static_cast<int64_t>(head) * D + threadIdx.x] =
      __float2bfloat16_rn(total == 0.f ? 0.f : all / total);
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

// The largest team (its heads are read together) that keeps the warps within a twentieth of
// as busy as the best one: 8 of 16 or 55 heads, 4 of 12, 1 of 5.
TeamShape team_shape(int hq, int hkv) {
  const int group = hq / hkv, chunks = (group + 7) / 8, vheads = hkv * chunks;
  auto shape = [&](int hg) {
    return TeamShape{chunks, hg, (vheads + hg - 1) / hg, kWarps / hg};
  };
  // warp slots that a walk over all heads takes, per head
  auto cost = [&](const TeamShape& s) {
    return static_cast<float>(s.nhg) * kWarps / (static_cast<float>(s.teams_per_cta) * vheads);
  };
  float least = 1e30f;
  for (int hg = 1; hg <= kWarps && hg <= vheads; ++hg) least = std::min(least, cost(shape(hg)));
  int hg = kWarps < vheads ? kWarps : vheads;
  while (cost(shape(hg)) > 1.05f * least) --hg;
  return shape(hg);
}

int64_t squads_of(const TeamShape& s) {
  const int64_t n = static_cast<int64_t>(sm_count()) * s.teams_per_cta / s.nhg;
  return n > 1 ? n : 1;
}

int64_t parts_bytes(const TeamShape& s, int hq, int hkv, int d) {
  const int gm = hq / hkv < 8 ? hq / hkv : 8;
  return squads_of(s) * 2 * hkv * s.chunks * gm * (d + 2) * 4;
}

constexpr int64_t kHeaderBytes = 16 + (kMaxRows + 4) * 4;  // the share, the rows' prefix

template <int D, bool INT8, bool MHA, int STAGES>
int launch_one(Q8AttentionParams& p, cudaStream_t stream) {
  auto kernel = q8_attention_kernel<D, INT8, MHA, STAGES>;
  const int smem = kWarps * STAGES * stage_bytes<D>() + (3 * p.rows + 1) * 4;
  static std::atomic<uint64_t> allowed{0};  // devices whose limit is raised already
  int dev = 0;
  LSB_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    LSB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  kWarps * STAGES * stage_bytes<D>() + (3 * kMaxRows + 1) * 4));
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  // one CTA per SM, more only where one squad's heads need them
  const int ctas = std::max(sm_count(), (p.nhg + p.teams_per_cta - 1) / p.teams_per_cta);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  // both kernels start under the end of the one before and wait for it
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  LSB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  if (int rc = check_launch("lsb_paged_attention_q8")) return rc;
  // a row has squads / rows parts and one or two more
  const bool few = p.rows * 8 <= p.squads;
  const unsigned items = static_cast<unsigned>(p.rows) * p.hq;
  cfg.gridDim = dim3(few ? items : (items + kMergeWarps - 1) / kMergeWarps);
  cfg.blockDim = dim3(32 * kMergeWarps);
  cfg.dynamicSmemBytes = 0;
  LSB_CUDA(cudaLaunchKernelEx(&cfg, few ? q8_attention_merge_kernel<D, true>
                                        : q8_attention_merge_kernel<D, false>, p));
  return check_launch("lsb_paged_attention_q8 (merge)");
}

template <bool INT8, bool MHA>
int launch_dim(Q8AttentionParams& p, int head_dim, cudaStream_t stream) {
  switch (head_dim) {  // rings of about 200 KB per SM
    case 32: return launch_one<32, INT8, MHA, 8>(p, stream);
    case 64: return launch_one<64, INT8, MHA, 5>(p, stream);
    case 96: return launch_one<96, INT8, MHA, 3>(p, stream);
    case 128: return launch_one<128, INT8, MHA, 3>(p, stream);
  }
  return fail(LSB_ERR_UNSUPPORTED, "lsb_paged_attention_q8: head_dim %d", head_dim);
}

// Which kernel takes a call of several rows per request. This one's time grows with the rows (it
// walks the keys once per row and KV head, all SMs together); the prompt kernel's with its CTAs of
// 256 packed rows, filled or not, of which 148 walk the keys at a time. Per key and at 128 dims
// one CTA of that kernel takes as long as 460 rows of this one (20 ns and 0.043 ns), more at
// fewer dims, where this one has less to read; groups of more than 8 heads cost it more than one
// pass. Measured, decode kernel and prompt kernel in us, 2000 keys a request: 16 KV heads of 128,
// 16 requests: 61 and 83 with 3 rows each, 76 and 83 with 4, 137 and 84 with 8; 100 requests: 358
// and 457 with 3, 474 and 457 with 4; 55 heads of 96, 16 requests: 226 and 219 with 4; 4 heads of
// 32, 100 requests: 66 and 113 with 4, 121 and 113 with 8; 8 heads on one of 128, 100 requests: 39
// and 48 with 4, 68 and 49 with 8; one request of 16000 keys, 16 heads: 142 and 273 with 16 rows,
// 271 and 273 with 32. Lengths are the device's alone, so the rule has none.
bool use_prefill(int64_t rows, int64_t num_reqs, int hkv, int group, int head_dim) {
  const int force = attention_forced_kernel();
  if (force) return force == 1;
  if (rows <= num_reqs) return false;
  const double ctas = static_cast<double>(hkv) *
                      std::max(static_cast<double>(num_reqs), static_cast<double>(rows) * group / 256);
  const double decode = static_cast<double>(rows) * hkv * std::max(16, 8 + group) / 16;
  return decode >= 5.0 * (220 - head_dim) * std::max(1.0, ctas / 148);
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
  LSB_REQUIRE(slot_stride < (int64_t(1) << 31), "%s: slot stride too large", what);
  LSB_REQUIRE(q_stride >= (int64_t)hq * head_dim && out_stride >= (int64_t)hq * head_dim &&
                  slot_stride >= (int64_t)hkv * head_dim,
              "%s: strides too small", what);
  if (rows <= 0) return LSB_OK;
  const int64_t need = lsb_paged_attention_q8_workspace_size(rows, hq, hkv, head_dim);
  LSB_REQUIRE(workspace && workspace_bytes >= need && aligned(workspace, 16),
              "%s: workspace of %lld bytes needed", what, (long long)need);
  if (use_prefill(rows, num_reqs, hkv, hq / hkv, head_dim)) {
    Q8PrefillParams pp{};
    pp.out = static_cast<bf16*>(out);
    pp.out_stride = out_stride;
    pp.q = static_cast<const bf16*>(q);
    pp.q_stride = q_stride;
    pp.k = static_cast<const uint8_t*>(k_cache);
    pp.v = static_cast<const uint8_t*>(v_cache);
    pp.slot_stride = slot_stride;
    pp.num_slots = num_slots;
    pp.ks = k_scale;
    pp.vs = v_scale;
    while ((1 << pp.block_shift) < block) ++pp.block_shift;
    pp.page_table = page_table;
    pp.pt_stride = pt_stride;
    pp.cache_seqlens = cache_seqlens;
    pp.cu_seqlens_q = cu_seqlens_q;
    pp.num_reqs = static_cast<int>(num_reqs);
    pp.rows = rows;
    pp.hkv = hkv;
    pp.group = hq / hkv;
    pp.page_size = page_size;
    pp.max_seqlen = max_seqlen;
    pp.scale_log2 = scale * kLog2e;
    pp.error_flag = lsb_device_error_flag();
    return launch_q8_prefill(pp, head_dim, code == LSB_Q8_INT8, as_stream(stream));
  }
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
  p.squads = static_cast<int>(squads_of(ts));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.share_out = reinterpret_cast<int32_t*>(ws);
  p.prefix_out = reinterpret_cast<int32_t*>(ws + 16);
  p.part_o = reinterpret_cast<float*>(ws + kHeaderBytes);
  const int gm = p.group < 8 ? p.group : 8;
  p.part_ml = p.part_o + squads_of(ts) * 2 * hkv * ts.chunks * gm * head_dim;
  p.error_flag = lsb_device_error_flag();
  // rows per launch: their table's size, and tile counts (rounded up to shares) within 32 bits
  const int64_t tiles = (max_seqlen + kTile - 1) / kTile;
  int64_t per = ((int64_t(1) << 31) - 1 - p.squads) / tiles;
  if (per > kMaxRows) per = kMaxRows;
  for (int64_t r = 0; r < rows; r += per) {
    p.row0 = r;
    p.rows = static_cast<int>(rows - r < per ? rows - r : per);
    auto* const run = code == LSB_Q8_INT8 ? (hq == hkv ? launch_dim<true, true> : launch_dim<true, false>)
                                          : (hq == hkv ? launch_dim<false, true> : launch_dim<false, false>);
    const int rc = run(p, head_dim, as_stream(stream));
    if (rc) return rc;
  }
  return LSB_OK;
}
