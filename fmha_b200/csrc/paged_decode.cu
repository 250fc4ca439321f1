// paged_decode.cu -- fmha_paged_decode: attention of one new token per
// sequence over a paged KV cache, split over the cache's length and joined.
//
// Mathematics. For one (sequence, kv head) the G = Hq/Hkv query heads share
// K and V. With s_j = scale*log2(e) * q.k_j, one pass over the keys keeps per
// query the running maximum m, l = sum 2^(s_j - m) and o = sum 2^(s_j - m) v_j
// (all fp32; o and l are scaled by 2^(m_old - m) when m rises). Two partial
// results join as m = max, l = sum l_i 2^(m_i - m), o alike. O = o / l.
//
// What bounds it: every cached byte is read once, 2*G flops per byte (16-bit
// cache), so HBM bandwidth. The contractions run on mma.sync (16x8x16): a
// query group is too short for a tcgen05 tile (64 rows at least), and the
// legacy tensor path needs a fifth of its rate to keep up with the reads.
//
// Precision: products are exact in the fp32 accumulators. P goes into the
// second MMA as two 16-bit parts (cut off, and what that left), so it keeps
// about 16 bits with bf16 and 22 with fp16, whose weights carry a factor of
// 2^15 to keep clear of its short exponent; for G <= 8 the second part rides
// in the MMA's idle rows 8..15, for larger groups it is a second MMA. e4m3
// codes convert exactly to fp16; a bf16 query then becomes fp16 after a shift
// by a power of two that puts its largest element just below 2^15.
//
// Split. A unit is one (sequence, kv head, up to 16 of its query heads); a
// tile is 16 of its tokens. All tiles of all units, one after the other, are
// dealt out to the CTAs in equal contiguous ranges whatever the lengths, so
// ragged batches and a single long sequence fill the card alike. Each CTA
// finds its range from a prefix sum over the lengths, which are only known on
// the device; a captured launch therefore stays right as sequences grow. A
// unit that crosses from one CTA into the next leaves partial results in the
// workspace (at most two per CTA), which a second small kernel joins. When
// the block table says that no unit can be longer than kWholeTiles tiles, CTAs
// take whole units and nothing is left to join.
//
// Inside a CTA the warps take tiles in turn. Each has its own ring of tiles
// in shared memory, filled by its own 16-byte cp.async (zero-filled behind
// the sequence's end, so that what lies in unused rows, NaN included, never
// meets the MMA), running on into the next unit while the current one is
// joined across the warps.
#include <cuda_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstring>

#include "../../include/fmha.h"
#include "decode_common.cuh"
#include "serving.hpp"
#include "serving_mma.cuh"

namespace fmha {
namespace {

constexpr int kTile = 16;          // tokens
constexpr int kMaxCtas = 160;      // parts the work is dealt into, at most
constexpr int kMaxRows = 16;       // query heads of a unit
constexpr int kWholeTiles = 32;    // units up to this length are not split
constexpr int kJoinThreads = 256;  // of the joining kernel

struct DecodeParams {
  const uint16_t* q;
  uint16_t* o;
  float* lse;  // or null
  fmha_paged_cache_t cache;
  int batch;
  int hkv;
  int g;       // query heads per kv head
  int rows;    // query heads of a unit (the last unit of a kv head may have fewer)
  int chunks;  // units per (sequence, kv head)
  int64_t q_stride, o_stride;
  float scale_log2;  // log2(e) * softmax_scale * k_scale
  int whole;         // CTAs take whole units
  int o_bf16;
  float shift;        // weight_shift of the kernel
  float* part_o;      // [ctas][2][rows][D]
  float2* part_ml;    // [ctas][2][rows]: (m, l)
  int2* part_unit;    // [ctas]: unit left for joining that starts here (or -1), its last CTA
  unsigned int* err;
};

// ------------------------------------------------------------ the work list

struct Place {  // a tile of a unit
  int b;        // sequence
  int hu;       // (kv head, chunk) of the sequence
  int tile;
};

__device__ __forceinline__ int tiles_of(const DecodeParams& P, int b) {
  const int n = P.cache.seqlens_kv[b];
  const int64_t most = (int64_t)P.cache.max_pages * P.cache.page_size;
  if (n < 0 || n > most) return 1;  // impossible: left out, and reported where it is met
  return n == 0 ? 1 : (n + kTile - 1) / kTile;  // an empty one still writes its zeros
}

// With the whole CTA: thread i takes a contiguous run of sequences, scan[i]
// becomes the tiles (of one unit each) before its run, and their total is
// returned.
template <int THREADS>
__device__ int64_t scan_lengths(const DecodeParams& P, int64_t* scan) {
  const int per = (P.batch + THREADS - 1) / THREADS;
  const int b0 = min(P.batch, (int)threadIdx.x * per), b1 = min(P.batch, b0 + per);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) mine += tiles_of(P, b);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inc = mine;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const int64_t y = __shfl_up_sync(kFullMask, inc, s);
    if (lane >= s) inc += y;
  }
  __shared__ int64_t warp_sum[THREADS / 32];
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  scan[threadIdx.x] = before + inc - mine;
  __syncthreads();
  return total;
}

// The thread whose run holds tile number `at` of the list of all tiles writes
// its place; a number past the list's end is the place behind it.
template <int THREADS>
__device__ void locate(const DecodeParams& P, const int64_t* scan, int64_t at, int64_t total,
                       Place* out) {
  const int hu = P.hkv * P.chunks;
  if (at >= total * hu) {
    if (threadIdx.x == 0) *out = {P.batch, 0, 0};
    return;
  }
  const int per = (P.batch + THREADS - 1) / THREADS;
  const int b0 = min(P.batch, (int)threadIdx.x * per), b1 = min(P.batch, b0 + per);
  int64_t base = scan[threadIdx.x] * hu;
  const int64_t next = (threadIdx.x + 1 < THREADS ? scan[threadIdx.x + 1] : total) * hu;
  if (at < base || at >= next) return;
  for (int b = b0; b < b1; ++b) {
    const int n = tiles_of(P, b);
    if (at < base + (int64_t)n * hu) {
      const int64_t r = at - base;
      *out = {b, (int)(r / n), (int)(r % n)};
      return;
    }
    base += (int64_t)n * hu;
  }
}

// ------------------------------------------------------------ the kernel

template <int D, bool F8>
struct DecodeShape {
  static constexpr int kElem = F8 ? 1 : 2;
  static constexpr int kRowBytes = D * kElem;
  static constexpr int kChunks = kRowBytes / 16;       // 16-byte pieces of a row
  static constexpr int kHalf = kTile * kRowBytes;      // K or V of a tile
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kWarps = D == 128 ? 8 : F8 ? 6 : 4;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kStages = D == 128 && F8 ? 6 : 3;
  static constexpr int kPad = D + 4;  // floats of a row of partial results
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kJoinO = kWarps * 8 * kPad * 4;
  static constexpr int kSmem = kRing + kJoinO;
  static_assert(kSmem <= 230400, "2 KB of a CTA's 227 KB are left to static arrays");
};

// log2 of the factor that weights carry: largest weight 2^15 in fp16.
template <bool BF16, bool F8>
__host__ __device__ constexpr float weight_shift() {
  return BF16 && !F8 ? 0.0f : 15.0f;
}

// Element offset of a token's row in the pages, or -1 where there is none.
__device__ __forceinline__ int64_t token_offset(const DecodeParams& P, int b, int token, int len) {
  if (token >= len) return -1;
  const int in_table = token / P.cache.page_size;
  const int page = P.cache.block_table[b * P.cache.table_stride + in_table];
  if (page < 0 || page >= P.cache.num_pages) {
    report_device_error(P.err, FMHA_ERR_INVALID_ARG, kSiteDecodePage);
    return -1;
  }
  return page * P.cache.page_stride +
         (int64_t)(token - in_table * P.cache.page_size) * P.cache.token_stride;
}

template <int D, bool BF16, bool F8, bool WIDE>
__global__ void __launch_bounds__((DecodeShape<D, F8>::kThreads), 1)
    paged_decode_kernel(const __grid_constant__ DecodeParams P) {
  using S = DecodeShape<D, F8>;
  constexpr bool kB = BF16 && !F8;  // type of the MMA's operands: e4m3 goes through fp16
  constexpr int kSteps = D / 16;    // MMA steps along head_dim
  constexpr float kShift = weight_shift<BF16, F8>();
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Place range[2];
  __shared__ float2 join_ml[S::kWarps][kMaxRows];
  __shared__ uint32_t tile_mask[S::kWarps][S::kStages];
  allow_dependent_launch();
  grid_dependency_wait();

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gr = lane >> 2, gc = lane & 3;
  const int HU = P.hkv * P.chunks;
  int64_t per = 0;  // tiles of a CTA

  // This CTA's range of tiles, [range[0], range[1]).
  if (P.whole) {
    if (threadIdx.x < 2) {
      const int64_t u = (int64_t)P.batch * HU * (blockIdx.x + threadIdx.x) / gridDim.x;
      range[threadIdx.x] = {(int)(u / HU), (int)(u % HU), 0};
    }
  } else {
    int64_t* const scan = reinterpret_cast<int64_t*>(smem);  // before the ring is in use
    const int64_t total = scan_lengths<S::kThreads>(P, scan);
    per = (total * HU + gridDim.x - 1) / gridDim.x;
    if (per < S::kWarps) per = S::kWarps;
    locate<S::kThreads>(P, scan, per * blockIdx.x, total, &range[0]);
    locate<S::kThreads>(P, scan, per * (blockIdx.x + 1), total, &range[1]);
    if (threadIdx.x == 0) P.part_unit[blockIdx.x] = make_int2(-1, 0);
  }
  __syncthreads();
  const Place from = range[0], to = range[1];

  // The loader: walks this warp's tiles, kStages - 1 ahead of the arithmetic.
  const uint32_t ring = smem_u32(smem) + warp * S::kStages * S::kStage;
  Place next = from;  // unit the loader is in; its tiles from next.tile on
  int next_len = 0, next_end = 0;
  int next_tile = 0;  // its tile, relative to the start of the CTA's part of the unit
  auto enter = [&](const Place& p, int& len, int& end) {  // length and last tile in this CTA
    len = 0;
    end = 0;
    if (p.b < P.batch && (p.b < to.b || p.hu < to.hu || (p.hu == to.hu && p.tile < to.tile))) {
      const int n = P.cache.seqlens_kv[p.b];
      const int64_t most = (int64_t)P.cache.max_pages * P.cache.page_size;
      len = n >= 0 && n <= most ? n : -1;
      end = len > 0 ? (len + kTile - 1) / kTile : 1;
      if (p.b == to.b && p.hu == to.hu && to.tile < end) end = to.tile;
    }
  };
  auto past = [&](Place& p) {  // on to the next unit
    p.tile = 0;
    if (++p.hu == HU) {
      p.hu = 0;
      ++p.b;
    }
  };
  auto beyond = [&](const Place& p) {
    return p.b > to.b || (p.b == to.b && (p.hu > to.hu || (p.hu == to.hu && p.tile >= to.tile))) ||
           p.b >= P.batch;
  };
  enter(next, next_len, next_end);
  next_tile = next.tile + warp;
  auto settle = [&]() {  // to the unit that holds the loader's tile
    while (!beyond(next) && next_tile >= next_end) {
      next_tile -= next_end;
      past(next);
      enter(next, next_len, next_end);
    }
  };
  settle();
  int64_t next_off = -1;  // lane < 16: token offset of the loader's tile
  auto look_up = [&]() {
    next_off = -1;
    if (!beyond(next) && lane < kTile)
      next_off = token_offset(P, next.b, next_tile * kTile + lane, next_len);
  };
  look_up();
  int load_slot = 0;
  auto load = [&]() {
    if (!beyond(next)) {
      const uint32_t ok = __ballot_sync(kFullMask, next_off >= 0) & 0xffffu;
      if (lane == 0) tile_mask[warp][load_slot] = ok;
      const uint32_t base = ring + load_slot * S::kStage;
      const int64_t head = (next.hu / P.chunks) * P.cache.head_stride;
      const uint8_t* const kb = static_cast<const uint8_t*>(P.cache.k) + head * S::kElem;
      const uint8_t* const vb = static_cast<const uint8_t*>(P.cache.v) + head * S::kElem;
      constexpr int kRowsPer = 32 / S::kChunks;  // rows one warp-wide copy covers
#pragma unroll
      for (int i = 0; i < kTile / kRowsPer; ++i) {
        const int r = i * kRowsPer + lane / S::kChunks, ch = lane % S::kChunks;
        const int64_t off = __shfl_sync(kFullMask, next_off, r);
        const int64_t src = (off < 0 ? 0 : off) * S::kElem + ch * 16;
        const uint32_t dst = base + r * S::kRowBytes + ((ch ^ (r & 7)) << 4);
        cp_async16(dst, kb + src, off < 0 ? 0 : 16);
        cp_async16(dst + S::kHalf, vb + src, off < 0 ? 0 : 16);
      }
      next_tile += S::kWarps;
      settle();
      look_up();
    }
    cp_async_commit();
    load_slot = load_slot + 1 == S::kStages ? 0 : load_slot + 1;
  };
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) load();

  int slot = 0;
  int turn = 0;  // tiles of this CTA before the current unit's, modulo the warps
  for (Place p = from; !beyond(p); past(p)) {
    int len, end;
    enter(p, len, end);
    const int first = p.tile;
    const int tiles = end - first;
    const int kvh = p.hu / P.chunks, head0 = kvh * P.g + (p.hu % P.chunks) * P.rows;
    const int rows = min(P.rows, P.g - (p.hu % P.chunks) * P.rows);
    const bool bad = len < 0;
    if (bad && threadIdx.x == 0)
      report_device_error(P.err, FMHA_ERR_INVALID_ARG, kSiteDecodeLength);
    int mine = warp - turn;  // this warp's first tile here
    if (mine < 0) mine += S::kWarps;
    turn = (turn + tiles) % S::kWarps;

    // Query fragments: row gr (and gr + 8). Element order along head_dim is
    // the one K's fragments come in: natural for 16-bit rows, and for e4m3
    // rows 4c..4c+3 of each 16 (two to each half of the MMA's 16).
    uint32_t qa[kSteps][WIDE ? 4 : 2];
    float qs[WIDE ? 2 : 1];  // per-row factor of the scores
#pragma unroll
    for (int half = 0; half < (WIDE ? 2 : 1); ++half) {
      const int row = gr + 8 * half;
      const bool have = row < rows;
      const uint16_t* const src =
          P.q + p.b * P.q_stride + (int64_t)(head0 + (have ? row : 0)) * D;
      qs[half] = P.scale_log2;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        uint32_t w0 = 0, w1 = 0;
        if (have && mine < tiles) {
          if constexpr (F8) {
            const uint2 w = *reinterpret_cast<const uint2*>(src + 16 * s + 4 * gc);
            w0 = w.x;
            w1 = w.y;
          } else {
            w0 = *reinterpret_cast<const uint32_t*>(src + 16 * s + 2 * gc);
            w1 = *reinterpret_cast<const uint32_t*>(src + 16 * s + 2 * gc + 8);
          }
        }
        qa[s][half] = w0;
        qa[s][(WIDE ? 2 : 1) + half] = w1;
      }
      if constexpr (F8 && BF16) {
        // bf16 -> fp16: the row times 2^e, e such that its largest element
        // lies in [2^14, 2^15); the scores take 2^-e back. Elements 2^-29
        // below the largest and smaller lose bits: less than an fp32 sum does.
        // A row with infinity or NaN keeps e = 0 and stays what it is.
        float top = 0.0f;
        bool odd = false;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 f = unpack2<true>(qa[s][j * (WIDE ? 2 : 1) + half]);
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
            odd |= !(fabsf(f.x) <= FLT_MAX) || !(fabsf(f.y) <= FLT_MAX);
          }
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
        odd |= __shfl_xor_sync(kFullMask, (int)odd, 1) != 0;
        odd |= __shfl_xor_sync(kFullMask, (int)odd, 2) != 0;
        // Exponents beyond +-100 would leave fp32's range of scale factors.
        int e = odd || top == 0.0f ? 0 : 14 - ilogbf(top);
        e = max(-100, min(100, e));
        const float up = exp2f((float)e);
        qs[half] = P.scale_log2 * exp2f((float)-e);
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t& w = qa[s][j * (WIDE ? 2 : 1) + half];
            const float2 f = unpack2<true>(w);
            w = pack2<false>(f.x * up, f.y * up);
          }
      }
    }

    float acc[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
    float m[WIDE ? 2 : 1], l[WIDE ? 2 : 1];
#pragma unroll
    for (int h = 0; h < (WIDE ? 2 : 1); ++h) {
      m[h] = -INFINITY;
      l[h] = 0.0f;
    }

    for (int t = mine; t < tiles; t += S::kWarps) {
      cp_async_wait<S::kStages - 2>();
      __syncwarp();
      load();  // into the slot of the tile before this one
      const uint32_t kt = ring + slot * S::kStage, vt = kt + S::kHalf;
      const uint32_t ok = tile_mask[warp][slot];
      slot = slot + 1 == S::kStages ? 0 : slot + 1;

      // Scores of 16 tokens: two 8-token column tiles.
      float sc[2][4] = {};
      if constexpr (F8) {
        // One ldmatrix.x4: 16 tokens x 32 bytes; each lane gets 4 adjacent
        // codes of its token per 16 bytes.
#pragma unroll
        for (int s = 0; s < kSteps; s += 2) {
          const int r = (lane & 7) + ((lane >> 4) << 3), ch = s + ((lane >> 3) & 1);
          uint32_t w[4];
          ldsm4(w, kt + r * S::kRowBytes + ((ch ^ (r & 7)) << 4));
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t x = w[2 * n + j];
              const uint32_t b0 = e4m3x2_to_half2(x & 0xffffu), b1 = e4m3x2_to_half2(x >> 16);
              if constexpr (WIDE)
                mma16<kB>(sc[n], qa[s + j][0], qa[s + j][1], qa[s + j][2], qa[s + j][3], b0, b1);
              else
                mma16<kB>(sc[n], qa[s + j][0], 0u, qa[s + j][1], 0u, b0, b1);
            }
        }
      } else {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const int r = (lane & 7) + ((lane >> 4) << 3), ch = 2 * s + ((lane >> 3) & 1);
          uint32_t w[4];
          ldsm4(w, kt + r * S::kRowBytes + ((ch ^ (r & 7)) << 4));
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            if constexpr (WIDE)
              mma16<kB>(sc[n], qa[s][0], qa[s][1], qa[s][2], qa[s][3], w[2 * n], w[2 * n + 1]);
            else
              mma16<kB>(sc[n], qa[s][0], 0u, qa[s][1], 0u, w[2 * n], w[2 * n + 1]);
          }
        }
      }

      // Running maximum, and P as two 16-bit parts in A-fragment order.
      uint32_t hi[2][2], lo[2][2];  // [row half][column tile]
      float down[WIDE ? 2 : 1];
      bool rose = false;
#pragma unroll
      for (int h = 0; h < (WIDE ? 2 : 1); ++h) {
        float s4[4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            s4[2 * n + j] = (ok >> (8 * n + 2 * gc + j)) & 1u ? sc[n][2 * h + j] * qs[h] : -INFINITY;
        float top = fmaxf(fmaxf(s4[0], s4[1]), fmaxf(s4[2], s4[3]));
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
        top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
        const float now = fmaxf(m[h], top);
        const float ref = now == -INFINITY ? 0.0f : now;  // nothing seen yet: weights 2^-inf = 0
        down[h] = exp2f(m[h] - ref);
        rose |= now != m[h];
        m[h] = now;
        float pr[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) pr[j] = exp2f(s4[j] - (ref - kShift));
        l[h] = l[h] * down[h] + ((pr[0] + pr[1]) + (pr[2] + pr[3]));
        split2<kB>(pr[0], pr[1], hi[h][0], lo[h][0]);
        split2<kB>(pr[2], pr[3], hi[h][1], lo[h][1]);
      }
      if (__any_sync(kFullMask, rose)) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          acc[i][0] *= down[0];
          acc[i][1] *= down[0];
          acc[i][2] *= down[WIDE ? 1 : 0];
          acc[i][3] *= down[WIDE ? 1 : 0];
        }
      }

      // P.V: one ldmatrix.x4.trans covers 16 tokens x 32 bytes of head_dim.
#pragma unroll
      for (int i = 0; i < S::kChunks; i += 2) {
        const int r = (lane & 7) + (((lane >> 3) & 1) << 3), ch = i + (lane >> 4);
        uint32_t w[4];
        ldsm4_trans(w, vt + r * S::kRowBytes + ((ch ^ (r & 7)) << 4));
        auto pv = [&](float (&a)[4], uint32_t b0, uint32_t b1) {
          if constexpr (WIDE) {
            mma16<kB>(a, hi[0][0], hi[1][0], hi[0][1], hi[1][1], b0, b1);
            mma16<kB>(a, lo[0][0], lo[1][0], lo[0][1], lo[1][1], b0, b1);
          } else {
            mma16<kB>(a, hi[0][0], lo[0][0], hi[0][1], lo[0][1], b0, b1);
          }
        };
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if constexpr (F8) {
            // Each 32-bit word: two tokens x two adjacent columns; tile 2k
            // takes the even columns of a 16-byte piece, tile 2k+1 the odd.
            const uint32_t x = w[2 * j], y = w[2 * j + 1];
            pv(acc[2 * (i + j)], e4m3x2_to_half2(__byte_perm(x, 0, 0x4420)),
               e4m3x2_to_half2(__byte_perm(y, 0, 0x4420)));
            pv(acc[2 * (i + j) + 1], e4m3x2_to_half2(__byte_perm(x, 0, 0x4431)),
               e4m3x2_to_half2(__byte_perm(y, 0, 0x4431)));
          } else {
            pv(acc[i + j], w[2 * j], w[2 * j + 1]);
          }
        }
      }
    }

    // Join across the warps. Rows 8..15 of a narrow group hold the low parts.
#pragma unroll
    for (int h = 0; h < (WIDE ? 2 : 1); ++h) {
      l[h] += __shfl_xor_sync(kFullMask, l[h], 1);
      l[h] += __shfl_xor_sync(kFullMask, l[h], 2);
      if (gc == 0) join_ml[warp][gr + 8 * h] = make_float2(m[h], l[h]);
    }
    const bool starts = first == 0;
    const bool ends = P.whole || bad || end == (len > 0 ? (len + kTile - 1) / kTile : 1);
    const int part = starts ? 1 : 0;  // a unit that began earlier lies in part 0
    if (!(starts && ends) && threadIdx.x == 0 && starts) {
      // The CTA that holds the unit's last tile, from the even deal.
      const int n = (len + kTile - 1) / kTile;
      const int64_t here = per * (blockIdx.x + 1);  // tile number of this CTA's end
      const int64_t last = here + (n - end) - 1;
      P.part_unit[blockIdx.x] = make_int2(p.b * HU + p.hu, (int)(last / per));
    }
    float* const jo = reinterpret_cast<float*>(smem + S::kRing);
#pragma unroll
    for (int h = 0; h < (WIDE ? 2 : 1); ++h) {
      if (h == 1) __syncthreads();  // the rows before are out of the buffer
      float* const row = jo + (warp * 8 + gr) * S::kPad;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        float x0, x1;
        if constexpr (WIDE) {
          x0 = acc[i][2 * h];
          x1 = acc[i][2 * h + 1];
        } else {
          x0 = acc[i][0] + acc[i][2];
          x1 = acc[i][1] + acc[i][3];
        }
        if constexpr (F8) {
          // tile 2k + e, column n -> head_dim 16k + 2n + e
          row[16 * (i / 2) + 4 * gc + (i & 1)] = x0;
          row[16 * (i / 2) + 4 * gc + 2 + (i & 1)] = x1;
        } else {
          *reinterpret_cast<float2*>(row + 8 * i + 2 * gc) = make_float2(x0, x1);
        }
      }
      __syncthreads();
      const int here = min(8, rows - 8 * h);
      for (int e = threadIdx.x * 2; e < here * D; e += 2 * S::kThreads) {
        const int r = e / D, d = e % D;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < S::kWarps; ++w) top = fmaxf(top, join_ml[w][8 * h + r].x);
        const float ref = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f, x0 = 0.0f, x1 = 0.0f;
#pragma unroll
        for (int w = 0; w < S::kWarps; ++w) {
          const float2 ml = join_ml[w][8 * h + r];
          const float f = exp2f(ml.x - ref);
          const float2 v = *reinterpret_cast<const float2*>(jo + (w * 8 + r) * S::kPad + d);
          sum += ml.y * f;
          x0 += v.x * f;
          x1 += v.y * f;
        }
        if (bad) continue;
        if (starts && ends) {
          const float inv = P.cache.v_scale / sum;  // 0/0 where every score is -inf
          x0 = len == 0 ? 0.0f : x0 * inv;
          x1 = len == 0 ? 0.0f : x1 * inv;
          uint32_t* const out = reinterpret_cast<uint32_t*>(
              P.o + p.b * P.o_stride + (int64_t)(head0 + 8 * h + r) * D + d);
          *out = P.o_bf16 ? pack2<true>(x0, x1) : pack2<false>(x0, x1);
          if (P.lse && d == 0)
            P.lse[(int64_t)p.b * P.hkv * P.g + head0 + 8 * h + r] =
                (top + (log2f(sum) - kShift)) * 0.69314718055994531f;
        } else {
          const int64_t at = ((int64_t)blockIdx.x * 2 + part) * P.rows + 8 * h + r;
          *reinterpret_cast<float2*>(P.part_o + at * D + d) = make_float2(x0, x1);
          if (d == 0) P.part_ml[at] = make_float2(top, sum);
        }
      }
    }
    __syncthreads();
  }
  cp_async_wait<0>();
}

// Joins the parts of the unit that starts in CTA blockIdx.x and ends in a
// later one, for query row blockIdx.y: part 1 of the first CTA, part 0 of the
// others. Each warp sums every eighth part.
template <int D>
__global__ void __launch_bounds__(kJoinThreads)
    paged_join_kernel(const __grid_constant__ DecodeParams P) {
  __shared__ float warp_o[kJoinThreads / 32][D];
  __shared__ float2 warp_ml[kJoinThreads / 32];
  allow_dependent_launch();
  grid_dependency_wait();
  const int2 who = P.part_unit[blockIdx.x];
  const int r = blockIdx.y;
  if (who.x < 0) return;
  const int HU = P.hkv * P.chunks;
  const int b = who.x / HU, hu = who.x % HU;
  const int chunk = hu % P.chunks;
  if (chunk * P.rows + r >= P.g) return;
  const int head = (hu / P.chunks) * P.g + chunk * P.rows + r;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int V = D / 128;  // float4s of a lane
  float4 x[V];
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = -INFINITY, l = 0.0f;
#pragma unroll 4
  for (int c = blockIdx.x + warp; c <= who.y; c += kJoinThreads / 32) {
    const int64_t at = ((int64_t)c * 2 + (c == (int)blockIdx.x ? 1 : 0)) * P.rows + r;
    const float2 ml = P.part_ml[at];
    const float now = fmaxf(m, ml.x);
    const float ref = now == -INFINITY ? 0.0f : now;
    const float f0 = exp2f(m - ref), f1 = exp2f(ml.x - ref);
    m = now;
    l = l * f0 + ml.y * f1;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float4 y = *reinterpret_cast<const float4*>(P.part_o + at * D + 128 * i + 4 * lane);
      x[i].x = x[i].x * f0 + y.x * f1;
      x[i].y = x[i].y * f0 + y.y * f1;
      x[i].z = x[i].z * f0 + y.z * f1;
      x[i].w = x[i].w * f0 + y.w * f1;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    *reinterpret_cast<float4*>(&warp_o[warp][128 * i + 4 * lane]) = x[i];
  if (lane == 0) warp_ml[warp] = make_float2(m, l);
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) top = fmaxf(top, warp_ml[w].x);
  const float ref = top == -INFINITY ? 0.0f : top;
  const int d = 2 * threadIdx.x;
  if (d >= D) return;
  float sum = 0.0f, x0 = 0.0f, x1 = 0.0f;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) {
    const float f = exp2f(warp_ml[w].x - ref);
    sum += warp_ml[w].y * f;
    x0 += warp_o[w][d] * f;
    x1 += warp_o[w][d + 1] * f;
  }
  const float inv = P.cache.v_scale / sum;
  uint32_t* const out = reinterpret_cast<uint32_t*>(P.o + b * P.o_stride + (int64_t)head * D + d);
  *out = P.o_bf16 ? pack2<true>(x0 * inv, x1 * inv) : pack2<false>(x0 * inv, x1 * inv);
  if (P.lse && d == 0)
    P.lse[(int64_t)b * P.hkv * P.g + head] = (top + (log2f(sum) - P.shift)) * 0.69314718055994531f;
}

using DecodeFn = void (*)(const DecodeParams);

template <int D, bool BF16, bool F8>
DecodeFn decode_fn_wide(bool wide) {
  return wide ? paged_decode_kernel<D, BF16, F8, true> : paged_decode_kernel<D, BF16, F8, false>;
}

template <int D>
DecodeFn decode_fn(bool bf16, bool f8, bool wide) {
  if (bf16) return f8 ? decode_fn_wide<D, true, true>(wide) : decode_fn_wide<D, true, false>(wide);
  return f8 ? decode_fn_wide<D, false, true>(wide) : decode_fn_wide<D, false, false>(wide);
}

template <int D>
int decode_smem(bool f8) {
  return f8 ? DecodeShape<D, true>::kSmem : DecodeShape<D, false>::kSmem;
}
template <int D>
int decode_threads(bool f8) {
  return f8 ? DecodeShape<D, true>::kThreads : DecodeShape<D, false>::kThreads;
}

// Query heads of a unit, and the units of a kv head.
void unit_rows(int g, int* rows, int* chunks) {
  *chunks = (g + kMaxRows - 1) / kMaxRows;
  *rows = (g + *chunks - 1) / *chunks;
}

// The workspace: partial outputs, then (m, l), then the units to join.
int64_t workspace_bytes_for(int rows, int d) {
  return (int64_t)kMaxCtas * 2 * rows * (d * 4 + 8) + (int64_t)kMaxCtas * 8;
}

}  // namespace
}  // namespace fmha

using namespace fmha;

extern "C" int64_t fmha_paged_decode_workspace(int num_heads_q, int num_heads_kv, int head_dim) {
  if (check_heads(num_heads_q, num_heads_kv, head_dim) != FMHA_OK) return -1;
  int rows, chunks;
  unit_rows(num_heads_q / num_heads_kv, &rows, &chunks);
  return workspace_bytes_for(rows, head_dim);
}

extern "C" fmha_status_t fmha_paged_decode(const void* Q, const fmha_paged_cache_t* cache, void* O,
                                           float* LSE, int batch, int num_heads_q,
                                           int num_heads_kv, int head_dim, int64_t q_stride,
                                           int64_t o_stride, float softmax_scale, int dtype,
                                           int o_dtype, void* workspace, int64_t workspace_bytes,
                                           fmha_stream_t stream) {
  if (batch < 0) return FMHA_ERR_INVALID_ARG;
  fmha_status_t st = check_heads(num_heads_q, num_heads_kv, head_dim);
  if (st != FMHA_OK) return st;
  if (dtype != FMHA_DTYPE_BF16 && dtype != FMHA_DTYPE_FP16) return FMHA_ERR_UNSUPPORTED;
  if (o_dtype != FMHA_DTYPE_BF16 && o_dtype != FMHA_DTYPE_FP16) return FMHA_ERR_UNSUPPORTED;
  if (!(softmax_scale >= 0.0f) || std::isinf(softmax_scale)) return FMHA_ERR_INVALID_ARG;
  if (batch == 0) return FMHA_OK;
  if ((st = check_rows(Q, q_stride, num_heads_q, head_dim)) != FMHA_OK ||
      (st = check_rows(O, o_stride, num_heads_q, head_dim)) != FMHA_OK)
    return st;
  DecodeParams P;
  std::memset(&P, 0, sizeof(P));
  if ((st = check_cache(cache, num_heads_kv, head_dim, dtype, &P.cache)) != FMHA_OK) return st;
  if (reinterpret_cast<uintptr_t>(LSE) & 3u) return FMHA_ERR_MISALIGNED;
  P.g = num_heads_q / num_heads_kv;
  unit_rows(P.g, &P.rows, &P.chunks);
  if (!workspace || workspace_bytes < workspace_bytes_for(P.rows, head_dim))
    return FMHA_ERR_INVALID_ARG;
  if (!aligned16(workspace)) return FMHA_ERR_MISALIGNED;
  if ((int64_t)batch * num_heads_kv * P.chunks > (int64_t)1 << 30) return FMHA_ERR_UNSUPPORTED;
  ServingDevice dev;
  if ((st = serving_device(&dev)) != FMHA_OK) return st;
  P.q = static_cast<const uint16_t*>(Q);
  P.o = static_cast<uint16_t*>(O);
  P.lse = LSE;
  P.batch = batch;
  P.hkv = num_heads_kv;
  P.q_stride = q_stride;
  P.o_stride = o_stride;
  const double scale =
      softmax_scale > 0.0f ? (double)softmax_scale : 1.0 / std::sqrt((double)head_dim);
  P.scale_log2 = (float)(1.4426950408889634 * scale * P.cache.k_scale);
  P.o_bf16 = o_dtype == FMHA_DTYPE_BF16;
  P.err = dev.err;
  const int64_t units = (int64_t)batch * num_heads_kv * P.chunks;
  const int64_t longest = (int64_t)P.cache.max_pages * P.cache.page_size;  // tokens
  P.whole = longest <= kWholeTiles * kTile;
  int ctas = dev.sms < kMaxCtas ? dev.sms : kMaxCtas;
  if (P.whole && units < ctas) ctas = (int)units;
  char* w = static_cast<char*>(workspace);
  P.part_o = reinterpret_cast<float*>(w);
  w += (int64_t)kMaxCtas * 2 * P.rows * head_dim * 4;
  P.part_ml = reinterpret_cast<float2*>(w);
  w += (int64_t)kMaxCtas * 2 * P.rows * 8;
  P.part_unit = reinterpret_cast<int2*>(w);

  const bool f8 = P.cache.dtype == FMHA_DTYPE_E4M3, wide = P.rows > 8;
  const bool bf16 = dtype == FMHA_DTYPE_BF16;
  P.shift = bf16 && !f8 ? weight_shift<true, false>() : weight_shift<false, false>();
  const DecodeFn fn = head_dim == 128 ? decode_fn<128>(bf16, f8, wide)
                                      : decode_fn<256>(bf16, f8, wide);
  const int smem = head_dim == 128 ? decode_smem<128>(f8) : decode_smem<256>(f8);
  const int threads = head_dim == 128 ? decode_threads<128>(f8) : decode_threads<256>(f8);
  if ((st = ensure_smem(reinterpret_cast<const void*>(fn), smem)) != FMHA_OK) return st;
  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  st = launch_serving(fn, dim3(ctas), threads, smem, cs, P);
  if (st != FMHA_OK || P.whole) return st;
  return launch_serving(head_dim == 128 ? paged_join_kernel<128> : paged_join_kernel<256>,
                        dim3(ctas, P.rows), kJoinThreads, 0, cs, P);
}
