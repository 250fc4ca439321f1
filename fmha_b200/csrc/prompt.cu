// prompt.cu -- fmha_prompt: attention over packed prompts of different
// lengths, causal or not, with grouped query heads.
//
// Mathematics: per query row one pass over the keys with the running maximum
// m and sum l of 2^(s - m), s = scale*log2(e) * q.k, and o = sum 2^(s - m) v
// (fp32); O = o / l.
//
// Split: a CTA takes 64 query rows of one (sequence, head), 16 to a warp, and
// walks the sequence's keys in tiles through a two-stage cp.async ring.
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>

#include "../../include/fmha.h"
#include "decode_common.cuh"
#include "serving.hpp"
#include "serving_mma.cuh"

namespace fmha {
namespace {

struct PromptParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  float* lse;  // or null
  const int32_t* cu_q;
  const int32_t* cu_kv;
  int total_q, total_kv, batch, hq, hkv;
  int64_t q_stride, k_stride, v_stride, o_stride;
  float scale_log2;
  int causal;
  int o_bf16;
  unsigned int* err;
};

constexpr int kRowsQ = 64;
constexpr int kPromptThreads = 128;

template <int D>
struct PromptShape {
  static constexpr int kKeys = D == 128 ? 64 : 32;
  static constexpr int kRow = D * 2;
  static constexpr int kQ = kRowsQ * kRow;
  static constexpr int kKV = kKeys * kRow;
  static constexpr int kSmem = kQ + 4 * kKV;
};

// Sequence and first row of query tile `at`; false behind the last one.
__device__ bool find_tile(const PromptParams& P, int at, int* b_out, int* row_out) {
  const int lane = threadIdx.x & 31;
  for (int b0 = 0; b0 < P.batch; b0 += 32) {
    const int b = b0 + lane;
    int n = 0;
    if (b < P.batch) n = (max(0, P.cu_q[b + 1] - P.cu_q[b]) + kRowsQ - 1) / kRowsQ;
    int inc = n;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const int y = __shfl_up_sync(kFullMask, inc, s);
      if (lane >= s) inc += y;
    }
    const unsigned hit = __ballot_sync(kFullMask, at < inc);
    if (hit) {
      const int w = __ffs(hit) - 1;
      *b_out = b0 + w;
      *row_out = (at - __shfl_sync(kFullMask, inc - n, w)) * kRowsQ;
      return true;
    }
    at -= __shfl_sync(kFullMask, inc, 31);
  }
  return false;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kPromptThreads) prompt_kernel(const __grid_constant__ PromptParams P) {
  using S = PromptShape<D>;
  constexpr int kSteps = D / 16;
  constexpr int kCh = D / 8;
  extern __shared__ __align__(1024) uint8_t smem[];
  allow_dependent_launch();
  grid_dependency_wait();
  int b, row0;
  if (!find_tile(P, blockIdx.x, &b, &row0)) return;
  const int head = blockIdx.y, kvh = head / (P.hq / P.hkv);
  const int q0 = P.cu_q[b], nq = P.cu_q[b + 1] - q0;
  const int k0 = P.cu_kv[b], nk = P.cu_kv[b + 1] - k0;
  if (q0 < 0 || q0 + (int64_t)nq > P.total_q || k0 < 0 || nk < 0 || k0 + (int64_t)nk > P.total_kv) {
    if (threadIdx.x == 0) report_device_error(P.err, FMHA_ERR_INVALID_ARG, kSitePromptLength);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gr = lane >> 2, gc = lane & 3;
  const uint32_t sq = smem_u32(smem), skv = sq + S::kQ;
  auto fill = [&](uint32_t dst, const uint16_t* base, int64_t stride, int rows, int have) {
    for (int e = threadIdx.x; e < rows * kCh; e += kPromptThreads) {
      const int r = e / kCh, ch = e % kCh;
      cp_async16(dst + r * S::kRow + ((ch ^ (r & 7)) << 4), base + (r < have ? r : 0) * stride + ch * 8,
                 r < have ? 16 : 0);
    }
  };
  const int ahead = nk - nq;
  const int last_row = min(row0 + kRowsQ, nq) - 1;
  const int keys = P.causal ? max(0, min(nk, last_row + ahead + 1)) : nk;
  const int tiles = (keys + S::kKeys - 1) / S::kKeys;
  fill(sq, P.q + (int64_t)(q0 + row0) * P.q_stride + (int64_t)head * D, P.q_stride, kRowsQ, nq - row0);
  auto load = [&](int t) {
    if (t < tiles) {
      const uint32_t at = skv + (t & 1) * 2 * S::kKV;
      const int64_t r = k0 + (int64_t)t * S::kKeys;
      fill(at, P.k + r * P.k_stride + (int64_t)kvh * D, P.k_stride, S::kKeys, nk - t * S::kKeys);
      fill(at + S::kKV, P.v + r * P.v_stride + (int64_t)kvh * D, P.v_stride, S::kKeys,
           nk - t * S::kKeys);
    }
    cp_async_commit();
  };
  load(0);
  float acc[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  const int my0 = row0 + warp * 16 + gr;  // and + 8
  for (int t = 0; t < tiles; ++t) {
    load(t + 1);
    cp_async_wait<1>();
    __syncthreads();
    const uint32_t kt = skv + (t & 1) * 2 * S::kKV, vt = kt + S::kKV;
    float sc[S::kKeys / 8][4] = {};
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      uint32_t a[4];
      const int ra = warp * 16 + (lane & 15), ca = 2 * s + (lane >> 4);
      ldsm4(a, sq + ra * S::kRow + ((ca ^ (ra & 7)) << 4));
#pragma unroll
      for (int n = 0; n < S::kKeys / 16; ++n) {
        const int r = n * 16 + (lane & 7) + ((lane >> 4) << 3), ch = 2 * s + ((lane >> 3) & 1);
        uint32_t w[4];
        ldsm4(w, kt + r * S::kRow + ((ch ^ (r & 7)) << 4));
        mma16<BF16>(sc[2 * n], a[0], a[1], a[2], a[3], w[0], w[1]);
        mma16<BF16>(sc[2 * n + 1], a[0], a[1], a[2], a[3], w[2], w[3]);
      }
    }
    float down[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int seen = P.causal ? min(nk, my0 + 8 * h + ahead + 1) : nk;  // keys of this row
      float top = m[h];
#pragma unroll
      for (int n = 0; n < S::kKeys / 8; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int key = t * S::kKeys + n * 8 + 2 * gc + j;
          float& x = sc[n][2 * h + j];
          x = key < seen ? x * P.scale_log2 : -INFINITY;
          top = fmaxf(top, x);
        }
      top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 1));
      top = fmaxf(top, __shfl_xor_sync(kFullMask, top, 2));
      const float ref = top == -INFINITY ? 0.0f : top;
      down[h] = exp2f(m[h] - ref);
      m[h] = top;
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < S::kKeys / 8; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float& x = sc[n][2 * h + j];
          x = exp2f(x - ref);
          sum += x;
        }
      l[h] = l[h] * down[h] + sum;
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] *= down[j >> 1];
#pragma unroll
    for (int n = 0; n < S::kKeys / 16; ++n) {
      uint32_t hi[4], lo[4];
      split2<BF16>(sc[2 * n][0], sc[2 * n][1], hi[0], lo[0]);
      split2<BF16>(sc[2 * n][2], sc[2 * n][3], hi[1], lo[1]);
      split2<BF16>(sc[2 * n + 1][0], sc[2 * n + 1][1], hi[2], lo[2]);
      split2<BF16>(sc[2 * n + 1][2], sc[2 * n + 1][3], hi[3], lo[3]);
#pragma unroll
      for (int i = 0; i < kCh; i += 2) {
        const int r = n * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), ch = i + (lane >> 4);
        uint32_t w[4];
        ldsm4_trans(w, vt + r * S::kRow + ((ch ^ (r & 7)) << 4));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mma16<BF16>(acc[i + j], hi[0], hi[1], hi[2], hi[3], w[2 * j], w[2 * j + 1]);
          mma16<BF16>(acc[i + j], lo[0], lo[1], lo[2], lo[3], w[2 * j], w[2 * j + 1]);
        }
      }
    }
    __syncthreads();
  }
  cp_async_wait<0>();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(kFullMask, l[h], 1);
    l[h] += __shfl_xor_sync(kFullMask, l[h], 2);
    const int row = my0 + 8 * h;
    if (row >= nq) continue;
    const bool none = nk == 0 || (P.causal && row + ahead < 0);
    const float inv = 1.0f / l[h];
    uint16_t* const out = P.o + (int64_t)(q0 + row) * P.o_stride + (int64_t)head * D;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const float x = none ? 0.0f : acc[i][2 * h] * inv, y = none ? 0.0f : acc[i][2 * h + 1] * inv;
      *reinterpret_cast<uint32_t*>(out + 8 * i + 2 * gc) =
          P.o_bf16 ? pack2<true>(x, y) : pack2<false>(x, y);
    }
    if (P.lse && gc == 0)
      P.lse[(int64_t)(q0 + row) * P.hq + head] = (m[h] + log2f(l[h])) * 0.69314718055994531f;
  }
}

using PromptFn = void (*)(const PromptParams);

}  // namespace
}  // namespace fmha

using namespace fmha;

extern "C" fmha_status_t fmha_prompt(const void* Q, const void* K, const void* V, void* O,
                                     float* LSE, const int32_t* cu_seqlens_q,
                                     const int32_t* cu_seqlens_kv, int total_q, int total_kv,
                                     int batch, int num_heads_q, int num_heads_kv, int head_dim,
                                     int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                     int64_t o_stride, float softmax_scale, int causal, int dtype,
                                     int o_dtype, fmha_stream_t stream) {
  if (total_q < 0 || total_kv < 0 || batch < 0) return FMHA_ERR_INVALID_ARG;
  fmha_status_t st = check_heads(num_heads_q, num_heads_kv, head_dim);
  if (st != FMHA_OK) return st;
  if (dtype != FMHA_DTYPE_BF16 && dtype != FMHA_DTYPE_FP16) return FMHA_ERR_UNSUPPORTED;
  if (o_dtype != FMHA_DTYPE_BF16 && o_dtype != FMHA_DTYPE_FP16) return FMHA_ERR_UNSUPPORTED;
  if (!(softmax_scale >= 0.0f) || std::isinf(softmax_scale)) return FMHA_ERR_INVALID_ARG;
  if (total_q == 0 || batch == 0) return FMHA_OK;
  if ((st = check_rows(Q, q_stride, num_heads_q, head_dim)) != FMHA_OK ||
      (st = check_rows(O, o_stride, num_heads_q, head_dim)) != FMHA_OK)
    return st;
  if (total_kv > 0 && ((st = check_rows(K, k_stride, num_heads_kv, head_dim)) != FMHA_OK ||
                       (st = check_rows(V, v_stride, num_heads_kv, head_dim)) != FMHA_OK))
    return st;
  if (!cu_seqlens_q) return FMHA_ERR_INVALID_ARG;
  if (!cu_seqlens_kv && total_kv != total_q) return FMHA_ERR_INVALID_ARG;
  if ((reinterpret_cast<uintptr_t>(LSE) | reinterpret_cast<uintptr_t>(cu_seqlens_q) |
       reinterpret_cast<uintptr_t>(cu_seqlens_kv)) & 3u)
    return FMHA_ERR_MISALIGNED;
  ServingDevice dev;
  if ((st = serving_device(&dev)) != FMHA_OK) return st;
  PromptParams P;
  std::memset(&P, 0, sizeof(P));
  P.q = static_cast<const uint16_t*>(Q);
  P.k = static_cast<const uint16_t*>(K);
  P.v = static_cast<const uint16_t*>(V);
  P.o = static_cast<uint16_t*>(O);
  P.lse = LSE;
  P.cu_q = cu_seqlens_q;
  P.cu_kv = cu_seqlens_kv ? cu_seqlens_kv : cu_seqlens_q;
  P.total_q = total_q;
  P.total_kv = total_kv;
  P.batch = batch;
  P.hq = num_heads_q;
  P.hkv = num_heads_kv;
  P.q_stride = q_stride;
  P.k_stride = k_stride;
  P.v_stride = v_stride;
  P.o_stride = o_stride;
  const double scale =
      softmax_scale > 0.0f ? (double)softmax_scale : 1.0 / std::sqrt((double)head_dim);
  P.scale_log2 = (float)(1.4426950408889634 * scale);
  P.causal = causal != 0;
  P.o_bf16 = o_dtype == FMHA_DTYPE_BF16;
  P.err = dev.err;
  const bool bf16 = dtype == FMHA_DTYPE_BF16;
  const PromptFn fn = head_dim == 128 ? (bf16 ? prompt_kernel<128, true> : prompt_kernel<128, false>)
                                      : (bf16 ? prompt_kernel<256, true> : prompt_kernel<256, false>);
  const int smem = head_dim == 128 ? PromptShape<128>::kSmem : PromptShape<256>::kSmem;
  if ((st = ensure_smem(reinterpret_cast<const void*>(fn), smem)) != FMHA_OK) return st;
  // No more tiles than this, whatever the lengths: each sequence has one that is not full.
  const int64_t tiles = (int64_t)batch + total_q / kRowsQ;
  if (tiles > 0x7fffffff) return FMHA_ERR_UNSUPPORTED;
  return launch_serving(fn, dim3((unsigned)tiles, num_heads_q), kPromptThreads, smem,
                        reinterpret_cast<cudaStream_t>(stream), P);
}
