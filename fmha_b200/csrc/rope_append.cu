// rope_append.cu -- fmha_rope_append: position rotation of the new tokens'
// queries and keys, and the write of the new keys and values into the paged
// cache, in one pass.
//
// A pair (x1, x2) of a head is turned by its position's angle:
//   y1 = x1*cos - x2*sin,  y2 = x2*cos + x1*sin
// in fp32, rounded once to the output's type. Every element is read once and
// written once, so HBM bandwidth bounds long prompts and launch latency a
// decode step.
//
// Split. One thread turns 16 elements of one head: two 16-byte vectors that
// hold both halves of 8 pairs (for interleaved pairs, and for elements behind
// rotary_dim, two adjacent vectors). Its chunk of the head is the same for
// all its heads, so it loads the 8 cosines and sines of a token once for all
// of them. A block takes a contiguous range of tokens and walks the heads
// (queries, keys, values) of one token at a time, up to kBatch of them with
// their loads in flight before the first is used; the token's sequence,
// position and page are looked up behind those loads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstring>

#include "../../include/fmha.h"
#include "decode_common.cuh"
#include "serving.hpp"

namespace fmha {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kBatch = 2;  // heads in flight per thread

struct AppendParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* q_out;
  uint16_t* k_out;  // or null
  fmha_paged_cache_t cache;
  const int32_t* cu;  // or null: token t is sequence t's
  const float* cos_table;
  const float* sin_table;
  int total_tokens;
  int batch;
  int hq;
  int hkv;
  int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
  int rot;
  int max_position;
  unsigned int* err;
};

template <bool BF16>
__device__ __forceinline__ void unpack16(const uint4 w, float (&f)[8]) {
  if constexpr (BF16) {
    unpack8(w, f);
  } else {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
}

template <bool BF16>
__device__ __forceinline__ uint4 pack16(const float (&f)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&p);
    } else {
      const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// 8 values divided by the cache's scale, as saturated e4m3 codes.
__device__ __forceinline__ uint2 pack_e4m3(const float (&f)[8], float scale) {
  uint32_t u[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i] / scale, f[4 * i + 1] / scale),
                                                 __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(
        make_float2(f[4 * i + 2] / scale, f[4 * i + 3] / scale), __NV_SATFINITE, __NV_E4M3);
    u[i] = lo | (hi << 16);
  }
  return make_uint2(u[0], u[1]);
}

__device__ __forceinline__ uint4 ld16(const uint16_t* p) {
  return __ldcs(reinterpret_cast<const uint4*>(p));
}

template <bool BF16, bool F8, bool INTER, int D>
__global__ void __launch_bounds__(kAppendThreads)
    rope_append_kernel(const __grid_constant__ AppendParams P) {
  constexpr int kChunks = D / 16;                   // threads of one head
  constexpr int kSlots = kAppendThreads / kChunks;  // heads side by side
  allow_dependent_launch();
  grid_dependency_wait();
  const int c = threadIdx.x % kChunks;
  const int slot = threadIdx.x / kChunks;
  const bool turned = c * 16 < P.rot;
  // Offsets of the thread's two vectors in a rotated head; values keep to
  // adjacent vectors.
  const int lo = !INTER && turned ? 8 * c : 16 * c;
  const int hi = !INTER && turned ? 8 * c + P.rot / 2 : 16 * c + 8;
  const int heads = P.hq + 2 * P.hkv;
  const int first = blockIdx.y * kSlots + slot;
  const int step = gridDim.y * kSlots;

  const int t0 = (int)((int64_t)P.total_tokens * blockIdx.x / gridDim.x);
  const int t1 = (int)((int64_t)P.total_tokens * (blockIdx.x + 1) / gridDim.x);
  int b = -1;
  for (int t = t0; t < t1; ++t) {
    const uint16_t* const q = P.q + t * P.q_stride;
    const uint16_t* const k = P.k + t * P.k_stride;
    const uint16_t* const v = P.v + t * P.v_stride;
    auto source = [&](int h, int off, bool second) {
      if (h < P.hq) return q + (int64_t)h * D + off;
      if (h < P.hq + P.hkv) return k + (int64_t)(h - P.hq) * D + off;
      return v + (int64_t)(h - P.hq - P.hkv) * D + 16 * c + (second ? 8 : 0);
    };
    uint4 x[kBatch][2];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = first + i * step;
      if (h < heads) {
        x[i][0] = ld16(source(h, lo, false));
        x[i][1] = ld16(source(h, hi, true));
      }
    }

    // The token's sequence (the last one that starts at or before t),
    // position, page and angles.
    int pos;
    if (P.cu) {
      if (b < 0) {
        int l = 0, r = P.batch;  // cu[l] <= t < cu[r], if t is anyone's
        while (r - l > 1) {
          const int m = (l + r) >> 1;
          if (P.cu[m] <= t) l = m; else r = m;
        }
        b = l;
      }
      while (b + 1 < P.batch && P.cu[b + 1] <= t) ++b;
      const int end = P.cu[b + 1];
      if (t < P.cu[b] || t >= end) continue;  // behind the last sequence
      pos = P.cache.seqlens_kv[b] - (end - t);
      if (pos < t - P.cu[b]) pos = -1;  // fewer tokens than new ones
    } else {
      b = t;
      pos = P.cache.seqlens_kv[b] - 1;
    }
    const int in_table = pos / P.cache.page_size;
    if (pos < 0 || in_table >= P.cache.max_pages || (P.rot > 0 && pos >= P.max_position)) {
      if (threadIdx.x == 0) report_device_error(P.err, FMHA_ERR_INVALID_ARG, kSiteAppendPosition);
      continue;
    }
    const int page = P.cache.block_table[b * P.cache.table_stride + in_table];
    if (page < 0 || page >= P.cache.num_pages) {
      if (threadIdx.x == 0) report_device_error(P.err, FMHA_ERR_INVALID_ARG, kSiteAppendPage);
      continue;
    }
    const int64_t row = page * P.cache.page_stride +
                        (int64_t)(pos - in_table * P.cache.page_size) * P.cache.token_stride;
    float cs[8], sn[8];
    if (turned) {
      const int64_t at = (int64_t)pos * (P.rot / 2) + 8 * c;
      const float4* const pc = reinterpret_cast<const float4*>(P.cos_table + at);
      const float4* const ps = reinterpret_cast<const float4*>(P.sin_table + at);
      const float4 c0 = __ldg(pc), c1 = __ldg(pc + 1), s0 = __ldg(ps), s1 = __ldg(ps + 1);
      cs[0] = c0.x; cs[1] = c0.y; cs[2] = c0.z; cs[3] = c0.w;
      cs[4] = c1.x; cs[5] = c1.y; cs[6] = c1.z; cs[7] = c1.w;
      sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w;
      sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
    }

    auto put = [&](int h, const uint4 (&in)[2]) {
      const bool value = h >= P.hq + P.hkv;
      float a[8], z[8];
      uint4 out0 = in[0], out1 = in[1];
      if (F8 || (turned && !value)) {
        unpack16<BF16>(in[0], a);
        unpack16<BF16>(in[1], z);
      }
      if (turned && !value) {
        if constexpr (INTER) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float a1 = a[2 * i], a2 = a[2 * i + 1], z1 = z[2 * i], z2 = z[2 * i + 1];
            a[2 * i] = a1 * cs[i] - a2 * sn[i];
            a[2 * i + 1] = a2 * cs[i] + a1 * sn[i];
            z[2 * i] = z1 * cs[4 + i] - z2 * sn[4 + i];
            z[2 * i + 1] = z2 * cs[4 + i] + z1 * sn[4 + i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float x1 = a[i], x2 = z[i];
            a[i] = x1 * cs[i] - x2 * sn[i];
            z[i] = x2 * cs[i] + x1 * sn[i];
          }
        }
        out0 = pack16<BF16>(a);
        out1 = pack16<BF16>(z);
      }
      if (h < P.hq) {
        uint16_t* const o = P.q_out + t * P.q_out_stride + (int64_t)h * D;
        *reinterpret_cast<uint4*>(o + lo) = out0;
        *reinterpret_cast<uint4*>(o + hi) = out1;
        return;
      }
      const int kvh = value ? h - P.hq - P.hkv : h - P.hq;
      const int l = value ? 16 * c : lo, r = value ? 16 * c + 8 : hi;
      const int64_t at = row + kvh * P.cache.head_stride;
      if constexpr (F8) {
        uint8_t* const o = static_cast<uint8_t*>(value ? P.cache.v : P.cache.k) + at;
        const float scale = value ? P.cache.v_scale : P.cache.k_scale;
        *reinterpret_cast<uint2*>(o + l) = pack_e4m3(a, scale);
        *reinterpret_cast<uint2*>(o + r) = pack_e4m3(z, scale);
      } else {
        uint16_t* const o = static_cast<uint16_t*>(value ? P.cache.v : P.cache.k) + at;
        *reinterpret_cast<uint4*>(o + l) = out0;
        *reinterpret_cast<uint4*>(o + r) = out1;
      }
      if (!value && P.k_out) {
        uint16_t* const o = P.k_out + t * P.k_out_stride + (int64_t)kvh * D;
        *reinterpret_cast<uint4*>(o + lo) = out0;
        *reinterpret_cast<uint4*>(o + hi) = out1;
      }
    };
    for (int h0 = first; h0 < heads; h0 += kBatch * step) {
      if (h0 != first) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int h = h0 + i * step;
          if (h < heads) {
            x[i][0] = ld16(source(h, lo, false));
            x[i][1] = ld16(source(h, hi, true));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i)
        if (h0 + i * step < heads) put(h0 + i * step, x[i]);
    }
  }
}

using AppendFn = void (*)(const AppendParams);

template <bool BF16, bool F8, bool INTER>
AppendFn append_fn_d(int d) {
  return d == 128 ? rope_append_kernel<BF16, F8, INTER, 128>
                  : rope_append_kernel<BF16, F8, INTER, 256>;
}

AppendFn append_fn(bool bf16, bool f8, bool inter, int d) {
  if (bf16) {
    if (f8) return inter ? append_fn_d<true, true, true>(d) : append_fn_d<true, true, false>(d);
    return inter ? append_fn_d<true, false, true>(d) : append_fn_d<true, false, false>(d);
  }
  if (f8) return inter ? append_fn_d<false, true, true>(d) : append_fn_d<false, true, false>(d);
  return inter ? append_fn_d<false, false, true>(d) : append_fn_d<false, false, false>(d);
}

}  // namespace
}  // namespace fmha

using namespace fmha;

extern "C" fmha_status_t fmha_rope_append(const fmha_rope_append_args_t* args,
                                          fmha_stream_t stream) {
  if (!args) return FMHA_ERR_INVALID_ARG;
  const fmha_rope_append_args_t& A = *args;
  if (A.total_tokens < 0 || A.batch < 0 || A.rotary_dim < 0) return FMHA_ERR_INVALID_ARG;
  fmha_status_t st = check_heads(A.num_heads_q, A.num_heads_kv, A.head_dim);
  if (st != FMHA_OK) return st;
  if (A.dtype != FMHA_DTYPE_BF16 && A.dtype != FMHA_DTYPE_FP16) return FMHA_ERR_UNSUPPORTED;
  if (A.rotary_dim % 16 != 0 || A.rotary_dim > A.head_dim) return FMHA_ERR_UNSUPPORTED;
  if (!A.cu_seqlens_q && A.total_tokens != A.batch) return FMHA_ERR_INVALID_ARG;
  if (A.total_tokens == 0 || A.batch == 0) return FMHA_OK;
  const int hq = A.num_heads_q, hkv = A.num_heads_kv, d = A.head_dim;
  if ((st = check_rows(A.q, A.q_stride, hq, d)) != FMHA_OK ||
      (st = check_rows(A.k, A.k_stride, hkv, d)) != FMHA_OK ||
      (st = check_rows(A.v, A.v_stride, hkv, d)) != FMHA_OK ||
      (st = check_rows(A.q_out, A.q_out_stride, hq, d)) != FMHA_OK ||
      (A.k_out && (st = check_rows(A.k_out, A.k_out_stride, hkv, d)) != FMHA_OK))
    return st;
  if (A.rotary_dim > 0) {
    if (!A.cos_table || !A.sin_table || A.max_position <= 0) return FMHA_ERR_INVALID_ARG;
    if (!aligned16(A.cos_table) || !aligned16(A.sin_table)) return FMHA_ERR_MISALIGNED;
  }
  if (reinterpret_cast<uintptr_t>(A.cu_seqlens_q) & 3u) return FMHA_ERR_MISALIGNED;
  // In place only row upon row: another stride would write rows still to be read.
  if ((A.q_out == A.q && A.q_out_stride != A.q_stride) ||
      (A.k_out && A.k_out == A.k && A.k_out_stride != A.k_stride))
    return FMHA_ERR_INVALID_ARG;
  AppendParams P;
  std::memset(&P, 0, sizeof(P));
  if ((st = check_cache(A.cache, hkv, d, A.dtype, &P.cache)) != FMHA_OK) return st;
  ServingDevice dev;
  if ((st = serving_device(&dev)) != FMHA_OK) return st;
  P.q = static_cast<const uint16_t*>(A.q);
  P.k = static_cast<const uint16_t*>(A.k);
  P.v = static_cast<const uint16_t*>(A.v);
  P.q_out = static_cast<uint16_t*>(A.q_out);
  P.k_out = static_cast<uint16_t*>(A.k_out);
  P.cu = A.cu_seqlens_q;
  P.cos_table = A.cos_table;
  P.sin_table = A.sin_table;
  P.total_tokens = A.total_tokens;
  P.batch = A.batch;
  P.hq = hq;
  P.hkv = hkv;
  P.q_stride = A.q_stride;
  P.k_stride = A.k_stride;
  P.v_stride = A.v_stride;
  P.q_out_stride = A.q_out_stride;
  P.k_out_stride = A.k_out_stride;
  P.rot = A.rotary_dim;
  P.max_position = A.max_position;
  P.err = dev.err;
  // A block per token while they fit side by side; with few tokens the heads
  // of each are dealt to several blocks.
  const int slots = kAppendThreads / (d / 16);
  const int heads = hq + 2 * hkv;
  const int resident = dev.sms * 6;
  const int gx = A.total_tokens < resident ? A.total_tokens : resident;
  int gy = 1;
  const int most = (heads + slots - 1) / slots;
  while (gy < most && gx * gy * 2 <= resident) ++gy;
  return launch_serving(append_fn(A.dtype == FMHA_DTYPE_BF16, P.cache.dtype == FMHA_DTYPE_E4M3,
                                  A.interleaved != 0, d),
                        dim3(gx, gy), kAppendThreads, 0, reinterpret_cast<cudaStream_t>(stream),
                        P);
}
