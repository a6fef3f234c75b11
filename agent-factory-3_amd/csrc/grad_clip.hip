// The norm of many gradients taken as one vector, and its clipping.  (The reference's
// training step calls torch's clip_grad_norm_ through accelerate, whose form for many
// tensors is a norm per tensor, a norm of the norms and a product per tensor.)
//
//   n = (sum |g|^p)^(1/p), p = 1 or 2, or max |g|;   g *= min(1, max_norm / (n + 1e-6))
//
// Adapters are hundreds of tensors of some 10^4 to 10^8 elements, so what counts is to
// reach all of them in few launches: their addresses and lengths go into the kernel's
// arguments (kTabN tensors a launch, nothing is copied to the card, and a captured graph
// holds them), the launch's blocks take one chunk of one tensor each, and a block finds
// its tensor with one look of a wave over the chunks' prefix sums.
//   norm:  a block adds up its chunk in 64 bits (bf16 and fp32 gradients of any size
//     neither overflow nor vanish; a 16-byte load is 4 to 8 conversions and 64-bit
//     multiply-adds, under the load's time) and writes one partial.
//   scale: every block adds up the partials in the same order (16 KB from the L2 where
//     there are 2048 of them), so norm and factor need no launch of their own; with a
//     factor of 1 it ends there and the gradients are not touched.
// HBM bounds both.  Measured, us: 192 fp32 tensors of 8 million elements, norm 9
// and scale 12 (they stay in the last-level cache); 36 bf16 tensors of 531 million, norm
// 209 (5.1 TB/s) and scale 379 (5.6 read and written), with a factor of 1 5.5.
#include "af3_common.h"

#include <stdlib.h>

#include <algorithm>

namespace {

constexpr int kTabN = 192;      // tensors per launch: 3.8 KB of arguments (4 KB are the limit)
// Chunks aimed at (1024, 2048, 4096: 96 tensors of 4 million fp32 elements 1008, 958, 942 us,
// 192 of 207360 80, 76, 77), and the least that is worth a block.
constexpr int kClipBlocks = 2048;
constexpr int kClipMinChunk = 8192;

struct ClipTab {
  uint64_t ptr[kTabN];
  uint32_t chunks[kTabN];       // chunks of the tensors before this one
  uint64_t size[kTabN];         // elements << 1 | (1: fp32, 0: bf16)
};

struct ClipPos {
  const void* p;
  int64_t n;  // elements of the chunk
  int f32;
};

// the chunk of block b
__device__ __forceinline__ ClipPos clip_find(const ClipTab& tab, int n_tab, int64_t chunk, uint32_t b) {
  const int lane = threadIdx.x & 63;
  int at = -1;
#pragma unroll
  for (int i = 0; i < kTabN / 64; ++i) {
    const int j = i * 64 + lane;
    at += __popcll(__ballot(j < n_tab && tab.chunks[j < n_tab ? j : 0] <= b));
  }
  at = __builtin_amdgcn_readfirstlane(at);
  const uint64_t size = tab.size[at];
  const int64_t n = (int64_t)(size >> 1), begin = (int64_t)(b - tab.chunks[at]) * chunk;
  ClipPos c;
  c.f32 = (int)(size & 1);
  c.p = (const void*)(tab.ptr[at] + (uint64_t)begin * (c.f32 ? 4 : 2));
  c.n = min(chunk, n - begin);
  return c;
}

template <int P>
__device__ __forceinline__ void clip_add(double& s, float f) {
  if constexpr (P == 2)
    s = fma((double)f, (double)f, s);
  else if constexpr (P == 1)
    s += fabs((double)f);
  else  // the largest; a NaN stays
    s = (fabsf(f) > s || f != f) ? (double)fabsf(f) : s;
}
template <int P>
__device__ __forceinline__ double clip_join(double a, double b) {
  if constexpr (P == 0)
    return (a != a || a > b) ? a : b;  // (b NaN: returned, as a > NaN is false)
  else
    return a + b;
}

template <int P>
__device__ __forceinline__ double clip_block_sum(double s, double* lds) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) s = clip_join<P>(s, __shfl_xor(s, o));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  s = lds[0];
#pragma unroll
  for (int w = 1; w < 4; ++w) s = clip_join<P>(s, lds[w]);
  return s;
}

template <int P>
__global__ __launch_bounds__(256) void clip_norm_kernel(const ClipTab tab, int n_tab, int64_t chunk, double* partials) {
  __shared__ double lds[4];
  const ClipPos c = clip_find(tab, n_tab, chunk, blockIdx.x);
  double s[2] = {0.0, 0.0};
  if (c.f32) {
    const float* const p = (const float*)c.p;
    const int64_t nv = c.n / 4;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < nv; i += 256) {
      float f[4];
      __builtin_memcpy(f, p + i * 4, 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) clip_add<P>(s[k & 1], f[k]);
    }
    for (int64_t i = nv * 4 + threadIdx.x; i < c.n; i += 256) clip_add<P>(s[0], p[i]);
  } else {
    const uint16_t* const p = (const uint16_t*)c.p;
    const int64_t nv = c.n / 8;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < nv; i += 256) {
      uint32_t w[4];
      __builtin_memcpy(w, p + i * 8, 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        clip_add<P>(s[0], af3_bf16_to_f32(w[k]));
        clip_add<P>(s[1], af3_bf16_to_f32(w[k] >> 16));
      }
    }
    for (int64_t i = nv * 8 + threadIdx.x; i < c.n; i += 256) clip_add<P>(s[0], af3_bf16_to_f32(p[i]));
  }
  const double total = clip_block_sum<P>(clip_join<P>(s[0], s[1]), lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = total;
}

// the partials' sum (or largest), the same in every block
template <int P>
__device__ __forceinline__ double clip_total(const double* partials, int n, double* lds) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) s = clip_join<P>(s, partials[i]);
  return clip_block_sum<P>(s, lds);
}

template <int P>
__device__ __forceinline__ double clip_norm_of(double s) {
  return P == 2 ? sqrt(s) : s;
}

template <int P>
__global__ __launch_bounds__(256) void clip_sum_kernel(const double* partials, int n, double* sum, float* norm) {
  __shared__ double lds[4];
  const double s = clip_total<P>(partials, n, lds);
  if (threadIdx.x == 0) {
    if (sum) *sum = s;
    if (norm) *norm = (float)clip_norm_of<P>(s);
  }
}

template <int P>
__global__ __launch_bounds__(256) void clip_scale_kernel(const ClipTab tab, int n_tab, int64_t chunk,
                                                         const double* partials, int n_partials, double max_norm,
                                                         float* norm_out) {
  __shared__ double lds[4];
  const double norm = clip_norm_of<P>(clip_total<P>(partials, n_partials, lds));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  // the factor is every gradient's, so it is rounded once, from 64 bits.  (A norm that is infinite in fp32, as
  // it is returned, scales by 0.)
  const double factor = max_norm / (isinf((float)norm) ? (double)INFINITY : norm + 1e-6);
  if (factor >= 1.0) return;  // (a NaN norm goes on, and makes every gradient NaN)
  const float f = (float)factor;
  const ClipPos c = clip_find(tab, n_tab, chunk, blockIdx.x);
  if (c.f32) {
    float* const p = (float*)c.p;
    const int64_t nv = c.n / 4;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < nv; i += 256) {
      float v[4];
      __builtin_memcpy(v, p + i * 4, 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] *= f;
      __builtin_memcpy(p + i * 4, v, 16);
    }
    for (int64_t i = nv * 4 + threadIdx.x; i < c.n; i += 256) p[i] *= f;
  } else {
    uint16_t* const p = (uint16_t*)c.p;
    const int64_t nv = c.n / 8;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < nv; i += 256) {
      uint32_t w[4];
      __builtin_memcpy(w, p + i * 8, 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = af3_pack_bf16x2(af3_bf16_to_f32(w[k]) * f, af3_bf16_to_f32(w[k] >> 16) * f);
      __builtin_memcpy(p + i * 8, w, 16);
    }
    for (int64_t i = nv * 8 + threadIdx.x; i < c.n; i += 256)
      p[i] = (uint16_t)af3_f32_to_bf16(af3_bf16_to_f32(p[i]) * f);
  }
}

// elements per chunk for gradients of `total` elements: a multiple of 8192
int64_t clip_chunk(int64_t total) {
  const int64_t c = af3_cdiv(af3_cdiv(total, kClipBlocks), kClipMinChunk) * kClipMinChunk;
  return c < kClipMinChunk ? kClipMinChunk : c;
}

int clip_check(const char* who, const uint64_t* ptrs, const int64_t* sizes, const uint8_t* is_f32, int n, int norm_type,
               int64_t* total, int64_t* chunks) {
  AF3_REQUIRE(n >= 0 && (n == 0 || (ptrs && sizes && is_f32)), "%s: null arrays", who);
  AF3_REQUIRE(norm_type >= 0 && norm_type <= 2, "%s: norm_type %d (1, 2, or 0 for the largest)", who, norm_type);
  *total = 0;
  for (int i = 0; i < n; ++i) {
    AF3_REQUIRE(sizes[i] > 0 && sizes[i] < (int64_t)1 << 40 && ptrs[i], "%s: tensor %d is empty, null or too large", who, i);
    AF3_REQUIRE(ptrs[i] % (is_f32[i] ? 4 : 2) == 0, "%s: tensor %d is not aligned to its elements", who, i);
    *total += sizes[i];
  }
  const int64_t c = clip_chunk(*total);
  *chunks = 0;
  for (int i = 0; i < n; ++i) *chunks += af3_cdiv(sizes[i], c);
  AF3_REQUIRE(*chunks < (int64_t)1 << 30, "%s: too many tensors", who);
  return 0;
}

// whether no two tensors share memory (they are scaled side by side)
int clip_apart(const char* who, const uint64_t* ptrs, const int64_t* sizes, const uint8_t* is_f32, int n) {
  struct Span {
    uint64_t begin, end;
  };
  if (n < 2) return 0;
  Span* const s = (Span*)malloc(sizeof(Span) * (size_t)n);
  AF3_REQUIRE(s, "%s: out of host memory", who);
  for (int i = 0; i < n; ++i) s[i] = {ptrs[i], ptrs[i] + (uint64_t)sizes[i] * (is_f32[i] ? 4 : 2)};
  std::sort(s, s + n, [](const Span& a, const Span& b) { return a.begin < b.begin; });
  bool apart = true;
  for (int i = 1; i < n; ++i) apart = apart && s[i].begin >= s[i - 1].end;
  free(s);
  AF3_REQUIRE(apart, "%s: two tensors share memory", who);
  return 0;
}

// one launch per kTabN tensors
template <class F>
void clip_tables(const uint64_t* ptrs, const int64_t* sizes, const uint8_t* is_f32, int n, int64_t chunk, F launch) {
  int64_t before = 0;
  for (int i = 0; i < n; i += kTabN) {
    ClipTab tab;
    const int m = n - i < kTabN ? n - i : kTabN;
    uint32_t at = 0;
    for (int j = 0; j < m; ++j) {
      tab.ptr[j] = ptrs[i + j];
      tab.chunks[j] = at;
      tab.size[j] = (uint64_t)sizes[i + j] << 1 | (is_f32[i + j] ? 1 : 0);
      at += (uint32_t)af3_cdiv(sizes[i + j], chunk);
    }
    for (int j = m; j < kTabN; ++j) tab.ptr[j] = 0, tab.chunks[j] = 0, tab.size[j] = 0;
    launch(tab, m, at, before);
    before += at;
  }
}

#define AF3_CLIP_P(norm_type, ...) \
  do {                              \
    if ((norm_type) == 2) {         \
      constexpr int P = 2;          \
      __VA_ARGS__;                  \
    } else if ((norm_type) == 1) {  \
      constexpr int P = 1;          \
      __VA_ARGS__;                  \
    } else {                        \
      constexpr int P = 0;          \
      __VA_ARGS__;                  \
    }                               \
  } while (0)

}  // namespace

extern "C" size_t af3_grad_norm_partials(const int64_t* sizes, int n) {
  int64_t total = 0, chunks = 0;
  for (int i = 0; i < n; ++i) total += sizes[i] > 0 ? sizes[i] : 0;
  const int64_t c = clip_chunk(total);
  for (int i = 0; i < n; ++i) chunks += sizes[i] > 0 ? af3_cdiv(sizes[i], c) : 0;
  return (size_t)chunks;
}

extern "C" int af3_grad_norm(const uint64_t* ptrs, const int64_t* sizes, const uint8_t* is_f32, int n, int norm_type,
                             double* partials, int64_t n_partials, double* sum, float* norm, void* stream_) {
  int64_t total, chunks;
  const int rc = clip_check("grad_norm", ptrs, sizes, is_f32, n, norm_type, &total, &chunks);
  if (rc) return rc;
  AF3_REQUIRE(n_partials >= chunks && (chunks == 0 || partials), "grad_norm: %lld partials are needed", (long long)chunks);
  hipStream_t st = (hipStream_t)stream_;
  const int64_t chunk = clip_chunk(total);
  clip_tables(ptrs, sizes, is_f32, n, chunk, [&](const ClipTab& tab, int m, uint32_t blocks, int64_t before) {
    AF3_CLIP_P(norm_type, hipLaunchKernelGGL((clip_norm_kernel<P>), dim3(blocks), dim3(256), 0, st, tab, m, chunk,
                                              partials + before));
  });
  if (sum || norm)
    AF3_CLIP_P(norm_type,
               hipLaunchKernelGGL((clip_sum_kernel<P>), dim3(1), dim3(256), 0, st, partials, (int)chunks, sum, norm));
  return af3::check_launch("grad_norm");
}

extern "C" int af3_grad_scale(const uint64_t* ptrs, const int64_t* sizes, const uint8_t* is_f32, int n, int norm_type,
                              const double* partials, int64_t n_partials, double max_norm, float* norm, void* stream_) {
  int64_t total, chunks;
  const int rc = clip_check("grad_scale", ptrs, sizes, is_f32, n, norm_type, &total, &chunks);
  if (rc) return rc;
  const int apart = clip_apart("grad_scale", ptrs, sizes, is_f32, n);
  if (apart) return apart;
  AF3_REQUIRE(n_partials >= 0 && n_partials < (int64_t)1 << 30 && (n_partials == 0 || partials), "grad_scale: bad partials");
  hipStream_t st = (hipStream_t)stream_;
  const int64_t chunk = clip_chunk(total);
  clip_tables(ptrs, sizes, is_f32, n, chunk, [&](const ClipTab& tab, int m, uint32_t blocks, int64_t before) {
    AF3_CLIP_P(norm_type, hipLaunchKernelGGL((clip_scale_kernel<P>), dim3(blocks), dim3(256), 0, st, tab, m, chunk,
                                              partials, (int)n_partials, max_norm, before ? nullptr : norm));
  });
  return af3::check_launch("grad_scale");
}
