// The router's load-balancing loss, the tokens per expert and the gradient of
// the logits.  (No kernel of the reference: its router takes no gradient,
// quantization.py:421, and mlp_forward returns the logits alone, 639-668.)
//
//   p_t = softmax(logits_t),  n = tokens counted (token_mask),
//   c_e = tokens counted whose K experts hold e (the given ids, or the top K:
//         ties to the lower id, NaN lowest, as the routing picks them),
//   loss = E sum_e (c_e / n) (sum_t p_te / n)            (0 when n = 0)
//   d logits_te = g E / n  p_te (c_e / n - sum_x p_tx c_x / n)
//
// The logits are read once per direction and the gradient written once; p is made
// again in the backward (two shuffled reductions over values already in registers)
// instead of being stored.  A row's E logits lie in LPR = E / 8 lanes (a power of
// two, 4 to 64), 8 consecutive experts each (one 16-byte load; 16 past 512 experts),
// so a wave takes 64 / LPR rows at a time, the top K are K maxima over
// (order-preserving logit bits, inverted id) keys, and a lane's column sums and
// counts stay in its registers over all its rows.  Column sums are fp32: a lane adds
// T / (4096 (64 / LPR)) rows once there are 512 blocks (128000 tokens of 128 experts:
// 8; ten million of 1024: 2441, whose additions are off by at most 2^-24 of the sum
// each, at random about 3e-6 in all), then lanes, waves and blocks are joined in a fixed order.
//
// 128000 tokens of 128 experts, ids given: sums 12.5 us (35 MB: 2.8 TB/s), join 4.6,
// gradient 20.2 (66 MB: 3.3 TB/s; a copy of as much takes 9.9); 16384 tokens, top 4:
// 9.7, 3.8 and 7.6.  The vector unit is busy 78% of the sums' cycles and 60% of the
// gradient's (67% and 27% at 16384 tokens): a row's exponentials and reductions, and
// for the top K its K rounds of maxima; the rest is waiting for loads a pass ahead.
// A call of 77 tokens is one launch of 5.2 us and one of 2.8.
#include "af3_common.h"

namespace {

constexpr int kBalThreads = 512;
constexpr int kBalMaxBlocks = 512;
constexpr int kBalMaxE = 1024;
constexpr float kLog2e = 1.4426950408889634f;

// bf16 bits -> 16-bit key in float order (-0 as +0; NaN lowest)
__device__ __forceinline__ uint32_t b_key16(uint32_t b) {
  if ((b & 0x7FFFu) > 0x7F80u) return 0u;
  if (b == 0x8000u) b = 0u;
  return (b & 0x8000u) ? (~b & 0xFFFFu) : (b | 0x8000u);
}

template <int CTRL>
__device__ __forceinline__ uint32_t b_dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xF, 0xF, true);
}

// value of the lane's partner at distance 1, 2, 4, 8 (row operations: after the
// smaller distances are joined, mirrored lanes hold the partner's value), 16, 32
template <int O>
__device__ __forceinline__ uint32_t b_partner(uint32_t x) {
  if constexpr (O == 1) return b_dpp<0xB1>(x);        // quad 1 0 3 2
  else if constexpr (O == 2) return b_dpp<0x4E>(x);   // quad 2 3 0 1
  else if constexpr (O == 4) return b_dpp<0x141>(x);  // mirror of 8
  else if constexpr (O == 8) return b_dpp<0x140>(x);  // mirror of 16
  else return (uint32_t)__shfl_xor((int)x, O);
}

template <int LPR, int O = 1>
__device__ __forceinline__ uint32_t b_max_u32(uint32_t x) {
  if constexpr (O < LPR) return b_max_u32<LPR, O * 2>(max(x, b_partner<O>(x)));
  else return x;
}
template <int LPR, int O = 1>
__device__ __forceinline__ float b_max(float x) {
  if constexpr (O < LPR) return b_max<LPR, O * 2>(fmaxf(x, __uint_as_float(b_partner<O>(__float_as_uint(x)))));
  else return x;
}
template <int LPR, int O = 1>
__device__ __forceinline__ float b_sum(float x) {
  if constexpr (O < LPR) return b_sum<LPR, O * 2>(x + __uint_as_float(b_partner<O>(__float_as_uint(x))));
  else return x;
}

// 8 C logits of a lane (experts c LPR 8 + lane 8 + i); -inf past E
template <int LPR, int C, bool VEC>
__device__ __forceinline__ void b_load(const uint16_t* row, int E, int l, uint32_t (&w)[4 * C]) {
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int x0 = (c * LPR + l) * 8;
    if constexpr (VEC) {  // E % 8 == 0
      const af3_u32x4 v = x0 < E ? *(const af3_u32x4*)(row + x0)
                                 : af3_u32x4{0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u};
#pragma unroll
      for (int i = 0; i < 4; ++i) w[4 * c + i] = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = x0 + 2 * i < E ? row[x0 + 2 * i] : 0xFF80u;
        const uint32_t b = x0 + 2 * i + 1 < E ? row[x0 + 2 * i + 1] : 0xFF80u;
        w[4 * c + i] = a | (b << 16);
      }
    }
  }
}

// exp(z - max) of the lane's logits, and their sum over the row
template <int LPR, int C>
__device__ __forceinline__ float b_exps(const uint32_t (&w)[4 * C], float (&e)[8 * C]) {
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < 8 * C; ++i) {
    e[i] = __uint_as_float((i & 1) ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    mx = fmaxf(mx, e[i]);
  }
  mx = b_max<LPR>(mx);
  // The rounding of mx log2(e) is a factor common to the row, which its sum takes out
  // again, while it is small: past 2^20 (experts all masked by the type's lowest value,
  // say) the row's differences come first.  (Taken first for every row, they cost the
  // sums of 128000 rows 4%: 13.0 us instead of 12.5.)
  if (__builtin_expect(fabsf(mx) > 1048576.f, 0)) {
#pragma unroll
    for (int i = 0; i < 8 * C; ++i) e[i] -= mx;
    mx = 0.f;
  }
  mx *= kLog2e;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8 * C; ++i) {
    e[i] = __builtin_amdgcn_exp2f(fmaf(e[i], kLog2e, -mx));
    s += e[i];
  }
  return b_sum<LPR>(s);
}

struct BalParams {
  const uint16_t* logits;
  int64_t ld;
  const int32_t* ids;      // [T][K] or NULL: the top K
  const uint8_t* mask;     // [T] or NULL
  int64_t T;
  int E, K, n_blocks;
  float* part;             // [n_blocks][E] column sums, then [n_blocks][E + 1] counts and tokens, then a ticket
  int32_t* part_n;
  uint32_t* ticket;
  float* colsum;           // [E]
  float* loss;
  int32_t* counts;         // [E]
  int32_t* stats;          // [E + 1]: counts and n, kept for the backward
};

// loss from the column sums and counts, by one wave (fixed order)
__device__ __forceinline__ void b_finish(const float* colsum, const int32_t* stats, int E, float* loss, int lane) {
  const double n = (double)stats[E];
  double s = 0.;
  for (int e = lane; e < E; e += 64) s += (double)stats[e] * (double)colsum[e];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (lane == 0) loss[0] = n > 0. ? (float)((double)E * s / (n * n)) : 0.f;
}

template <int LPR, int C, bool VEC, bool TOPK>
__global__ __launch_bounds__(kBalThreads) void balance_sums_kernel(BalParams p) {
  constexpr int RPW = 64 / LPR;              // rows of a wave
  constexpr int NW = kBalThreads / 64;
  constexpr int SLOTS = 8 * C * LPR;         // >= E
  __shared__ float cs[NW][SLOTS];
  __shared__ int32_t cn[SLOTS + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane % LPR, sub = lane / LPR;
  for (int i = threadIdx.x; i <= SLOTS; i += kBalThreads) cn[i] = 0;
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0u;
  float sum[8 * C];
  int32_t cnt[8 * C];
#pragma unroll
  for (int i = 0; i < 8 * C; ++i) sum[i] = 0.f, cnt[i] = 0;
  int32_t n = 0;
  const int64_t step = (int64_t)p.n_blocks * NW * RPW;
  const int64_t first = ((int64_t)blockIdx.x * NW + wave) * RPW;
  uint32_t nw[4 * C];  // the next rows, loaded a pass ahead (a pass alone costs a load's latency)
  uint8_t nm = 1;
  auto fetch = [&](int64_t t0) {
    const int64_t t = min(t0 + sub, p.T - 1);
    b_load<LPR, C, VEC>(p.logits + t * p.ld, p.E, l, nw);
    if (p.mask) nm = p.mask[t];
  };
  if (first < p.T) fetch(first);
  for (int64_t t0 = first; t0 < p.T; t0 += step) {
    const int64_t t = t0 + sub;
    const bool on = t < p.T && nm;
    uint32_t w[4 * C];
#pragma unroll
    for (int i = 0; i < 4 * C; ++i) w[i] = nw[i];
    if (t0 + step < p.T) fetch(t0 + step);
    float e[8 * C];
    const float inv = 1.f / b_exps<LPR, C>(w, e);
    if (on) {
      n += l == 0;
#pragma unroll
      for (int i = 0; i < 8 * C; ++i) sum[i] = fmaf(e[i], inv, sum[i]);
    }
    if constexpr (TOPK) {
      uint32_t key[8 * C];
#pragma unroll
      for (int i = 0; i < 8 * C; ++i) {
        const int x = ((i / 8) * LPR + l) * 8 + i % 8;
        const uint32_t b = (i & 1) ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu;
        key[i] = x < p.E ? (b_key16(b) << 16) | (0xFFFFu - (uint32_t)x) : 0u;
      }
      for (int j = 0; j < p.K; ++j) {
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < 8 * C; ++i) m = max(m, key[i]);
        m = b_max_u32<LPR>(m);
#pragma unroll
        for (int i = 0; i < 8 * C; ++i) {
          const bool hit = key[i] == m;
          cnt[i] += hit && on;
          key[i] = hit ? 0u : key[i];
        }
      }
    } else if (on) {
      for (int j = l; j < p.K; j += LPR) {
        const int e = p.ids[t * p.K + j];
        if (e >= 0 && e < p.E) atomicAdd(&cn[e], 1);  // whole numbers: any order gives the same
      }
    }
  }
  // join the wave's rows, then the block's waves
#pragma unroll
  for (int i = 0; i < 8 * C; ++i) {
    float s = sum[i];
    int32_t c = cnt[i];
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1) {
      s += __shfl_xor(s, o);
      if constexpr (TOPK) c += __shfl_xor(c, o);
    }
    if (sub == 0) {
      const int x = ((i / 8) * LPR + l) * 8 + i % 8;
      cs[wave][x] = s;
      if constexpr (TOPK) {
        if (c) atomicAdd(&cn[x], c);
      }
    }
  }
  if (n) atomicAdd(&cn[SLOTS], n);
  __syncthreads();
  const bool alone = p.n_blocks == 1;
  float* ps = alone ? p.colsum : p.part + (int64_t)blockIdx.x * p.E;
  int32_t* pn = alone ? p.stats : p.part_n + (int64_t)blockIdx.x * (p.E + 1);
  for (int e = threadIdx.x; e < p.E; e += kBalThreads) {
    float s = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) s += cs[x][e];
    ps[e] = s;
    pn[e] = cn[e];
    if (alone) p.counts[e] = cn[e];
  }
  if (threadIdx.x == 0) pn[p.E] = cn[SLOTS];
  if (alone) {
    __syncthreads();
    if (wave == 0) b_finish(p.colsum, p.stats, p.E, p.loss, lane);
  }
}

// column sums and counts over the blocks' partials: 16 experts per block, 64
// threads each with all their loads in flight; the block that ends last makes the loss
__global__ __launch_bounds__(1024) void balance_join_kernel(BalParams p) {
  constexpr int Y = 64, PER = kBalMaxBlocks / Y;
  __shared__ float cs[Y][17];
  __shared__ int32_t cn[Y][17];
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
  const int e = blockIdx.x * 16 + x;  // column E: the number of tokens
  float v[PER];
  int32_t n[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = y + i * Y;
    v[i] = b < p.n_blocks && e < p.E ? p.part[(int64_t)b * p.E + e] : 0.f;
    n[i] = b < p.n_blocks && e <= p.E ? p.part_n[(int64_t)b * (p.E + 1) + e] : 0;
  }
  float s = 0.f;
  int32_t c = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) s += v[i], c += n[i];
  cs[y][x] = s;
  cn[y][x] = c;
  for (int o = Y / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (y < o) {
      cs[y][x] += cs[y + o][x];
      cn[y][x] += cn[y + o][x];
    }
  }
  if (threadIdx.x >= 64) return;
  // the first wave alone writes, takes the ticket (which releases what it wrote)
  // and, if it is the last, makes the loss
  if (y == 0 && e <= p.E) {
    if (e < p.E) {
      p.colsum[e] = cs[0][x];
      p.counts[e] = cn[0][x];
    }
    p.stats[e] = cn[0][x];
  }
  uint32_t t = 0;
  if (threadIdx.x == 0) t = __hip_atomic_fetch_add(p.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
  if (__builtin_amdgcn_readfirstlane(t) != gridDim.x - 1) return;
  b_finish(p.colsum, p.stats, p.E, p.loss, threadIdx.x);
}

template <int LPR, int C, bool VEC>
__global__ __launch_bounds__(256) void balance_grad_kernel(const uint16_t* __restrict__ logits, int64_t ld,
                                                           const uint8_t* __restrict__ mask, int64_t T, int E,
                                                           const int32_t* __restrict__ stats,
                                                           const float* __restrict__ g, uint16_t* __restrict__ out) {
  constexpr int RPW = 64 / LPR;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l = lane % LPR, sub = lane / LPR;
  uint32_t nw[4 * C];  // the next rows, loaded a pass ahead (the first before the counts)
  uint8_t nm = 1;
  auto fetch = [&](int64_t t0) {
    const int64_t t = min(t0 + sub, T - 1);
    b_load<LPR, C, VEC>(logits + t * ld, E, l, nw);
    if (mask) nm = mask[t];
  };
  const int64_t first = ((int64_t)blockIdx.x * 4 + wave) * RPW;
  if (first < T) fetch(first);
  const float n = (float)stats[E];
  const float inv_n = n > 0.f ? 1.f / n : 0.f;
  const float scale = g[0] * (float)E * inv_n;
  float f[8 * C];
#pragma unroll
  for (int i = 0; i < 8 * C; ++i) {
    const int x = ((i / 8) * LPR + l) * 8 + i % 8;
    f[i] = x < E ? (float)stats[x] * inv_n : 0.f;
  }
  const int64_t step = (int64_t)gridDim.x * 4 * RPW;
  for (int64_t t0 = first; t0 < T; t0 += step) {
    const int64_t t = t0 + sub;
    const bool in = t < T, on = in && nm;
    uint32_t w[4 * C];
#pragma unroll
    for (int i = 0; i < 4 * C; ++i) w[i] = nw[i];
    if (t0 + step < T) fetch(t0 + step);
    // with e = exp(z - max): p = e / sum, p (f - p.f) scale = e (f k - d k), k = scale / sum, d = e.f / sum
    float e[8 * C];
    const float inv = 1.f / b_exps<LPR, C>(w, e);
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < 8 * C; ++i) d = fmaf(e[i], f[i], d);
    const float k = inv * scale;
    d = b_sum<LPR>(d) * inv * k;
    if (!in) continue;
    uint16_t* row = out + t * E;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int x0 = (c * LPR + l) * 8;
      af3_u32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 8 * c + 2 * i;
        const uint32_t y = af3_pack_bf16x2(e[j] * fmaf(f[j], k, -d), e[j + 1] * fmaf(f[j + 1], k, -d));
        v[i] = on ? y : 0u;  // (whatever the logits of a token left out are)
      }
      if constexpr (VEC) {
        if (x0 < E) *(af3_u32x4*)(row + x0) = v;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (x0 + i < E) row[x0 + i] = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
      }
    }
  }
}

int b_lanes(int E) {
  int l = 4;
  while (l < 64 && l * 8 < E) l *= 2;
  return l;
}

// one block while its waves take at most 4 passes; then as many as give each wave 4, up to kBalMaxBlocks
int b_blocks(int64_t T, int E) {
  const int64_t per = (int64_t)(kBalThreads / 64) * (64 / b_lanes(E)) * 4;
  const int64_t n = af3_cdiv(T, per);
  return n < 1 ? 1 : n > kBalMaxBlocks ? kBalMaxBlocks : (int)n;
}

template <int LPR, int C>
void b_launch_sums(const BalParams& p, bool vec, hipStream_t s) {
  const dim3 g(p.n_blocks), b(kBalThreads);
  if (p.ids) {
    if (vec) hipLaunchKernelGGL((balance_sums_kernel<LPR, C, true, false>), g, b, 0, s, p);
    else hipLaunchKernelGGL((balance_sums_kernel<LPR, C, false, false>), g, b, 0, s, p);
  } else {
    if (vec) hipLaunchKernelGGL((balance_sums_kernel<LPR, C, true, true>), g, b, 0, s, p);
    else hipLaunchKernelGGL((balance_sums_kernel<LPR, C, false, true>), g, b, 0, s, p);
  }
}

template <int LPR, int C>
void b_launch_grad(const uint16_t* logits, int64_t ld, const uint8_t* mask, int64_t T, int E, const int32_t* stats,
                   const float* g, uint16_t* out, bool vec, hipStream_t s) {
  const int64_t n = af3_cdiv(T, 4 * (64 / LPR));
  const dim3 grid((unsigned)(n < 2048 ? n : 2048)), b(256);
  if (vec) hipLaunchKernelGGL((balance_grad_kernel<LPR, C, true>), grid, b, 0, s, logits, ld, mask, T, E, stats, g, out);
  else hipLaunchKernelGGL((balance_grad_kernel<LPR, C, false>), grid, b, 0, s, logits, ld, mask, T, E, stats, g, out);
}

#define B_BY_LANES(E, FN, ...)                       \
  do {                                               \
    if ((E) > 512) FN<64, 2>(__VA_ARGS__);           \
    else switch (b_lanes(E)) {                       \
      case 4: FN<4, 1>(__VA_ARGS__); break;          \
      case 8: FN<8, 1>(__VA_ARGS__); break;          \
      case 16: FN<16, 1>(__VA_ARGS__); break;        \
      case 32: FN<32, 1>(__VA_ARGS__); break;        \
      default: FN<64, 1>(__VA_ARGS__); break;        \
    }                                                \
  } while (0)

}  // namespace

extern "C" size_t af3_balance_loss_workspace_bytes(int64_t n_tokens, int n_expts) {
  if (n_tokens < 0 || n_expts <= 0 || n_expts > kBalMaxE) return 0;
  const int nb = b_blocks(n_tokens, n_expts);
  return ((size_t)nb * (2 * n_expts + 1) + n_expts + 1) * 4;
}

extern "C" int af3_balance_loss_fwd(const uint16_t* logits, int64_t ld_logits, const int32_t* expt_indx,
                                    const uint8_t* token_mask, int64_t n_tokens, int n_expts_tot, int n_expts_act,
                                    float* loss, int32_t* counts, int32_t* stats, void* workspace, size_t ws_bytes,
                                    void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  const int64_t T = n_tokens;
  const int E = n_expts_tot, K = n_expts_act;
  AF3_REQUIRE(T >= 0 && E > 0 && E <= kBalMaxE && K > 0 && K <= E, "balance_loss: bad sizes (E <= %d)", kBalMaxE);
  AF3_REQUIRE(T * K < 0x7fffffffLL, "balance_loss: too many tokens");
  AF3_REQUIRE((T == 0 || logits) && loss && counts && stats && workspace, "balance_loss: null pointer");
  AF3_REQUIRE(ld_logits >= E || T <= 1, "balance_loss: rows overlap");
  AF3_REQUIRE(ws_bytes >= af3_balance_loss_workspace_bytes(T, E) && ((uintptr_t)workspace & 3) == 0,
              "balance_loss: workspace too small");
  BalParams p = {};
  p.logits = logits; p.ld = ld_logits; p.ids = expt_indx; p.mask = token_mask;
  p.T = T; p.E = E; p.K = K;
  p.n_blocks = b_blocks(T, E);
  p.part = (float*)workspace;
  p.part_n = (int32_t*)(p.part + (int64_t)p.n_blocks * E);
  p.colsum = (float*)(p.part_n + (int64_t)p.n_blocks * (E + 1));
  p.ticket = (uint32_t*)(p.colsum + E);
  p.loss = loss; p.counts = counts; p.stats = stats;
  const bool vec = E % 8 == 0 && ld_logits % 8 == 0 && ((uintptr_t)logits & 15) == 0;
  B_BY_LANES(E, b_launch_sums, p, vec, stream);
  if (p.n_blocks > 1)
    hipLaunchKernelGGL(balance_join_kernel, dim3(E / 16 + 1), dim3(1024), 0, stream, p);
  return af3::check_launch("balance_loss_fwd");
}

extern "C" int af3_balance_loss_bwd(const uint16_t* logits, int64_t ld_logits, const uint8_t* token_mask,
                                    int64_t n_tokens, int n_expts_tot, const int32_t* stats, const float* dloss,
                                    uint16_t* dlogits, void* stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  const int64_t T = n_tokens;
  const int E = n_expts_tot;
  AF3_REQUIRE(T >= 0 && E > 0 && E <= kBalMaxE, "balance_loss_bwd: bad sizes (E <= %d)", kBalMaxE);
  if (T == 0) return 0;
  AF3_REQUIRE(logits && stats && dloss && dlogits, "balance_loss_bwd: null pointer");
  AF3_REQUIRE(ld_logits >= E || T <= 1, "balance_loss_bwd: rows overlap");
  const bool vec = E % 8 == 0 && ld_logits % 8 == 0 && ((uintptr_t)logits & 15) == 0 && ((uintptr_t)dlogits & 15) == 0;
  B_BY_LANES(E, b_launch_grad, logits, ld_logits, token_mask, T, E, stats, dloss, dlogits, vec, stream);
  return af3::check_launch("balance_loss_bwd");
}
