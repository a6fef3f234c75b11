// Root-mean-square norms with the residual stream, forward and backward.  (No kernel
// of the reference, whose layers run transformers' GptOssDecoderLayer: residual adds
// and GptOssRMSNorm as separate elementwise passes.)
//
//   u = x,  or  post_weight * x * s_x,        s_v = 1 / sqrt(mean(v^2) + eps)
//   r = residual + scale * gate * u           (r = x where there is no residual)
//   h = weight * r * s_r
// and, with dr, dh the gradients that arrive at r and h,
//   g = dr + B(dh, r, weight, s_r),   B(d, v, w, s) = s (d w - v s^2 mean(d w v))
//   dresidual = g,  du = scale gate g,  dgate = scale sum g u  (over what the gate is shared by)
//   dx = du,  or  B(du, x, post_weight, s_x)
//   dweight = sum_rows dh r s_r,  dpost_weight = sum_rows du x s_x
//
// Everything between the tensors' types is fp32; h comes from r before its rounding
// (one rounding per output).  The backward reads r as it was stored, except where the
// weight's gradient is wanted and r is bf16: its sum over rows would be 1.45 bf16 roundings
// off instead of 1, so r is made again from x and the residual (REC: one more tensor
// read, 5 for 4, where neither norm nor gate needs x anyway).
//
// A row stays in registers from its loads to its stores, so each direction reads and
// writes every tensor once: HBM bounds both.  NW waves share a row, a lane holding CPL
// chunks of 8 consecutive elements:
//   without a post norm or gate: a wave alone up to H = 1024 (its reductions are shuffles,
//     no barrier; the backward from 512 rows on), else four waves to 4096, eight to 16384;
//   with one (FULL): the forward four waves to 4096, the backward eight, eight above.
// Rows may start at any element: 16-byte loads need no alignment here, and a row's last
// H % 8 elements come out of a load of its last 8.
//
// Measured, us (TB/s of the tensors read and written): 128000 x 2880 bf16 with a residual
// forward 494 to 513 (5.7 to 6.0), backward with dweight 732 to 760 (5.8 to 6.0; 640 without it),
// joining 5; 8192 x 2880 29 and 47; 3 x 1021 rows with post_weight and a gate 22 and 40; 1 row 2.5.
// A wave a row against four: 8192 x 512 forward 6.6 for 11.3, 300 rows 3.0 for 3.1, one
// row of 1024 2.8 for 2.7; at 2880 (six chunks a lane) 8192 rows 29.0 for 29.2, but 300
// rows 5.3 for 3.6.  Backward, 8192 x 960 24.5 for 32.8, 300 x 1024 8.4 for 8.0.  FULL has no
// wave a row: its forward would take, with launch, 12.1 for 22.2 (8192 x 512), 16.3 for 24.1
// (8192 x 1024), 59 for 181 (128000 x 64), 6.8 for 6.3 (300 x 1024).
//
// Column sums (dweight, dpost_weight, dgate): a lane adds up its columns over all its
// rows, the waves of a block are joined through LDS, each block writes one row of fp32
// partials, and a second launch adds the blocks' rows: fixed order, no atomics.  A gate's
// sums are over each group of rows that share it: some blocks per group, or, where there
// are more groups than blocks, groups that a block finishes by itself (OWN).
#include "af3_common.h"

namespace {

constexpr int kNormMinH = 8, kNormMaxH = 16384;
constexpr int kNormWaveRows = 512;  // rows from which a wave of the backward has a row of its own
// Blocks of the backward's row pass: 256 with a post norm or gate (eight waves a row) and for
// up to 1024 rows of several waves, else twice as many (of four waves, or of eight with a row
// each): more only add partials.  8192 x 2880 with 256, 512, 1024 blocks: four waves a row 73,
// 57, 62 us, eight (FULL) 66, 70, 78 (FULL with four, 130); 500 rows 11.2, 12.3, 13.1.
constexpr int kNormBwdBlocks = 256;
constexpr int64_t kNormGrid = 1 << 22;  // blocks per launch of the forward: a launch holds less than 2^32 threads

struct NormArgs {
  const void* x;
  int64_t ldx;
  const void* res;   // forward: residual; backward: r as stored
  int64_t ldr;
  const void* weight;
  const void* post;
  const void* gate;
  int w_f32, post_f32, gate_f32;
  int gate_cols;      // 0: no gate, 1: one value a row, else H
  int64_t gate_rows;  // rows that share a gate row
  float scale, eps;
  int64_t rows;
  int H;
  // forward
  int64_t row0;       // the launch's first row
  void* out_r;
  void* out_h;
  float* rstd;
  float* rstd_x;
  // backward
  const void* dr;
  int64_t lddr;
  const void* dh;
  int64_t lddh;
  const float* s_r;
  const float* s_x;
  void* dx;
  void* dres;
  float* part_w;     // [blocks][H] each, or null
  float* part_post;
  float* part_gate;
  float* gate_dots;  // [rows] fp32: a one-value gate's row sums
  void* dgate;       // a gate of x's own shape: its gradient, no sums
  int blocks_per_group;
  int64_t groups;    // OWN: of rows that share a gate row, and the gate's gradient
  void* dgate_sum;
};

// 8 elements at any address that is a multiple of the element's size, as fp32
__device__ __forceinline__ void n_unpack(const uint32_t (&w)[4], float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = af3_bf16_to_f32(w[i]);
    f[2 * i + 1] = af3_bf16_to_f32(w[i] >> 16);
  }
}

// chunk at element e of a row of H >= 8 elements; elements past the row are 0.  A chunk
// that the row ends in is read as the row's last 8 elements and shifted down.
__device__ __forceinline__ void n_words(const uint16_t* row, int e, int H, uint32_t (&w)[4]) {
  w[0] = w[1] = w[2] = w[3] = 0;
  if (e < H) {
    __builtin_memcpy(w, row + min(e, H - 8), 16);
    if (e + 8 > H) {
      const int s = 16 * (e + 8 - H);  // bits, 16 to 112
      uint64_t lo = w[0] | (uint64_t)w[1] << 32, hi = w[2] | (uint64_t)w[3] << 32;
      lo = s >= 64 ? hi >> (s - 64) : (lo >> s) | (hi << (64 - s));
      hi = s >= 64 ? 0 : hi >> s;
      w[0] = (uint32_t)lo, w[1] = (uint32_t)(lo >> 32), w[2] = (uint32_t)hi, w[3] = (uint32_t)(hi >> 32);
    }
  }
}
__device__ __forceinline__ void n_get(const uint16_t* row, int e, int H, float (&f)[8]) {
  uint32_t w[4];
  n_words(row, e, H, w);
  n_unpack(w, f);
}
__device__ __forceinline__ void n_get(const float* row, int e, int H, float (&f)[8]) {
  if (e < H) {
    __builtin_memcpy(f, row + min(e, H - 8), 32);
    if (e + 8 > H) {
      const int s = e + 8 - H;  // 1 to 7
#pragma unroll
      for (int k = 1; k < 8; k *= 2)
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = (s & k) ? (i + k < 8 ? f[i + k] : 0.f) : f[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
  }
}
__device__ __forceinline__ void n_get(const void* row, int f32, int64_t off, int e, int H, float (&f)[8]) {
  if (f32)
    n_get((const float*)row + off, e, H, f);
  else
    n_get((const uint16_t*)row + off, e, H, f);
}

// a chunk as loaded: bf16 pairs stay packed until they are used
template <class T>
struct NRaw {
  float f[8];
  __device__ __forceinline__ void load(const T* row, int e, int H) { n_get(row, e, H, f); }
  __device__ __forceinline__ void value(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f[i];
  }
};
template <>
struct NRaw<uint16_t> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const uint16_t* row, int e, int H) { n_words(row, e, H, w); }
  __device__ __forceinline__ void value(float (&v)[8]) const { n_unpack(w, v); }
};

template <class W>
__device__ __forceinline__ void n_put_tail(W* p, W (&w)[8], int n) {  // the first n < 8 words
  if (n & 4) {
    __builtin_memcpy(p, w, 4 * sizeof(W));
    p += 4;
#pragma unroll
    for (int i = 0; i < 3; ++i) w[i] = w[i + 4];
  }
  if (n & 2) {
    __builtin_memcpy(p, w, 2 * sizeof(W));
    p += 2;
    w[0] = w[2];
  }
  if (n & 1) *p = w[0];
}
__device__ __forceinline__ void n_set(uint16_t* row, int e, int H, const float (&f)[8]) {
  if (e + 8 <= H) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = af3_pack_bf16x2(f[2 * i], f[2 * i + 1]);
    __builtin_memcpy(row + e, w, 16);
  } else if (e < H) {
    uint16_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = (uint16_t)af3_f32_to_bf16(f[i]);
    n_put_tail(row + e, w, H - e);
  }
}
__device__ __forceinline__ void n_set(float* row, int e, int H, const float (&f)[8]) {
  if (e + 8 <= H) {
    __builtin_memcpy(row + e, f, 32);
  } else if (e < H) {
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = f[i];
    n_put_tail(row + e, w, H - e);
  }
}

template <int CTRL>
__device__ __forceinline__ float n_dpp(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xF, 0xF, true));
}

// sum over the NW waves of a row, every lane gets it.  turn: alternates between a
// kernel's sums, so that one barrier serves each.
template <int NW>
__device__ __forceinline__ float n_sum(float s, float (*lds)[NW > 1 ? NW : 1], int wave, int& turn) {
  s += n_dpp<0xB1>(s);   // lanes 1, 2, 4, 8 apart by row operations, 16 and 32 by shuffles
  s += n_dpp<0x4E>(s);
  s += n_dpp<0x141>(s);
  s += n_dpp<0x140>(s);
  s += __shfl_xor(s, 16);
  s += __shfl_xor(s, 32);
  if constexpr (NW > 1) {
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) lds[turn][wave] = s;
    // (a barrier for LDS alone: __syncthreads would also wait for the next row's loads)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    s = lds[turn][0];
#pragma unroll
    for (int w = 1; w < NW; ++w) s += lds[turn][w];
  }
  return s;
}

__device__ __forceinline__ float n_rstd(float sum, int H, float eps) { return 1.0f / sqrtf(sum / (float)H + eps); }

__device__ __forceinline__ float n_gate1(const NormArgs& a, int64_t grow) {
  return a.gate_f32 ? ((const float*)a.gate)[grow] : af3_bf16_to_f32(((const uint16_t*)a.gate)[grow]);
}

// RES: a residual; FULL: the norm of x and the gate, where they are given
template <class XT, class RT, int NW, int CPL, bool RES, bool FULL>
__global__ __launch_bounds__(NW == 8 ? 512 : 256) void norm_fwd_kernel(const NormArgs a) {
  constexpr int WPB = NW == 1 ? 4 : NW;
  __shared__ float lds[2][NW];
  int turn = 0;
  const int wave = threadIdx.x >> 6;
  const int64_t row = a.row0 + (NW == 1 ? (int64_t)blockIdx.x * WPB + wave : (int64_t)blockIdx.x);
  if (NW == 1 && row >= a.rows) return;
  const int t = NW == 1 ? (threadIdx.x & 63) : threadIdx.x;
  const int H = a.H;
  const XT* const x = (const XT*)a.x + row * a.ldx;
  float v[CPL][8], b[CPL][8];
#pragma unroll
  for (int c = 0; c < CPL; ++c) n_get(x, (c * 64 * NW + t) * 8, H, v[c]);
  if constexpr (RES) {
    const RT* const res = (const RT*)a.res + row * a.ldr;
#pragma unroll
    for (int c = 0; c < CPL; ++c) n_get(res, (c * 64 * NW + t) * 8, H, b[c]);
    if constexpr (FULL) {
      if (a.post) {
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < CPL; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) ss += v[c][i] * v[c][i];
        const float sx = n_rstd(n_sum<NW>(ss, lds, wave, turn), H, a.eps);
        if (a.rstd_x && t == 0) a.rstd_x[row] = sx;
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          float w[8];
          n_get(a.post, a.post_f32, 0, (c * 64 * NW + t) * 8, H, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[c][i] *= sx * w[i];
        }
      }
      if (a.gate_cols) {
        const int64_t grow = (uint32_t)row / (uint32_t)a.gate_rows;
        const float g1 = a.gate_cols == 1 ? n_gate1(a, grow) : 0.f;
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          float g[8];
          if (a.gate_cols > 1) n_get(a.gate, a.gate_f32, grow * H, (c * 64 * NW + t) * 8, H, g);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[c][i] *= a.gate_cols > 1 ? g[i] : g1;
        }
      }
    }
    RT* const out_r = (RT*)a.out_r + row * H;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] = b[c][i] + a.scale * v[c][i];
      n_set(out_r, (c * 64 * NW + t) * 8, H, v[c]);
    }
  }
  if (RES && !a.out_h) return;
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < CPL; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += v[c][i] * v[c][i];
  const float s = n_rstd(n_sum<NW>(ss, lds, wave, turn), H, a.eps);
  if (a.rstd && t == 0) a.rstd[row] = s;
  XT* const out_h = (XT*)a.out_h + row * H;
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    float w[8];
    n_get(a.weight, a.w_f32, 0, (c * 64 * NW + t) * 8, H, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] *= v[c][i] * s;
    n_set(out_h, (c * 64 * NW + t) * 8, H, w);
  }
}

// acc[CPL][8] of the block's waves -> one row of partials (NW == 1: the waves hold the
// same columns and are added in order; else each column has one owner)
template <int NW, int WPB, int CPL>
__device__ __forceinline__ void n_join(const float (&acc)[CPL][8], float* lds, int wave, int t, int H, float* out) {
  if constexpr (NW > 1) {
#pragma unroll
    for (int c = 0; c < CPL; ++c) n_set(out, (c * 64 * NW + t) * 8, H, acc[c]);
  } else {
    for (int w = 0; w < WPB; ++w) {
      __syncthreads();
      if (wave == w) {
#pragma unroll
        for (int c = 0; c < CPL; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) {  // (element 64 i + t of the chunk's 512: no bank conflicts)
            float* const p = lds + c * 512 + i * 64 + t;
            *p = w ? *p + acc[c][i] : acc[c][i];
          }
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < H; e += WPB * 64) {
      const int q = e & 511;
      out[e] = lds[(e >> 9) * 512 + (q & 7) * 64 + (q >> 3)];
    }
  }
}

typedef __attribute__((ext_vector_type(4))) float f32x4;

// One row of a backward with FULL and CPL chunks a lane, whose tensors would not fit in the
// registers beside the column sums: dh, r (x and the gate where r is made again) are read a
// second time, from the L2, after the first sum; du and x stay for the second.  Two of the
// column sums are in LDS: own[0] of post_weight, own[1] of the gate, a lane's own elements.
// 8192 x 16384 with post_weight: 537 us (kept whole it spilled, 3140).
template <class XT, class RT, int NW, int CPL, bool ACC, bool REC, int AC>
__device__ __forceinline__ void n_bwd_long(const NormArgs& a, int64_t row, int wave, int t, float (*sums)[NW], int& turn,
                                           float (&aw)[AC][8], f32x4 (*own)[ACC ? CPL : 1][2][ACC ? NW * 64 : 1]) {
  const int H = a.H;
  const int64_t grow = a.gate_cols ? (uint32_t)row / (uint32_t)a.gate_rows : 0;
  const float s_x = a.post ? a.s_x[row] : 1.f, g1 = a.gate_cols == 1 ? n_gate1(a, grow) : 1.f;
  const XT* const x_row = (const XT*)a.x + row * a.ldx;
  // chunk c's first element, opaque: its addresses in eight tensors are not kept over the rows
  auto at = [&](int c) __attribute__((always_inline)) {
    int e = (c * 64 * NW + t) * 8;
    asm volatile("" : "+v"(e));
    return e;
  };
  auto post = [&](int e, float (&w)[8]) __attribute__((always_inline)) {
    if (a.post) {
      n_get(a.post, a.post_f32, 0, e, H, w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = 1.f;
    }
  };
  auto gate = [&](int e, float (&w)[8]) __attribute__((always_inline)) {
    if (a.gate_cols > 1) {
      n_get(a.gate, a.gate_f32, grow * H, e, H, w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = g1;
    }
  };
  // r, from the residual as read and u's factors
  auto remake = [&](const float (&x)[8], const float (&p)[8], const float (&gt)[8], float (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float u = x[i];
      if (a.post) u *= s_x * p[i];
      if (a.gate_cols) u *= gt[i];
      v[i] += a.scale * u;
    }
  };
  float s = 0.f, m = 0.f;
  if (a.dh) {
    s = a.s_r[row];
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const int e = at(c);
      float d[8], v[8], w[8];
      n_get((const XT*)a.dh + row * a.lddh, e, H, d);
      n_get((const RT*)a.res + row * a.ldr, e, H, v);
      n_get(a.weight, a.w_f32, 0, e, H, w);
      if constexpr (REC) {
        float x[8], p[8], gt[8];
        n_get(x_row, e, H, x);
        post(e, p);
        gate(e, gt);
        remake(x, p, gt, v);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) dot += d[i] * w[i] * v[i];
    }
    m = n_sum<NW>(dot, sums, wave, turn) / (float)H * s * s;
  }
  float du[CPL][8];
  NRaw<XT> x_raw[CPL];
  float dot = 0.f, gdot = 0.f;
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int e = at(c);
    float x[8], p[8], gt[8], g[8];
    x_raw[c].load(x_row, e, H);
    x_raw[c].value(x);
    post(e, p);
    gate(e, gt);
    if (a.dr) {
      n_get((const RT*)a.dr + row * a.lddr, e, H, g);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = 0.f;
    }
    if (a.dh) {
      float d[8], v[8], w[8];
      n_get((const XT*)a.dh + row * a.lddh, e, H, d);
      n_get((const RT*)a.res + row * a.ldr, e, H, v);
      n_get(a.weight, a.w_f32, 0, e, H, w);
      if constexpr (REC) remake(x, p, gt, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (ACC) aw[c][i] += d[i] * (v[i] * s);
        g[i] += s * (d[i] * w[i] - v[i] * m);
      }
    }
    if (a.dres) n_set((RT*)a.dres + row * H, e, H, g);
    float gg[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      gg[i] = a.scale * g[i] * (x[i] * s_x * p[i]);  // the gate's gradient
      gdot += gg[i];
      const float dgu = a.scale * gt[i] * g[i];
      if constexpr (ACC) {
        own[0][c][i / 4][t][i % 4] += dgu * (x[i] * s_x);
        own[1][c][i / 4][t][i % 4] += gg[i];
      }
      du[c][i] = dgu * p[i];
      dot += du[c][i] * x[i];
    }
    if (a.dgate) {
      if (a.gate_f32)
        n_set((float*)a.dgate + row * H, e, H, gg);
      else
        n_set((uint16_t*)a.dgate + row * H, e, H, gg);
    }
  }
  if (a.gate_dots) {
    const float sum = n_sum<NW>(gdot, sums, wave, turn);
    if (t == 0) a.gate_dots[row] = sum;
  }
  if (a.post) {  // (du alone without a norm of x: an infinite x must not meet a 0)
    const float m_x = n_sum<NW>(dot, sums, wave, turn) / (float)H * s_x * s_x;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      float x[8];
      x_raw[c].value(x);
#pragma unroll
      for (int i = 0; i < 8; ++i) du[c][i] = s_x * (du[c][i] - x[i] * m_x);
    }
  }
  if (a.dx) {
#pragma unroll
    for (int c = 0; c < CPL; ++c) n_set((XT*)a.dx + row * H, at(c), H, du[c]);
  }
}

// ACC: some column sum is wanted; REC: a.res is the residual, and r is made of it and x; OWN: a
// block has whole groups of the gate, one after the other, and writes their sums itself (a kernel of
// its own: the test after each row costs the others 3 to 5%)
template <class XT, class RT, int NW, int CPL, bool RES, bool FULL, bool ACC, bool REC, bool OWN>
__global__ __launch_bounds__(NW == 4 ? 256 : 512) void norm_bwd_kernel(const NormArgs a) {
  constexpr int WPB = NW == 1 ? 8 : NW;
  constexpr int AC = ACC ? CPL : 1;
  __shared__ float sums[2][NW];
  __shared__ float lds[(ACC && NW == 1) ? CPL * 512 : 1];
  constexpr bool LONG = FULL && CPL > 2;
  __shared__ f32x4 own[LONG && ACC ? 2 : 1][LONG && ACC ? CPL : 1][2][LONG && ACC ? NW * 64 : 1];
  int turn = 0;
  const int wave = threadIdx.x >> 6;
  int t = NW == 1 ? (threadIdx.x & 63) : threadIdx.x;
  const int H = a.H;
  // the block's group: the rows that share a gate row (one group of all rows without column sums of a gate)
  const int64_t per = a.part_gate ? a.gate_rows : a.rows;
  const int64_t group = blockIdx.x / a.blocks_per_group;
  int64_t first = group * per + (int64_t)(blockIdx.x % a.blocks_per_group) * (NW == 1 ? WPB : 1) + (NW == 1 ? wave : 0);
  int64_t last = min(group * per + per, a.rows);
  int64_t step = (int64_t)a.blocks_per_group * (NW == 1 ? WPB : 1);
  int64_t group_end = 0;  // of the group that the block is in
  if constexpr (OWN) {
    first = (int64_t)blockIdx.x * a.groups / gridDim.x * a.gate_rows;
    last = min(((int64_t)blockIdx.x + 1) * a.groups / gridDim.x * a.gate_rows, a.rows);
    step = 1;
    group_end = first + a.gate_rows;
  }
  // whether a group's rows end with `row`, whose gradients are in the block's sums
  auto ends = [&](int64_t row) {
    if (row + 1 != group_end && row + 1 != last) return false;
    group_end += a.gate_rows;
    return true;
  };
  auto put_group = [&](int64_t row, int c, const float (&sum)[8]) {
    const int64_t at = (int64_t)((uint32_t)row / (uint32_t)a.gate_rows) * H;
    if (a.gate_f32)
      n_set((float*)a.dgate_sum + at, (c * 64 * NW + t) * 8, H, sum);
    else
      n_set((uint16_t*)a.dgate_sum + at, (c * 64 * NW + t) * 8, H, sum);
  };
  float aw[AC][8], ap[FULL ? AC : 1][8], ag[FULL ? AC : 1][8];
  if constexpr (ACC) {
#pragma unroll
    for (int c = 0; c < CPL; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        aw[c][i] = 0.f;
        if constexpr (FULL) ap[c][i] = ag[c][i] = 0.f;
      }
  }
  if constexpr (LONG) {
    if constexpr (ACC) {
#pragma unroll
      for (int j = 0; j < 4 * CPL; ++j) own[j / (2 * CPL)][j / 2 % CPL][j % 2][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int64_t row = first; row < last; row += step) {
      n_bwd_long<XT, RT, NW, CPL, ACC, REC>(a, row, wave, t, sums, turn, aw, own);
      if constexpr (OWN) {
        if (ends(row)) {
#pragma unroll 1
          for (int c = 0; c < CPL; ++c) {
            float g[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] = own[1][c][i / 4][t][i % 4];
            own[1][c][0][t] = own[1][c][1][t] = f32x4{0.f, 0.f, 0.f, 0.f};
            put_group(row, c, g);
          }
        }
      }
    }
    if constexpr (ACC) {
#pragma unroll
      for (int c = 0; c < CPL; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) ap[c][i] = own[0][c][i / 4][t][i % 4], ag[c][i] = own[1][c][i / 4][t][i % 4];
    }
  } else {
    // a row's loads, made while the row before it is worked on
    NRaw<RT> r_dr[CPL], r_r[CPL];
    constexpr bool X = FULL || REC;
    NRaw<XT> r_dh[CPL], r_x[X ? CPL : 1];
    float r_gate[FULL ? CPL : 1][8];
    float r_s = 0.f, r_sx = 1.f, r_g1 = 1.f;
    const bool has_dr = RES && a.dr, has_dh = !RES || a.dh;
    auto fetch = [&](int64_t row) {
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        const int e = (c * 64 * NW + t) * 8;
        if (has_dr) r_dr[c].load((const RT*)a.dr + row * a.lddr, e, H);
        if (has_dh) r_dh[c].load((const XT*)a.dh + row * a.lddh, e, H);
        if (has_dh) r_r[c].load((const RT*)a.res + row * a.ldr, e, H);
        if constexpr (X) r_x[c].load((const XT*)a.x + row * a.ldx, e, H);
      }
      if (has_dh) r_s = a.s_r[row];
      if constexpr (FULL) {
        if (a.post) r_sx = a.s_x[row];
        if (a.gate_cols) {
          const uint32_t grow = (uint32_t)row / (uint32_t)a.gate_rows;
          if (a.gate_cols == 1) {
            r_g1 = n_gate1(a, grow);
          } else {
#pragma unroll
            for (int c = 0; c < CPL; ++c)
              n_get(a.gate, a.gate_f32, (int64_t)grow * H, (c * 64 * NW + t) * 8, H, r_gate[c]);
          }
        }
      }
    };
    // (where the registers of two rows would not fit, a row's loads are its own, the weights' too)
    constexpr bool AHEAD = CPL * (FULL ? 2 : 1) <= 2;
    float w_h[AHEAD ? CPL : 1][8], w_post[FULL && AHEAD ? CPL : 1][8];
    if constexpr (AHEAD) {
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        const int e = (c * 64 * NW + t) * 8;
        if (has_dh) n_get(a.weight, a.w_f32, 0, e, H, w_h[c]);
        if constexpr (FULL) {
          if (a.post) n_get(a.post, a.post_f32, 0, e, H, w_post[c]);
        }
      }
    }
    if (AHEAD && first < last) fetch(first);
    for (int64_t row = first; row < last; row += step) {
      if (!AHEAD) {
        asm volatile("" : "+v"(t));  // (opaque: the addresses in eight tensors are not kept over the rows)
        fetch(row);
      }
      float g[CPL][8];  // the gradient of r
      float d[CPL][8], v[CPL][8], x[X ? CPL : 1][8], gate[FULL ? CPL : 1][8];
      const float s_r = r_s, s_x = r_sx, g1 = r_g1;
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        if (has_dr) {
          r_dr[c].value(g[c]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) g[c][i] = 0.f;
        }
        if (has_dh) {
          r_dh[c].value(d[c]);
          r_r[c].value(v[c]);
        }
        if constexpr (X) r_x[c].value(x[c]);
        if constexpr (FULL) {
#pragma unroll
          for (int i = 0; i < 8; ++i) gate[c][i] = r_gate[c][i];
        }
      }
      if constexpr (REC) {
        if (has_dh) {
#pragma unroll
          for (int c = 0; c < CPL; ++c) {
            float w[8];
            if constexpr (FULL && AHEAD) {
#pragma unroll
              for (int i = 0; i < 8; ++i) w[i] = w_post[c][i];
            } else if constexpr (FULL) {
              if (a.post) n_get(a.post, a.post_f32, 0, (c * 64 * NW + t) * 8, H, w);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float u = x[c][i];
              if constexpr (FULL) {
                if (a.post) u *= s_x * w[i];
                if (a.gate_cols) u *= a.gate_cols > 1 ? gate[c][i] : g1;
              }
              v[c][i] += a.scale * u;
            }
          }
        }
      }
      if (AHEAD && row + step < last) fetch(row + step);
      if (has_dh) {
        const float s = s_r;
        float dot = 0.f;
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          float w[8];
          if constexpr (AHEAD) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = w_h[c][i];
          } else {
            n_get(a.weight, a.w_f32, 0, (c * 64 * NW + t) * 8, H, w);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if constexpr (ACC) aw[c][i] += d[c][i] * (v[c][i] * s);
            d[c][i] *= w[i];
            dot += d[c][i] * v[c][i];
          }
        }
        const float m = n_sum<NW>(dot, sums, wave, turn) / (float)H * s * s;
#pragma unroll
        for (int c = 0; c < CPL; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) g[c][i] += s * (d[c][i] - v[c][i] * m);
      }
      if (a.dres) {
        RT* const dres = (RT*)a.dres + row * H;
#pragma unroll
        for (int c = 0; c < CPL; ++c) n_set(dres, (c * 64 * NW + t) * 8, H, g[c]);
      }
      if constexpr (!RES) continue;
      if constexpr (FULL) {
        const float s = s_x;
        float dot = 0.f, gdot = 0.f;
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          const int e = (c * 64 * NW + t) * 8;
          float w[8], gg[8];
          if constexpr (AHEAD) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = w_post[c][i];
          } else {
            if (a.post) n_get(a.post, a.post_f32, 0, e, H, w);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float wi = a.post ? w[i] : 1.f;
            const float gi = a.gate_cols > 1 ? gate[c][i] : g1;
            const float gu = a.scale * g[c][i] * (x[c][i] * s * wi);  // the gate's gradient
            gdot += gu;
            gg[i] = gu;
            if constexpr (ACC) ag[c][i] += gu;
            const float du = a.scale * gi * g[c][i];
            if constexpr (ACC) ap[c][i] += du * (x[c][i] * s);
            g[c][i] = du * wi;
            dot += g[c][i] * x[c][i];
          }
          if (a.dgate) {
            if (a.gate_f32)
              n_set((float*)a.dgate + row * H, e, H, gg);
            else
              n_set((uint16_t*)a.dgate + row * H, e, H, gg);
          }
        }
        if (a.gate_dots) {
          const float sum = n_sum<NW>(gdot, sums, wave, turn);
          if (t == 0) a.gate_dots[row] = sum;
        }
        if (a.post) {
          const float m = n_sum<NW>(dot, sums, wave, turn) / (float)H * s * s;
#pragma unroll
          for (int c = 0; c < CPL; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) g[c][i] = s * (g[c][i] - x[c][i] * m);
        }
      } else {
#pragma unroll
        for (int c = 0; c < CPL; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) g[c][i] *= a.scale;
      }
      if (a.dx) {
        XT* const dx = (XT*)a.dx + row * H;
#pragma unroll
        for (int c = 0; c < CPL; ++c) n_set(dx, (c * 64 * NW + t) * 8, H, g[c]);
      }
      if constexpr (OWN) {
        if (ends(row)) {
#pragma unroll
          for (int c = 0; c < CPL; ++c) {
            put_group(row, c, ag[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) ag[c][i] = 0.f;
          }
        }
      }
    }
  }
  if constexpr (ACC) {
    const int64_t at = (int64_t)blockIdx.x * H;
    if (a.part_w) n_join<NW, WPB>(aw, lds, wave, t, H, a.part_w + at);
    if constexpr (FULL) {
      if (a.part_post) n_join<NW, WPB>(ap, lds, wave, t, H, a.part_post + at);
      if (a.part_gate) n_join<NW, WPB>(ag, lds, wave, t, H, a.part_gate + at);
    }
  }
}

// columns of partials -> gradients, kJoinCols a block: of weight, post weight, then the gate's groups
struct JoinArgs {
  const float* part[3];
  void* out[3];
  int f32[3];
  int64_t blocks;
  int blocks_per_group;
  int H;
};
constexpr int kJoinCols = 16, kJoinRows = 64;  // 2880 columns: 180 blocks (45 of 64 columns took 11 us, these 5)

__global__ __launch_bounds__(kJoinCols* kJoinRows) void norm_join_kernel(const JoinArgs a) {
  __shared__ float lds[kJoinRows][kJoinCols];
  const unsigned ncb = (unsigned)af3_cdiv(a.H, kJoinCols), what = blockIdx.x / ncb;
  const int which = (int)min(what, 2u);
  const float* const part = a.part[which];
  if (!part) return;
  const int64_t group = which == 2 ? what - 2 : 0;
  const int64_t begin = which == 2 ? group * a.blocks_per_group : 0;
  const int64_t end = which == 2 ? begin + a.blocks_per_group : a.blocks;
  const int c = threadIdx.x % kJoinCols, w = threadIdx.x / kJoinCols;
  const int64_t col = (int64_t)(blockIdx.x % ncb) * kJoinCols + c;
  float s = 0.f;
  if (col < a.H)
#pragma unroll 4
    for (int64_t b = begin + w; b < end; b += kJoinRows) s += part[b * a.H + col];
  lds[w][c] = s;
  __syncthreads();
#pragma unroll
  for (int n = kJoinRows / 2; n > 1; n /= 2) {  // (pairs, the last two below)
    if (w < n) lds[w][c] = s = s + lds[w + n][c];
    __syncthreads();
  }
  if (w || col >= a.H) return;
  s += lds[1][c];
  const int64_t at = group * a.H + col;
  if (a.f32[which])
    ((float*)a.out[which])[at] = s;
  else
    ((uint16_t*)a.out[which])[at] = (uint16_t)af3_f32_to_bf16(s);
}

// a one-value gate's gradient: group g sums dots[g * per .. ) (a block at a time)
__global__ __launch_bounds__(256) void norm_gate_dots_kernel(const float* dots, int64_t rows, int64_t per,
                                                             int64_t groups, void* out, int f32) {
  __shared__ float lds[2][4];
  int turn = 0;
  for (int64_t g = blockIdx.x; g < groups; g += gridDim.x) {
    const int64_t end = min(g * per + per, rows);
    float s = 0.f;
    for (int64_t i = g * per + threadIdx.x; i < end; i += 256) s += dots[i];
    s = n_sum<4>(s, lds, threadIdx.x >> 6, turn);
    if (threadIdx.x == 0) {
      if (f32)
        ((float*)out)[g] = s;
      else
        ((uint16_t*)out)[g] = (uint16_t)af3_f32_to_bf16(s);
    }
  }
}

// the same with a gate value per row: no sums
__global__ __launch_bounds__(256) void norm_gate_rows_kernel(const float* dots, int64_t rows, void* out, int f32) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows) return;
  if (f32)
    ((float*)out)[i] = dots[i];
  else
    ((uint16_t*)out)[i] = (uint16_t)af3_f32_to_bf16(dots[i]);
}

// whether the backward gives a wave a row of its own
bool norm_bwd_wave_row(int64_t rows, int H, bool full) { return !full && H <= 64 * 8 * 2 && rows >= kNormWaveRows; }

template <class XT, class RT, bool RES, bool FULL>
void norm_fwd_launch(NormArgs a, hipStream_t st) {
  const int chunks = (int)af3_cdiv(a.H, 8);
#define AF3_NF(NW, CPL)                                                                                           \
  do {                                                                                                            \
    constexpr int RPB = NW == 1 ? 4 : 1;                                                                          \
    for (a.row0 = 0; a.row0 < a.rows; a.row0 += kNormGrid * RPB) {                                                \
      const int64_t left = af3_cdiv(a.rows - a.row0, RPB);                                                        \
      const dim3 grid((unsigned)(left < kNormGrid ? left : kNormGrid));                                           \
      hipLaunchKernelGGL((norm_fwd_kernel<XT, RT, NW, CPL, RES, FULL>), grid, dim3(NW == 8 ? 512 : 256), 0, st, a); \
    }                                                                                                             \
    return;                                                                                                       \
  } while (0)
  if constexpr (!FULL) if (chunks <= 64 * 2) AF3_NF(1, 2);
  if (chunks <= 64 * 8) AF3_NF(4, 2);
  if (chunks <= 64 * 16) AF3_NF(8, 2);
  AF3_NF(8, 4);
#undef AF3_NF
}

template <class XT, class RT, bool RES, bool FULL, bool ACC, bool REC>
void norm_bwd_launch(const NormArgs& a, unsigned blocks, hipStream_t st) {
  const int chunks = (int)af3_cdiv(a.H, 8);
#define AF3_NB(NW, CPL)                                                                                           \
  do {                                                                                                            \
    const dim3 block(NW == 4 ? 256 : 512);                                                                         \
    if constexpr (FULL && ACC) {                                                                                  \
      if (a.dgate_sum) {                                                                                          \
        hipLaunchKernelGGL((norm_bwd_kernel<XT, RT, NW, CPL, RES, FULL, ACC, REC, true>), dim3(blocks), block, 0, st, a); \
        return;                                                                                                   \
      }                                                                                                           \
    }                                                                                                             \
    hipLaunchKernelGGL((norm_bwd_kernel<XT, RT, NW, CPL, RES, FULL, ACC, REC, false>), dim3(blocks), block, 0, st, a); \
    return;                                                                                                       \
  } while (0)
  if constexpr (!FULL) if (norm_bwd_wave_row(a.rows, a.H, FULL)) AF3_NB(1, 2);
  if constexpr (FULL) {
    if (chunks <= 64 * 8) AF3_NB(8, 1);
  } else {
    if (chunks <= 64 * 8) AF3_NB(4, 2);
  }
  if (chunks <= 64 * 16) AF3_NB(8, 2);
  AF3_NB(8, 4);
#undef AF3_NB
}

// blocks of the backward's row pass and where its partials lie
struct NormPlan {
  int64_t groups, blocks;
  int blocks_per_group;
  int64_t off_w, off_post, off_gate, off_dots, bytes;
  bool own_groups;  // blocks have whole groups of a gate
};

NormPlan norm_plan(int64_t rows, int H, int gate_cols, int64_t gate_rows, bool full, int want_w, int want_post, int want_gate) {
  NormPlan p;
  bool sums = want_gate && gate_cols > 1 && gate_rows > 1;  // of a gate row over its group
  p.groups = sums ? af3_cdiv(rows, gate_rows) : 1;
  const bool wave_row = norm_bwd_wave_row(rows, H, full);
  const int64_t total = full || (!wave_row && rows < 4 * kNormBwdBlocks) ? kNormBwdBlocks : 2 * kNormBwdBlocks;
  // More groups than blocks: a block takes whole ones and writes their sums, so partials stay a row per block.
  // A block and a row of partials for each group instead, us: 8000 x 2 x 2880 bf16 4370 for 181, 300 x 10 with a
  // post norm and an fp32 stream 204 for 61, 257 x 100 608 for 500.
  p.own_groups = p.groups > total;
  if (p.own_groups) sums = false;
  const int64_t per = sums ? gate_rows : rows;
  const int64_t units = wave_row ? af3_cdiv(per, 8) : per;  // row steps of one block
  const int64_t bpg = p.own_groups ? total : total / p.groups;  // (not rounded up: a block too many is a second round)
  p.blocks_per_group = (int)(bpg < units ? bpg : units);
  p.blocks = p.own_groups ? total : p.groups * p.blocks_per_group;
  const int64_t part = p.blocks * H * 4;
  p.off_w = 0;
  p.off_post = p.off_w + (want_w ? part : 0);
  p.off_gate = p.off_post + (want_post ? part : 0);
  p.off_dots = p.off_gate + (sums ? part : 0);
  p.bytes = p.off_dots + (want_gate && gate_cols == 1 ? rows * 4 : 0);
  return p;
}

int norm_check(const char* who, int64_t rows, int H, int gate_cols, int64_t gate_rows, float eps) {
  AF3_REQUIRE(rows >= 0 && H > 0, "%s: bad sizes", who);
  AF3_REQUIRE(H >= kNormMinH && H <= kNormMaxH, "%s: %d channels (%d to %d)", who, H, kNormMinH, kNormMaxH);
  AF3_REQUIRE(rows < (int64_t)1 << 31, "%s: too many rows", who);
  AF3_REQUIRE(eps >= 0.f, "%s: eps must not be negative", who);
  AF3_REQUIRE(gate_cols == 0 || ((gate_cols == 1 || gate_cols == H) && gate_rows > 0 && gate_rows < (int64_t)1 << 32),
              "%s: a gate has 1 or H columns, and rows that share each of its rows", who);
  return 0;
}

}  // namespace

extern "C" int af3_residual_norm_fwd(const void* x, int x_f32, int64_t ldx, const void* residual, int r_f32,
                                     int64_t ldr, const void* weight, int w_f32, const void* post_weight, int post_f32,
                                     const void* gate, int gate_f32, int gate_cols, int64_t gate_rows, float scale,
                                     float eps, int64_t rows, int H, void* out_r, void* out_h, float* rstd,
                                     float* rstd_x, void* stream_) {
  const int rc = norm_check("residual_norm_fwd", rows, H, gate_cols, gate_rows, eps);
  if (rc) return rc;
  if (rows == 0) return 0;
  AF3_REQUIRE(x, "residual_norm_fwd: null pointer");
  AF3_REQUIRE((out_h != nullptr) == (weight != nullptr), "residual_norm_fwd: weight and out_h go together");
  AF3_REQUIRE(residual ? out_r != nullptr : (weight && !out_r && !post_weight && !gate_cols),
              "residual_norm_fwd: out_r goes with a residual, post_weight and gate only there");
  AF3_REQUIRE(!gate_cols || gate, "residual_norm_fwd: null gate");
  AF3_REQUIRE(!residual || r_f32 || !x_f32, "residual_norm_fwd: a bf16 residual needs a bf16 x");
  NormArgs a = {};
  a.x = x, a.ldx = ldx, a.res = residual, a.ldr = ldr, a.weight = weight, a.w_f32 = w_f32;
  a.post = post_weight, a.post_f32 = post_f32, a.gate = gate, a.gate_f32 = gate_f32, a.gate_cols = gate_cols;
  a.gate_rows = gate_rows, a.scale = scale, a.eps = eps, a.rows = rows, a.H = H;
  a.out_r = out_r, a.out_h = out_h, a.rstd = rstd, a.rstd_x = rstd_x;
  hipStream_t st = (hipStream_t)stream_;
  const bool full = post_weight || gate_cols;
  if (!residual) {
    if (x_f32)
      norm_fwd_launch<float, float, false, false>(a, st);
    else
      norm_fwd_launch<uint16_t, uint16_t, false, false>(a, st);
  } else if (x_f32) {
    if (full)
      norm_fwd_launch<float, float, true, true>(a, st);
    else
      norm_fwd_launch<float, float, true, false>(a, st);
  } else if (r_f32) {
    if (full)
      norm_fwd_launch<uint16_t, float, true, true>(a, st);
    else
      norm_fwd_launch<uint16_t, float, true, false>(a, st);
  } else {
    if (full)
      norm_fwd_launch<uint16_t, uint16_t, true, true>(a, st);
    else
      norm_fwd_launch<uint16_t, uint16_t, true, false>(a, st);
  }
  return af3::check_launch("residual_norm_fwd");
}

extern "C" size_t af3_residual_norm_bwd_workspace_bytes(int64_t rows, int H, int full, int gate_cols, int64_t gate_rows,
                                                        int want_w, int want_post, int want_gate) {
  if (rows <= 0 || H < kNormMinH || H > kNormMaxH || (gate_cols && gate_rows <= 0)) return 0;
  return (size_t)norm_plan(rows, H, gate_cols, gate_rows, full != 0, want_w, want_post, want_gate).bytes;
}

namespace {
template <class XT, class RT, bool RES, bool FULL>
void norm_bwd_pick(const NormArgs& a, unsigned blocks, bool acc, hipStream_t st) {
  if (acc)
    norm_bwd_launch<XT, RT, RES, FULL, true, false>(a, blocks, st);
  else
    norm_bwd_launch<XT, RT, RES, FULL, false, false>(a, blocks, st);
}
}  // namespace

extern "C" int af3_residual_norm_bwd(const void* dr, int64_t lddr, const void* dh, int64_t lddh, const void* r, int r_f32,
                                     int r_again, int64_t ldr, const void* x, int x_f32, int64_t ldx, const float* rstd,
                                     const float* rstd_x, const void* weight, int w_f32, const void* post_weight,
                                     int post_f32, const void* gate, int gate_f32, int gate_cols, int64_t gate_rows,
                                     float scale, int has_residual, int64_t rows, int H, void* dx, void* dresidual,
                                     void* dweight, void* dpost, void* dgate, void* workspace, size_t ws_bytes,
                                     void* stream_) {
  const int rc = norm_check("residual_norm_bwd", rows, H, gate_cols, gate_rows, 0.f);
  if (rc) return rc;
  AF3_REQUIRE(has_residual || (dh && (dresidual || dweight) && !dx && !dr && !post_weight && !gate_cols),
              "residual_norm_bwd: without a residual, x's gradient is dresidual, and only dh arrives");
  AF3_REQUIRE(!dpost || post_weight, "residual_norm_bwd: dpost without post_weight");
  AF3_REQUIRE(!dgate || gate_cols, "residual_norm_bwd: dgate without a gate");
  AF3_REQUIRE(!has_residual || r_f32 || !x_f32, "residual_norm_bwd: a bf16 residual needs a bf16 x");
  AF3_REQUIRE(!dweight || dh, "residual_norm_bwd: dweight without dh");
  if (rows == 0) return 0;
  const bool full = has_residual && (post_weight || gate_cols);
  AF3_REQUIRE(!dh || (r && rstd && weight), "residual_norm_bwd: dh needs r, rstd and weight");
  AF3_REQUIRE(dr || dh, "residual_norm_bwd: no gradient arrives");
  AF3_REQUIRE(!r_again || (has_residual && !r_f32 && !x_f32 && x && dh && dweight),
              "residual_norm_bwd: r_again goes with a bf16 residual, x, dh and dweight");
  AF3_REQUIRE(!full || (x && (!post_weight || rstd_x) && (!gate_cols || gate)), "residual_norm_bwd: null pointer");
  const NormPlan p = norm_plan(rows, H, gate_cols, gate_rows, full, dweight != nullptr, dpost != nullptr, dgate != nullptr);
  AF3_REQUIRE((size_t)p.bytes <= ws_bytes && (p.bytes == 0 || workspace), "residual_norm_bwd: workspace too small");
  hipStream_t st = (hipStream_t)stream_;
  uint8_t* const ws = (uint8_t*)workspace;
  const bool gate_sums = dgate && gate_cols > 1 && gate_rows > 1 && !p.own_groups;
  NormArgs a = {};
  a.x = x, a.ldx = ldx, a.res = r, a.ldr = ldr, a.weight = weight, a.w_f32 = w_f32;
  a.post = post_weight, a.post_f32 = post_f32, a.gate = gate, a.gate_f32 = gate_f32, a.gate_cols = gate_cols;
  a.gate_rows = gate_rows, a.scale = scale, a.rows = rows, a.H = H;
  a.dr = dr, a.lddr = lddr, a.dh = dh, a.lddh = lddh, a.s_r = rstd, a.s_x = rstd_x, a.dx = dx, a.dres = dresidual;
  a.part_w = dweight ? (float*)(ws + p.off_w) : nullptr;
  a.part_post = dpost ? (float*)(ws + p.off_post) : nullptr;
  a.part_gate = gate_sums ? (float*)(ws + p.off_gate) : nullptr;
  a.dgate = dgate && gate_cols > 1 && gate_rows == 1 ? dgate : nullptr;
  a.gate_dots = dgate && gate_cols == 1 ? (float*)(ws + p.off_dots) : nullptr;
  a.blocks_per_group = p.blocks_per_group;
  if (p.own_groups) a.groups = p.groups, a.dgate_sum = dgate;
  const bool join = a.part_w || a.part_post || a.part_gate, acc = join || a.dgate_sum;
  const unsigned blocks = (unsigned)p.blocks;
  if (!has_residual) {
    if (x_f32)
      norm_bwd_pick<float, float, false, false>(a, blocks, acc, st);
    else
      norm_bwd_pick<uint16_t, uint16_t, false, false>(a, blocks, acc, st);
  } else if (x_f32) {
    if (full)
      norm_bwd_pick<float, float, true, true>(a, blocks, acc, st);
    else
      norm_bwd_pick<float, float, true, false>(a, blocks, acc, st);
  } else if (r_f32) {
    if (full)
      norm_bwd_pick<uint16_t, float, true, true>(a, blocks, acc, st);
    else
      norm_bwd_pick<uint16_t, float, true, false>(a, blocks, acc, st);
  } else if (r_again) {
    if (full)
      norm_bwd_launch<uint16_t, uint16_t, true, true, true, true>(a, blocks, st);
    else
      norm_bwd_launch<uint16_t, uint16_t, true, false, true, true>(a, blocks, st);
  } else {
    if (full)
      norm_bwd_pick<uint16_t, uint16_t, true, true>(a, blocks, acc, st);
    else
      norm_bwd_pick<uint16_t, uint16_t, true, false>(a, blocks, acc, st);
  }
  int e = af3::check_launch("residual_norm_bwd");
  if (e) return e;
  if (join) {
    JoinArgs j = {};
    j.part[0] = a.part_w, j.part[1] = a.part_post, j.part[2] = a.part_gate;
    j.out[0] = dweight, j.out[1] = dpost, j.out[2] = dgate;
    j.f32[0] = w_f32, j.f32[1] = post_f32, j.f32[2] = gate_f32;
    j.blocks = p.blocks, j.blocks_per_group = p.blocks_per_group, j.H = H;
    const int64_t what = 2 + (gate_sums ? p.groups : 0);
    hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)(af3_cdiv(H, kJoinCols) * what)), dim3(kJoinCols * kJoinRows), 0,
                       st, j);
  }
  if (a.gate_dots) {
    if (gate_rows == 1)
      hipLaunchKernelGGL(norm_gate_rows_kernel, dim3((unsigned)af3_cdiv(rows, 256)), dim3(256), 0, st, a.gate_dots,
                         rows, dgate, gate_f32);
    else {
      const int64_t groups = af3_cdiv(rows, gate_rows);
      hipLaunchKernelGGL(norm_gate_dots_kernel, dim3((unsigned)(groups < kNormGrid ? groups : kNormGrid)), dim3(256), 0, st,
                         a.gate_dots, rows, gate_rows, groups, dgate, gate_f32);
    }
  }
  return af3::check_launch("residual_norm_bwd: sums");
}
