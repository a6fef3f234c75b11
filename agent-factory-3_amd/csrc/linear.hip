// Matrix products with a bias, an activation and a residual in the epilogue, and the
// products of their backward.  (The reference's attention projections are nn.Linear
// calls into a library, and the residual adds passes of their own.)
//
//   z = x W^T + b,  y = act(z) + residual
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum_rows dz,  dresidual = dy
//
// One kernel makes the three products, out[M][N] = sum_k P[m][k] Q[n][k], each operand
// stored with k contiguous (x, W of the forward) or, PT / QT, with its own index
// contiguous (W of dx; dz and x of dW), so nothing is transposed in memory.
//
// lin_kernel: a block of 4 waves (2 x 2) makes BM x BN of the output in 64-deep
// k-steps.  Both operands of a k-step go global -> LDS (16-byte copies) into one of ST
// stages while another is used; a wave's BM/2 x BN/2 part is TM x TN products
// v_mfma_f32_32x32x16_bf16.  With 128 x 128 per wave a fragment read from LDS is used
// four times: 64 bytes per clock and CU where the copies take another 32, under what
// the LDS gives (147; 111 for transposing reads); with 128 x 64 (eight waves) both would
// saturate it.  One wave per SIMD hides nothing by itself, so the loop is a fixed
// schedule: fragments of the next 16 k are read between the products of this one, one
// instruction per product, the k-step's last products run after the next barrier, and
// a later stage's copies are issued in the first half of a step (all of them in the first
// quarter, or spread over the whole, 3% slower).
// Fragments: lane (r, h) = (lane % 32, lane / 32) feeds row r, k = 16 s + 8 h + (0..7) of
// sub-step s.  k contiguous: one 16-byte read.  Else two transposing reads of 4 k each.
// LDS chunks of 16 bytes are XOR-swizzled so that either reads without bank conflicts.
// Q is the matrix unit's first operand, so a lane ends up with rows of the output, 4
// consecutive columns at a time; the epilogue turns them through LDS (32 rows of a wave
// at a time, fp32) into 16-byte accesses and rounds once.  Blocks stay for several tiles:
// the next one's first copies are issued before the last k-step of this, and this one's
// stores drain under the next's first.
//
// Measured (library product of the same operands in brackets), us: 8192 x 4096 from 2880
// 157 (140), 8192 x 2880 from 4096 with W as stored 168 (193), 16384 x 2880 from 4096 329
// (285), with bias and residual 335 (and an add of 55), 16384 x 4096 from 2880 with W as
// stored 309 (308), 2880 x 4096 from 16384 rows 326 (446); 1021 x 2880 from 2880 24 (26),
// 8192 x 512 from 2880 28 (29).  The large ones run 1.17 to 1.29 PFLOP/s: 73% of the CUs' busy
// cycles issue products, at a clock of 1.75 GHz (2.4 without load), so the card's power bounds
// them.  Products of 16 x 16 x 32 (3 to 5% less time in 128 x 128 tiles) leave the compiler
// moving accumulators between register files.
//
// Few tiles and a long k (dW of narrow layers): blocks share a tile's k-steps and write
// fp32 partials, which lin_join_kernel adds in order and gives the epilogue.
// Up to 32 rows: lin_skinny_kernel streams W once through registers.
#include "af3_common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef const __attribute__((address_space(3))) af3_bf16x8 lds_frag;

enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4 };

struct LinEpi {
  const void* bias;
  int bias_f32;
  int act;
  const uint16_t* res;
  int64_t ldr;
  uint16_t* y;  // [M][N]
  uint16_t* z;  // [M][N] before the activation, or null
};

struct LinArgs {
  const uint16_t* p;
  int64_t ldp;
  const uint16_t* q;
  int64_t ldq;
  int M, N, K;
  int tiles_m, tiles_n, group_m;
  int splits, steps_per_split;
  float* part;  // [splits][M][N]
  LinEpi e;
};

// 0.5 (1 + erf(z / sqrt 2)); e receives e^(-z^2 / 2).  The tail 0.5 erfc(|z| / sqrt 2) is
// e^(-z^2 / 2) t P(t) with t = 1 / (1 + 0.36 |z|): P, of degree 6, was fitted by least squares
// reweighted towards the least relative error, 1.2e-6 in fp32 for |z| up to 13.1 (where the
// exponential leaves fp32), so that gelu's negative tail keeps its digits: with the exponential
// 2^-16 at |z| = 13, within 2^-18 up to 5
__device__ __forceinline__ float lin_phi(float z, float& e) {
  const float t = __builtin_amdgcn_rcpf(1.f + 0.36f * fabsf(z));
  e = __expf(-0.5f * z * z);
  const float tail =
      e * (t * (0.143711373f +
                t * (0.141796127f +
                     t * (0.139589041f + t * (0.026906848f + t * (0.180434123f + t * (-0.179382592f + t * 0.0469447300f)))))));
  return z < 0.f ? tail : 1.f - tail;
}
// the argument of gelu's tanh as t = 1 / (1 + e^(-2 u)): (1 + tanh u) / 2
__device__ __forceinline__ float lin_half_tanh(float z) {
  const float u = 0.79788456f * (z + 0.044715f * z * z * z);
  return __builtin_amdgcn_rcpf(1.f + __expf(-2.f * u));
}
template <int N>
__device__ __forceinline__ void lin_act(float (&z)[N], int act) {
  float e;
  if (act == kActRelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = z[i] > 0.f ? z[i] : (z[i] != z[i] ? z[i] : 0.f);
  } else if (act == kActSilu) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = z[i] * __builtin_amdgcn_rcpf(1.f + __expf(-z[i]));
  } else if (act == kActGelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = z[i] * lin_phi(z[i], e);
  } else if (act == kActGeluTanh) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = z[i] * lin_half_tanh(z[i]);
  }
}
__device__ __forceinline__ float lin_slope(float z, int act) {
  if (act == kActRelu) return z > 0.f ? 1.f : 0.f;
  if (act == kActSilu) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
    return s * (1.f + z * (1.f - s));
  }
  if (act == kActGelu) {
    float e;
    const float phi = lin_phi(z, e);
    return phi + z * 0.39894228f * e;
  }
  if (act == kActGeluTanh) {
    z = z > 30.f ? 30.f : z < -30.f ? -30.f : z;  // (0 and 1 there; its square must not overflow.  A NaN stays)
    const float s = lin_half_tanh(z);
    return s + z * 2.f * s * (1.f - s) * 0.79788456f * (1.f + 0.134145f * z * z);
  }
  return 1.f;
}

// 8 elements of a row from p of which the first n are there, as fp32 (n >= 8: one access)
__device__ __forceinline__ void lin_get8(const uint16_t* p, int n, float (&v)[8]) {
  if (n >= 8) {
    uint32_t w[4];
    __builtin_memcpy(w, p, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = af3_bf16_to_f32(w[i]);
      v[2 * i + 1] = af3_bf16_to_f32(w[i] >> 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? af3_bf16_to_f32(p[i]) : 0.f;
  }
}
__device__ __forceinline__ void lin_put8(uint16_t* p, int n, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = af3_pack_bf16x2(v[2 * i], v[2 * i + 1]);
  if (n >= 8) {
    __builtin_memcpy(p, w, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
  }
}
// the bias of 8 columns from `col`
__device__ __forceinline__ void lin_bias(const LinEpi& e, int col, int N, float (&b)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = 0.f;
  if (!e.bias || col >= N) return;
  if (!e.bias_f32) {
    lin_get8((const uint16_t*)e.bias + col, N - col, b);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < N) b[i] = ((const float*)e.bias)[col + i];
  }
}
// sums v (bias added) and residual r of 8 columns from `col` of row m -> output
template <bool ACT>
__device__ __forceinline__ void lin_finish(const LinEpi& e, int64_t m, int col, int N, float (&v)[8], const float (&r)[8]) {
  const int64_t at = m * N + col;
  if (ACT) {
    if (e.z) lin_put8(e.z + at, N - col, v);
    lin_act(v, e.act);
  }
  if (e.res) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += r[i];
  }
  lin_put8(e.y + at, N - col, v);
}

__device__ __forceinline__ void lin_dma16(const void* sbase, uint32_t voff, uint32_t lds_byte_addr) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "{m0}"(lds_byte_addr) : "memory");
}

// an address that is the same in all lanes, in scalar registers
__device__ __forceinline__ const uint16_t* lin_uniform(const uint16_t* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  return (const uint16_t*)(uintptr_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v) |
                                      (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32)) << 32);
}

template <int V>
struct Int {
  static constexpr int value = V;
};
// f(Int<0>) .. f(Int<N - 1>)
template <int N, int I = 0, class F>
__device__ __forceinline__ void lin_unroll(F&& f) {
  if constexpr (I < N) {
    f(Int<I>{});
    lin_unroll<N, I + 1>(f);
  }
}

template <bool V>
struct Flag {
  static constexpr bool value = V;
};

// One operand of a tile: R of its rows (or columns, T) by 64 k in LDS.
template <int R, bool T>
struct LinTile {
  static constexpr int kRowB = T ? R * 2 : 128;       // bytes per LDS row: 64 k of a row, or a k of all rows
  static constexpr int kCh = kRowB / 16;              // 16-byte chunks per LDS row
  static constexpr int kBytes = R * 128;
  static constexpr int kCopies = kBytes / 1024 / 4;   // 1 KB copies per wave and k-step
  static_assert(kCopies * 4096 == kBytes, "whole copies per wave");
  // XOR of a chunk's index.  A 16-byte read takes 16 rows' equal chunks at a time, a
  // transposing read 4 rows' 4 chunks; over 64 banks (16 chunks) both fall into
  // distinct ones.
  static __device__ __forceinline__ int swz(int row) {
    if constexpr (!T) return (row >> 1) & 7;
    else if constexpr (kCh % 16 == 0) return (row & 3) << 2;
    else return (row & 2) << 1;  // (rows 8 chunks apart, modulo 16)
  }
  // element (LDS row, chunk) that lane `lane` of copy c of the block's 4 kCopies brings
  static __device__ __forceinline__ void place(int c, int lane, int& row, int& chunk) {
    const int id = c * 64 + lane;
    row = id / kCh;
    chunk = (id % kCh) ^ swz(row);
  }
};

// a wave's copies of a k-step of which the first `left` k are there: zeros past them
template <class TT, bool T>
__device__ __forceinline__ void lin_copy_tail(int wave, int lane, int left, int edge, const uint16_t* src, int64_t ld,
                                              uint32_t lds_byte_addr) {
#pragma unroll 1
  for (int j = 0; j < TT::kCopies; ++j) {
    int row, ch;
    TT::place(wave * TT::kCopies + j, lane, row, ch);
    const bool live = T ? row < left : ch * 8 < left;
    if (T) ch = min(ch, (edge + 7) / 8 - 1);
    else row = min(row, edge - 1);
    af3_u32x4 v = {0, 0, 0, 0};
    if (live) v = *(const af3_u32x4*)(src + row * ld + ch * 8);
    *(__attribute__((address_space(3))) af3_u32x4*)(uintptr_t)(lds_byte_addr + j * 1024 + lane * 16) = v;
  }
}

// BM x BN tile, see above.  RES: with a residual and no activation, whole tiles load it ahead
// (a kernel of its own: the registers that takes cost the others 5%).  MASKED outputs past M, N are not stored; loads there repeat the last row.
template <int BM, int BN, int ST, bool PT, bool QT, bool RES>
__global__ __launch_bounds__(256, BM * BN * ST <= 128 * 128 * 2 ? 2 : 1) void lin_kernel(const LinArgs a) {
  using TP = LinTile<BM, PT>;
  using TQ = LinTile<BN, QT>;
  constexpr int TM = BM / 64, TN = BN / 64;
  constexpr int STAGE = TP::kBytes + TQ::kBytes;
  constexpr int NC = TP::kCopies + TQ::kCopies;
  constexpr int NS = TM * TN;      // products per sub-step
  constexpr int NF = TM + TN;      // fragments per sub-step
  constexpr int EPI = 32 * (BN / 2 * 4);  // bytes per wave of the epilogue's turn
  static_assert(4 * EPI <= STAGE, "the epilogue fits a stage");
  constexpr int STORES = (32 + 64 / (BN / 16) - 1) / (64 / (BN / 16)) * TM;  // of a wave for a whole tile, at least
  static_assert(NC * (ST - 2) + STORES < 64, "vmcnt counts to 63");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[ST * STAGE];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 31, lh = lane >> 5;

  // work items: blocks go round robin over 8 XCDs; each XCD takes a run of the tiles, in
  // groups of group_m tile rows so that the ones in flight share operands in its L2, and
  // its blocks walk that run side by side
  const int tiles = a.tiles_m * a.tiles_n;
  const int total = tiles * a.splits;
  const int xcd = blockIdx.x & 7, stride = ((int)gridDim.x - xcd + 7) >> 3;
  const int items_end = (xcd + 1) * (total >> 3) + min(xcd + 1, total & 7);
  int item = xcd * (total >> 3) + min(xcd, total & 7) + (blockIdx.x >> 3);
  if (item >= items_end) return;
  const int wm0 = (wave >> 1) * (BM / 2), wn0 = (wave & 1) * (BN / 2);
  const int nk_all = (a.K + 63) / 64;

  // the item whose copies are issued next
  int split, m0, n0, nk;
  bool tail;                 // its last k-step is not whole
  const uint16_t *pk, *qk;   // of the next k-step to copy
  uint32_t off[NC];          // this lane's source of each copy: byte offsets from there
  const int64_t pstep = PT ? 64 * a.ldp : 64, qstep = QT ? 64 * a.ldq : 64;
  auto setup = [&]() {
    // (divisions run on the vector unit: their results go back to scalar registers)
    split = __builtin_amdgcn_readfirstlane(item / tiles);
    const int tile = item - split * tiles;
    const int gsz = a.group_m * a.tiles_n;
    const int grp = __builtin_amdgcn_readfirstlane(tile / gsz), in = tile - grp * gsz;
    const int gm = min(a.group_m, a.tiles_m - grp * a.group_m);
    const int tn = __builtin_amdgcn_readfirstlane(in / gm);
    m0 = (grp * a.group_m + in - tn * gm) * BM, n0 = tn * BN;
    const int k_first = split * a.steps_per_split;
    nk = __builtin_amdgcn_readfirstlane(min(a.steps_per_split, nk_all - k_first));
    tail = k_first + nk == nk_all && (a.K & 63);
    pk = lin_uniform(PT ? a.p + (int64_t)k_first * 64 * a.ldp + m0 : a.p + (int64_t)m0 * a.ldp + k_first * 64);
    qk = lin_uniform(QT ? a.q + (int64_t)k_first * 64 * a.ldq + n0 : a.q + (int64_t)n0 * a.ldq + k_first * 64);
#pragma unroll
    for (int j = 0; j < TP::kCopies; ++j) {
      int row, ch;
      TP::place(wave * TP::kCopies + j, lane, row, ch);
      off[j] = PT ? (uint32_t)(row * a.ldp * 2 + min(ch, (a.M - m0 + 7) / 8 - 1) * 16)
                  : (uint32_t)(min(row, a.M - m0 - 1) * a.ldp * 2 + ch * 16);
    }
#pragma unroll
    for (int j = 0; j < TQ::kCopies; ++j) {
      int row, ch;
      TQ::place(wave * TQ::kCopies + j, lane, row, ch);
      off[TP::kCopies + j] = QT ? (uint32_t)(row * a.ldq * 2 + min(ch, (a.N - n0 + 7) / 8 - 1) * 16)
                                : (uint32_t)(min(row, a.N - n0 - 1) * a.ldq * 2 + ch * 16);
    }
  };
  const uint32_t lds0 =
      __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)lds);
  auto lds_at = [&](int j, int stage) {
    return lds0 + (uint32_t)(stage * STAGE + (j < TP::kCopies ? (wave * TP::kCopies + j) * 1024
                                                              : TP::kBytes + (wave * TQ::kCopies + j - TP::kCopies) * 1024));
  };
  auto copy = [&](int j, int stage) { lin_dma16(j < TP::kCopies ? pk : qk, off[j], lds_at(j, stage)); };
  // the last k-step where K is not a multiple of 64: chunks past K are zeros
  auto copy_tail = [&](int stage) {
    lin_copy_tail<TP, PT>(wave, lane, a.K & 63, a.M - m0, pk, a.ldp, lds_at(0, stage));
    lin_copy_tail<TQ, QT>(wave, lane, a.K & 63, a.N - n0, qk, a.ldq, lds_at(TP::kCopies, stage));
  };

  // this lane's fragment addresses in stage 0
  constexpr int PA = PT ? TM : 4, QA = QT ? TN : 4;
  uint32_t pa[PA], qa[QA];
  {
    const int tr_r = 8 * lh + ((lane & 15) >> 2);             // k of the first transposing read
    const int tr_c = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);  // its column
#pragma unroll
    for (int i = 0; i < PA; ++i)
      pa[i] = lds0 + (PT ? tr_r * TP::kRowB + ((((wm0 + 32 * i + tr_c) >> 3) ^ TP::swz(tr_r)) << 4) + ((tr_c & 7) << 1)
                         : (wm0 + lr) * 128 + (((2 * i + lh) ^ TP::swz(lr)) << 4));
#pragma unroll
    for (int i = 0; i < QA; ++i)
      qa[i] = lds0 + TP::kBytes +
              (QT ? tr_r * TQ::kRowB + ((((wn0 + 32 * i + tr_c) >> 3) ^ TQ::swz(tr_r)) << 4) + ((tr_c & 7) << 1)
                  : (wn0 + lr) * 128 + (((2 * i + lh) ^ TQ::swz(lr)) << 4));
  }
  auto frag = [](bool trans, uint32_t addr, int row_bytes) {  // (8 k of one row)
    if (trans) {
      const bf16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(uintptr_t)addr);
      const bf16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(uintptr_t)(addr + 4 * row_bytes));
      return af3_bf16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    }
    return *(lds_frag*)(uintptr_t)addr;
  };
  auto frag_p = [&](int s, int tm, uint32_t stage) {
    return PT ? frag(true, pa[tm % PA] + stage + s * 16 * TP::kRowB, TP::kRowB)
              : frag(false, pa[s % PA] + stage + tm * 32 * 128, 0);
  };
  auto frag_q = [&](int s, int tn, uint32_t stage) {
    return QT ? frag(true, qa[tn % QA] + stage + s * 16 * TQ::kRowB, TQ::kRowB)
              : frag(false, qa[s % QA] + stage + tn * 32 * 128, 0);
  };

  af3_f32x16 acc[TM][TN];
  af3_bf16x8 fp[2][TM], fq[2][TN];

  // products of fragments c, between them the reads of sub-step s into c ^ 1 and, with
  // COPY, the next stage's copies
  auto phase = [&](auto copy_, auto c_, auto s_, uint32_t stage, int to) {
    constexpr int c = decltype(c_)::value, s = decltype(s_)::value;
    constexpr bool COPY = decltype(copy_)::value && s >= 0 && s < 2;
#pragma unroll
    for (int i = 0; i < (NS > NF ? NS : NF); ++i) {
      if (i < NS)
        acc[i / TN][i % TN] =
            __builtin_amdgcn_mfma_f32_32x32x16_bf16(fq[c][i % TN], fp[c][i / TN], acc[i / TN][i % TN], 0, 0, 0);
      if (s >= 0 && i < NF) {
        if (i < TN) fq[c ^ 1][i] = frag_q(s, i, stage);
        else fp[c ^ 1][i - TN] = frag_p(s, i - TN, stage);
      }
      if constexpr (COPY) {
        constexpr int NP = 2;
#pragma unroll
        for (int j = 0; j < NC; ++j)
          if (j * (NP * NS) / NC == s * NS + i) copy(j, to);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto ahead = [](int stage, int n) { return stage + n >= ST ? stage + n - ST : stage + n; };
  auto step = [&](auto copy_, int cur) {
    const uint32_t stage = (uint32_t)(cur * STAGE);
    const int to = ahead(cur, ST - 1);
    phase(copy_, Int<1>{}, Int<0>{}, stage, to);  // (the last step's last products; of zeros in the first)
    phase(copy_, Int<0>{}, Int<1>{}, stage, to);
    phase(copy_, Int<1>{}, Int<2>{}, stage, to);
    phase(copy_, Int<0>{}, Int<3>{}, stage, to);
  };
  // a k-step's copies have landed (all but the n youngest accesses), and every wave has
  // read the stage before it
#define LIN_WAIT(n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(n) : "memory")

  // an item's first k-steps, up to ST - 1 of them; pk and qk are left at the next one
  auto first_copies = [&](int stage) {
    const int whole = nk - (tail ? 1 : 0);
    if (whole == 0) {
      copy_tail(stage);
      return;
    }
#pragma unroll
    for (int s = 0; s < ST - 1; ++s)
      if (s < whole) {
#pragma unroll
        for (int j = 0; j < NC; ++j) copy(j, ahead(stage, s));
        pk += pstep, qk += qstep;
      }
  };

  setup();
  int cur = 0;   // stage of the next k-step
  first_copies(cur);
  bool stores = false;  // this wave's accesses since its first copies are STORES stores or more
  for (;;) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
#pragma unroll
    for (int i = 0; i < TM; ++i) fp[1][i] = af3_bf16x8{};
#pragma unroll
    for (int i = 0; i < TN; ++i) fq[1][i] = af3_bf16x8{};

    // (the last item's stores may still be under way: they are younger than the copies)
    const int whole = nk - (tail ? 1 : 0);
    if (ST > 2 && whole < ST - 1) LIN_WAIT(0);
    else if (stores) LIN_WAIT(NC * (ST - 2) + STORES);
    else LIN_WAIT(NC * (ST - 2));
    int left = whole - (ST - 1);  // k-steps that bring a whole one
    if (left > 0) {
      for (;;) {
        step(Flag<true>{}, cur);
        pk += pstep, qk += qstep;
        cur = ahead(cur, 1);
        LIN_WAIT(NC * (ST - 2));
        if (--left == 0) break;
      }
    }
    if (ST > 2 || (tail && nk > 1)) {
      for (left = min(ST - 1, whole) + (tail ? 1 : 0) - 1; left > 0; --left) {
        if (tail && left == 1) copy_tail(ahead(cur, 1));
        step(Flag<false>{}, cur);
        cur = ahead(cur, 1);
        LIN_WAIT(0);
      }
    }
    // the last k-step, and the next item's first copies
    const int em0 = m0 + wm0, en0 = n0 + wn0, es_split = split;
    const bool whole_tile = m0 + BM <= a.M && n0 + BN <= a.N;
    item += stride;
    const bool more = item < items_end;
    if (more) {
      setup();
      first_copies(ahead(cur, 1));
    }
    // what the epilogue reads from memory lands meanwhile: the bias of the lane's 8 columns, and
    // with RES the residual of a whole tile's first two bands of 32 rows
    constexpr int W = BN / 2;        // columns of a wave
    constexpr int LPR = W / 8;       // lanes per row when read back
    constexpr int RPI = 64 / LPR;    // rows a wave reads at a time: a lane keeps its 8 columns
    constexpr int IT = (32 + RPI - 1) / RPI;
    const int c8 = lane % LPR * 8, col = en0 + c8;
    float bias[8];
    lin_bias(a.e, lane < RPI * LPR ? col : a.N, a.N, bias);
    const bool plain = RES && whole_tile;
    auto there = [&](int g) { return g * RPI + lane / LPR < 32 && lane < RPI * LPR; };
    uint32_t res[2][RES ? IT : 1][4];
    auto fetch_res = [&](int tm, uint32_t (&r)[RES ? IT : 1][4]) __attribute__((always_inline)) {
#pragma unroll
      for (int g = 0; g < (RES ? IT : 0); ++g)
        __builtin_memcpy(r[g], a.e.res + (int64_t)(em0 + tm * 32 + min(g * RPI + lane / LPR, 31)) * a.e.ldr + col, 16);
    };
    if (plain) {
      fetch_res(0, res[0]);
      fetch_res(1, res[1]);
    }
    step(Flag<false>{}, cur);
    phase(Flag<false>{}, Int<1>{}, Int<-1>{}, 0, 0);

    // epilogue, in the last k-step's stage: lane (r, h) holds row r of a 32 x 32 part,
    // columns 8 j + 4 h + (0..3)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // (the bias is taken here whichever path uses it: left to some, its wait would stand in the
    // next tile's k-steps, and wait for the copies too)
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(bias[i]));
    constexpr int ROWB = W * 4;      // bytes of a staged row; 16-byte chunks XORed with the row's low bits
    const uint32_t es = lds0 + (uint32_t)(cur * STAGE + wave * EPI);
    auto staged = [&](int row, int chunk) { return es + (uint32_t)(row * ROWB + ((chunk ^ (row & 7)) << 4)); };
    // a wave's 32 rows of products into its part of the stage (its own LDS accesses are in
    // order, and the compiler keeps them so)
    auto put = [&](auto i_) __attribute__((always_inline)) {
      constexpr int i = decltype(i_)::value;
#pragma unroll
      for (int tn = 0; tn < TN; ++tn)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *(__attribute__((address_space(3))) f32x4*)(uintptr_t)staged(lr, tn * 8 + 2 * j + lh) =
              f32x4{acc[i][tn][4 * j], acc[i][tn][4 * j + 1], acc[i][tn][4 * j + 2], acc[i][tn][4 * j + 3]};
    };
    auto get = [&](int row, float (&v)[8]) __attribute__((always_inline)) {
      const f32x4 x = *(const __attribute__((address_space(3))) f32x4*)(uintptr_t)staged(row, c8 / 4);
      const f32x4 y = *(const __attribute__((address_space(3))) f32x4*)(uintptr_t)staged(row, c8 / 4 + 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = x[i], v[4 + i] = y[i];
    };
    auto read = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };  // (before the next 32 rows overwrite)
    // rows tm of the tile, U at a time; EDGE: rows and columns past the output are left out
    auto out = [&](int tm, auto edge_, auto act_, auto u_) __attribute__((always_inline)) {
      constexpr bool EDGE = decltype(edge_)::value, ACT = decltype(act_)::value;
      constexpr int U = decltype(u_)::value;
#pragma unroll 1
      for (int g = 0; g < IT; g += U) {
        float v[U][8], r[U][8];
        bool live[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int row = (g + u) * RPI + lane / LPR;
          const int64_t m = em0 + tm * 32 + row;
          live[u] = g + u < IT && there(g + u) && (!EDGE || (m < a.M && col < a.N));
          if (live[u]) {
            if (a.e.res) lin_get8(a.e.res + m * a.e.ldr + col, EDGE ? a.N - col : 8, r[u]);
            get(row, v[u]);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u][i] += bias[i];
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t m = em0 + tm * 32 + (g + u) * RPI + lane / LPR;
          if (live[u]) lin_finish<ACT>(a.e, m, col, a.N, v[u], r[u]);
        }
      }
    };
    if (whole_tile && !a.e.act && !a.part) {
      lin_unroll<TM>([&](auto tm_) __attribute__((always_inline)) {
        constexpr int tm = decltype(tm_)::value;
        put(tm_);
        if constexpr (RES) {
#pragma unroll
          for (int g = 0; g < IT; ++g) {
            const int row = min(g * RPI + lane / LPR, 31);  // (a lane past the rows repeats the last, and stores nothing)
            float v[8];
            uint32_t w[4];
            get(row, v);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = af3_pack_bf16x2(v[2 * i] + bias[2 * i] + af3_bf16_to_f32(res[tm & 1][g][i]),
                                     v[2 * i + 1] + bias[2 * i + 1] + af3_bf16_to_f32(res[tm & 1][g][i] >> 16));
            if (there(g)) __builtin_memcpy(a.e.y + (int64_t)(em0 + tm * 32 + row) * a.N + col, w, 16);
          }
          if constexpr (tm + 2 < TM) fetch_res(tm + 2, res[tm & 1]);
        } else {
          out(tm, Flag<false>{}, Flag<false>{}, Int<4>{});
        }
        read();
      });
    } else {
#pragma unroll 1
      for (int tm = 0; tm < TM; ++tm) {  // (one copy of the code: acc[0] becomes the next rows')
        put(Int<0>{});
#pragma unroll
        for (int i = 0; i + 1 < TM; ++i)
#pragma unroll
          for (int tn = 0; tn < TN; ++tn) acc[i][tn] = acc[i + 1][tn];
        if (!RES && a.part) {
#pragma unroll 2
          for (int g = 0; g < IT; ++g) {
            const int row = g * RPI + lane / LPR;
            const int64_t m = em0 + tm * 32 + row;
            if (!there(g) || m >= a.M || col >= a.N) continue;
            float v[8];
            get(row, v);
            float* const o = a.part + ((int64_t)es_split * a.M + m) * a.N + col;
            if (col + 8 <= a.N) {
              __builtin_memcpy(o, v, 32);
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (col + i < a.N) o[i] = v[i];
            }
          }
        } else if (!RES && a.e.act) {
          if (whole_tile) out(tm, Flag<false>{}, Flag<true>{}, Int<2>{});
          else out(tm, Flag<true>{}, Flag<true>{}, Int<2>{});
        } else {
          out(tm, Flag<true>{}, Flag<false>{}, Int<2>{});
        }
        read();
      }
      // (vmcnt(0), for the same reason: loads of edges and residuals that some path leaves open)
      if (!a.part) __builtin_amdgcn_s_waitcnt(0x0F70);
    }
    if (!more) break;
    stores = !a.part && whole_tile;
    cur = ahead(cur, 1);
  }
}

// partials of the splits, added in order, then the epilogue: 8 columns of a row per thread
__global__ __launch_bounds__(256) void lin_join_kernel(const float* part, int splits, int64_t M, int N, const LinEpi e) {
  const int ncol = (N + 7) / 8;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t m = id / ncol;
  const int col = (int)(id - m * ncol) * 8;
  if (m >= M) return;
  float v[8], r[8];
  lin_bias(e, col, N, v);
  if (e.res) lin_get8(e.res + m * e.ldr + col, N - col, r);
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float* const p = part + ((int64_t)s * M + m) * N + col;
    if (col + 8 <= N) {
      float f[8];
      __builtin_memcpy(f, p, 32);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += f[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < N) v[i] += p[i];
    }
  }
  if (e.act)
    lin_finish<true>(e, m, col, N, v, r);
  else
    lin_finish<false>(e, m, col, N, v, r);
}

// Up to 16 NT rows of x: a block makes 16 columns (rows of W).  Its 16 waves share k in
// units of 64, a wave's lane (r, g) taking k = 8 g + (0..7) and 32 more of row r of W and of
// x (two products of 32 k), so W is read once, 64 contiguous bytes of 16 rows at a time; the
// waves' sums meet in LDS.  A wave has the loads of U units in flight together where K brings it
// as many (U 4, or 2 for 17 to 32 rows: all waves from K = 1024 U on, none below 64 (16 U - 15),
// 3136 and 1088); units past a multiple of U go one after the other.
// Addresses need no alignment; elements past K are zeros.  One row at a stated N x K, us:
// 512 x 2880 5.2, 4096 x 2880 6.1, 2880 x 4096 6.7 (4.0 TB/s of W); 32 rows 9.7, 10.3, 12.9,
// where gathering x's 16-row fragments costs 3 to 6 of it.  Eight waves, two columns' tiles
// a block, or a start rotated by block gain nothing.
constexpr int kSkinnyWaves = 16;

// 8 elements at p of which the first n are there, zeros after them
__device__ __forceinline__ void lin_words(const uint16_t* p, int n, af3_u32x4& v) {
  if (n >= 8) {
    __builtin_memcpy(&v, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = 2 * i < n ? p[2 * i] : 0, hi = 2 * i + 1 < n ? p[2 * i + 1] : 0;
      v[i] = lo | hi << 16;
    }
  }
}

template <int NT>
__global__ __launch_bounds__(kSkinnyWaves * 64) void lin_skinny_kernel(const LinArgs a) {
  __shared__ float lds[kSkinnyWaves][NT * 16][17];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const uint16_t* const w = a.q + (int64_t)min(n0 + r, a.N - 1) * a.ldq + g * 8;
  const uint16_t* x[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) x[t] = a.p + (int64_t)min(t * 16 + r, a.M - 1) * a.ldp + g * 8;
  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto mul = [&](const af3_u32x4 (&wv)[2], const af3_u32x4 (&xv)[NT][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(af3_bf16x8, wv[i]),
                                                         __builtin_bit_cast(af3_bf16x8, xv[t][i]), acc[t], 0, 0, 0);
  };
  // U units' loads side by side (one after the other's latency costs 32 rows of 4096 14 us instead of 8)
  constexpr int U = NT == 1 ? 4 : 2;
  const int whole = a.K / 64;
  int u = wave;
  for (; u + (U - 1) * kSkinnyWaves < whole; u += U * kSkinnyWaves) {
    af3_u32x4 wv[U][2], xv[U][NT][2];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int k = (u + i * kSkinnyWaves) * 64;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        __builtin_memcpy(&wv[i][h], w + k + 32 * h, 16);
#pragma unroll
        for (int t = 0; t < NT; ++t) __builtin_memcpy(&xv[i][t][h], x[t] + k + 32 * h, 16);
      }
    }
#pragma unroll
    for (int i = 0; i < U; ++i) mul(wv[i], xv[i]);
  }
  for (; u * 64 < a.K; u += kSkinnyWaves) {  // fewer, and the one that K ends in
    af3_u32x4 wv[2], xv[NT][2];
    const int k = u * 64, n = a.K - k - g * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      lin_words(w + k + 32 * h, n - 32 * h, wv[h]);
#pragma unroll
      for (int t = 0; t < NT; ++t) lin_words(x[t] + k + 32 * h, n - 32 * h, xv[t][h]);
    }
    mul(wv, xv);
  }
  // lane (c, g): row c of x, columns 4 g + (0..3)
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) lds[wave][t * 16 + r][4 * g + i] = acc[t][i];
  __syncthreads();
  if (threadIdx.x >= NT * 256) return;
  const int m = threadIdx.x >> 4, c = threadIdx.x & 15, col = n0 + c;
  float f = 0.f;
#pragma unroll
  for (int v = 0; v < kSkinnyWaves; ++v) f += lds[v][m][c];
  if (m >= a.M || col >= a.N) return;
  const LinEpi& e = a.e;
  const int64_t at = (int64_t)m * a.N + col;
  if (e.bias) f += e.bias_f32 ? ((const float*)e.bias)[col] : af3_bf16_to_f32(((const uint16_t*)e.bias)[col]);
  if (e.act) {
    if (e.z) e.z[at] = (uint16_t)af3_f32_to_bf16(f);
    float one[1] = {f};
    lin_act(one, e.act);
    f = one[0];
  }
  if (e.res) f += af3_bf16_to_f32(e.res[(int64_t)m * e.ldr + col]);
  e.y[at] = (uint16_t)af3_f32_to_bf16(f);
}

// dz = dy act'(z) in bf16 with rows of ldz elements (zeros past N), and the columns' sums
// (of dz before rounding): a block takes 32 lanes x 8 columns by its share of the rows.
// HBM: 16384 x 2880 sums alone 19 us (5.0 TB/s), with gelu and dz 71 (4.0; the slope's
// exponential and two reciprocals per element beside it).  Two, four and eight rows' loads
// side by side: 19 and 63, 31 and 92, 42 and 129.
constexpr int kDzRows = 8;  // rows a block takes at a time

struct DzArgs {
  const uint16_t* dy;
  int64_t ldy;
  const uint16_t* z;  // [M][N], or null
  int act;
  int64_t M;
  int N;
  uint16_t* dz;       // or null
  int64_t ldz;
  float* part;        // [gridDim.y][N], or null
};

__global__ __launch_bounds__(256) void lin_dz_kernel(const DzArgs a) {
  __shared__ float lds[kDzRows][257];
  const int c = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int col = (blockIdx.x * 32 + c) * 8;
  float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  const int width = (int)min((int64_t)((a.N + 7) / 8 * 8), a.ldz);
  for (int64_t m = (int64_t)blockIdx.y * kDzRows + w; m < a.M; m += (int64_t)gridDim.y * kDzRows) {
    if (col >= a.N) break;
    uint16_t d[8], zz[8];
    const bool whole = col + 8 <= a.N;
    if (whole) {
      __builtin_memcpy(d, a.dy + m * a.ldy + col, 16);
      if (a.act) __builtin_memcpy(zz, a.z + m * a.N + col, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        d[i] = col + i < a.N ? a.dy[m * a.ldy + col + i] : 0;
        zz[i] = a.act && col + i < a.N ? a.z[m * a.N + col + i] : 0;
      }
    }
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] = af3_bf16_to_f32(d[i]);
      if (a.act) f[i] = (whole || col + i < a.N) ? f[i] * lin_slope(af3_bf16_to_f32(zz[i]), a.act) : 0.f;
      s[i] += f[i];
    }
    if (a.dz) {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = af3_pack_bf16x2(f[2 * i], f[2 * i + 1]);
      uint16_t* const p = a.dz + m * a.ldz + col;
      if (col + 8 <= width) {
        __builtin_memcpy(p, o, 16);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (col + i < width) p[i] = (uint16_t)(o[i >> 1] >> (16 * (i & 1)));
      }
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) lds[w][c * 8 + i] = s[i];
  __syncthreads();
  const int at = blockIdx.x * 256 + threadIdx.x;
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < kDzRows; ++i) t += lds[i][threadIdx.x];
  if (at < a.N) a.part[(int64_t)blockIdx.y * a.N + at] = t;
}

// partials' columns -> the bias's gradient: 16 columns a block, 64 lanes of rows joined in pairs
constexpr int kSumCols = 16, kSumRows = 64;

__global__ __launch_bounds__(kSumCols* kSumRows) void lin_colsum_kernel(const float* part, int n, int N, void* out, int f32) {
  __shared__ float lds[kSumRows][kSumCols];
  const int c = threadIdx.x % kSumCols, w = threadIdx.x / kSumCols;
  const int col = blockIdx.x * kSumCols + c;
  float s = 0.f;
  if (col < N) {
#pragma unroll 4
    for (int i = w; i < n; i += kSumRows) s += part[(int64_t)i * N + col];
  }
  lds[w][c] = s;
  __syncthreads();
#pragma unroll
  for (int h = kSumRows / 2; h > 0; h /= 2) {
    if (w < h) lds[w][c] = s = s + lds[w + h][c];
    __syncthreads();
  }
  if (w || col >= N) return;
  if (f32)
    ((float*)out)[col] = s;
  else
    ((uint16_t*)out)[col] = (uint16_t)af3_f32_to_bf16(s);
}

// Tile shape, ring depth and split of a product: what should take the least time, in us:
// k-steps of the tile's measured time, what its start and end leave uncovered, and for a
// split sum the joining launch and its read of the partials.  The card's power bounds full
// rounds (the clock falls to 1.75 GHz), so a round of fewer tiles takes their share of a
// full round's time, down to what one tile alone takes at the full clock.  Per k-step in a
// full round, alone, and per tile: 256 x 256 1.70, 1.20 and 7; 256 x 192 1.27, 0.90 and 6;
// 128 x 128 two to a CU (two stages each) 0.97, 0.70 and 2.7; one to a CU 0.50, 0.43 and
// 2.7 (four stages: three k-steps under way, where two stages leave 0.73, a copy's latency).
// 2880 x 4096 from 16384 rows: 192 tiles of 256 x 256 315 us, split in four 375.
struct LinPlan {
  int bm, bn, stages, splits, steps;
};

LinPlan lin_plan(int64_t M, int64_t N, int64_t K) {
  static const struct {
    int bm, bn, stages, slots;  // slots: tiles that run at a time
    double step, alone, ends;
  } shapes[] = {{256, 256, 2, 256, 1.70, 1.20, 7.0},
                {256, 192, 2, 256, 1.27, 0.90, 6.0},
                {128, 128, 2, 512, 0.97, 0.70, 2.7},
                {128, 128, 4, 256, 0.50, 0.43, 2.7}};
  const int64_t nk = af3_cdiv(K, 64);
  LinPlan best = {};
  double best_t = 1e300;
  for (const auto& s : shapes) {
    const int64_t tiles = af3_cdiv(M, s.bm) * af3_cdiv(N, s.bn);
    for (int sp = 1; sp <= 16; ++sp) {
      const int64_t steps = af3_cdiv(nk, sp);
      if (sp > 1 && (steps < 8 || tiles >= 2 * s.slots)) break;
      const int64_t used = af3_cdiv(nk, steps), items = tiles * used;
      const int64_t rounds = items / s.slots, rest = items % s.slots;
      const double part = s.step * (double)rest / s.slots;
      const double t = (double)steps * ((double)rounds * s.step + (rest ? (part > s.alone ? part : s.alone) : 0.0)) +
                       (double)af3_cdiv(items, s.slots) * s.ends +
                       (used > 1 ? (double)used * 4 * M * N / 5e6 + 6.0 : 0.0);
      if (t < best_t) best_t = t, best = {s.bm, s.bn, s.stages, (int)used, (int)steps};
    }
  }
  return best;
}

template <int BM, int BN, int ST>
void lin_launch(const LinArgs& a, bool pt, bool qt, hipStream_t st) {
  const int64_t items = (int64_t)a.tiles_m * a.tiles_n * a.splits, slots = BM * BN * ST <= 128 * 128 * 2 ? 512 : 256;
  const dim3 grid((unsigned)(items < slots ? items : slots));
  if (!pt && !qt && a.e.res && !a.e.act && !a.part)
    hipLaunchKernelGGL((lin_kernel<BM, BN, ST, false, false, true>), grid, dim3(256), 0, st, a);
  else if (!pt && !qt)
    hipLaunchKernelGGL((lin_kernel<BM, BN, ST, false, false, false>), grid, dim3(256), 0, st, a);
  else if (!pt)
    hipLaunchKernelGGL((lin_kernel<BM, BN, ST, false, true, false>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((lin_kernel<BM, BN, ST, true, true, false>), grid, dim3(256), 0, st, a);
}

// (the tiles instead, us: 512 x 2880 1 row 10.3, 16 11.2 for 7.2, 32 11.5 for 9.7; 2880 x 4096
// 32 rows 13.8 for 12.9, so a third row tile would lose)
constexpr int kSkinnyRows = 32;
bool lin_skinny(int64_t M, bool pt, bool qt) { return M <= kSkinnyRows && !pt && !qt; }

}  // namespace

extern "C" size_t af3_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int p_trans, int q_trans) {
  if (M <= 0 || N <= 0 || K <= 0 || lin_skinny(M, p_trans, q_trans)) return 0;
  const LinPlan p = lin_plan(M, N, K);
  return p.splits > 1 ? (size_t)p.splits * M * N * 4 : 0;
}

extern "C" int af3_linear_tile(int64_t M, int64_t N, int64_t K, int p_trans, int q_trans, int* tile) {
  AF3_REQUIRE(tile && M > 0 && N > 0 && K > 0 && M < (int64_t)1 << 30 && N < (int64_t)1 << 30 && K < (int64_t)1 << 30,
              "linear_tile: bad sizes");
  const LinPlan p = lin_skinny(M, p_trans, q_trans) ? LinPlan{} : lin_plan(M, N, K);
  tile[0] = p.bm, tile[1] = p.bn, tile[2] = p.stages, tile[3] = p.splits;
  return 0;
}

extern "C" int af3_linear(const uint16_t* p, int64_t ldp, int p_trans, const uint16_t* q, int64_t ldq, int q_trans,
                          int64_t M, int64_t N, int64_t K, const void* bias, int bias_f32, int act,
                          const uint16_t* residual, int64_t ldr, uint16_t* y, uint16_t* z, void* workspace,
                          size_t ws_bytes, void* stream_) {
  AF3_REQUIRE(M >= 0 && N >= 0 && K >= 0 && M < (int64_t)1 << 30 && N < (int64_t)1 << 30 && K < (int64_t)1 << 30,
              "linear: bad sizes");
  AF3_REQUIRE(act >= kActNone && act <= kActGeluTanh, "linear: activation %d", act);
  AF3_REQUIRE(!p_trans || q_trans, "linear: p_trans needs q_trans");
  if (M == 0 || N == 0) return 0;
  AF3_REQUIRE(K > 0, "linear: an empty sum");
  AF3_REQUIRE(p && q && y, "linear: null pointer");
  AF3_REQUIRE(M * N < (int64_t)1 << 40, "linear: output too large");
  hipStream_t st = (hipStream_t)stream_;
  LinArgs a = {};
  a.p = p, a.ldp = ldp, a.q = q, a.ldq = ldq, a.M = (int)M, a.N = (int)N, a.K = (int)K;
  a.e.bias = bias, a.e.bias_f32 = bias_f32, a.e.act = act, a.e.res = residual, a.e.ldr = ldr, a.e.y = y, a.e.z = z;
  if (lin_skinny(M, p_trans, q_trans)) {
    const dim3 grid((unsigned)af3_cdiv(N, 16)), block(kSkinnyWaves * 64);
    if (M <= 16)
      hipLaunchKernelGGL((lin_skinny_kernel<1>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((lin_skinny_kernel<2>), grid, block, 0, st, a);
    return af3::check_launch("linear");
  }
  AF3_REQUIRE(((uintptr_t)p & 15) == 0 && ((uintptr_t)q & 15) == 0 && ldp % 8 == 0 && ldq % 8 == 0,
              "linear: rows must be 16-byte aligned");
  AF3_REQUIRE(ldp >= af3_cdiv(p_trans ? M : K, 8) * 8 && ldq >= af3_cdiv(q_trans ? N : K, 8) * 8,
              "linear: rows must reach the next multiple of 8 elements");
  AF3_REQUIRE(ldp < (int64_t)1 << 22 && ldq < (int64_t)1 << 22, "linear: rows too far apart");
  const LinPlan pl = lin_plan(M, N, K);
  a.tiles_m = (int)af3_cdiv(M, pl.bm), a.tiles_n = (int)af3_cdiv(N, pl.bn), a.group_m = 4;
  AF3_REQUIRE((int64_t)a.tiles_m * a.tiles_n * pl.splits < (int64_t)1 << 30, "linear: output too large");
  a.splits = pl.splits, a.steps_per_split = pl.steps;
  if (pl.splits > 1) {
    AF3_REQUIRE(workspace && ws_bytes >= (size_t)pl.splits * M * N * 4, "linear: workspace too small");
    a.part = (float*)workspace;
  }
  if (pl.bm == 256 && pl.bn == 256)
    lin_launch<256, 256, 2>(a, p_trans, q_trans, st);
  else if (pl.bm == 256)
    lin_launch<256, 192, 2>(a, p_trans, q_trans, st);
  else if (pl.stages == 4)
    lin_launch<128, 128, 4>(a, p_trans, q_trans, st);
  else
    lin_launch<128, 128, 2>(a, p_trans, q_trans, st);
  if (pl.splits > 1) {
    const int64_t n = M * af3_cdiv(N, 8);
    hipLaunchKernelGGL(lin_join_kernel, dim3((unsigned)af3_cdiv(n, 256)), dim3(256), 0, st, a.part, pl.splits, M, (int)N,
                       a.e);
  }
  return af3::check_launch("linear");
}

namespace {
int lin_dz_blocks(int64_t M, int64_t N) {
  const int64_t cols = af3_cdiv(N, 256), rows = af3_cdiv(M, kDzRows);
  const int64_t want = af3_cdiv(1024, cols);  // four blocks per CU
  const int64_t b = want < rows ? want : rows;
  return (int)(b < 1 ? 1 : b);
}
}  // namespace

extern "C" size_t af3_linear_dz_workspace_bytes(int64_t M, int64_t N) {
  return M > 0 && N > 0 ? (size_t)lin_dz_blocks(M, N) * N * 4 : 0;
}

extern "C" int af3_linear_dz(const uint16_t* dy, int64_t ldy, const uint16_t* z, int act, int64_t M, int64_t N,
                             uint16_t* dz, int64_t ldz, void* dbias, int bias_f32, void* workspace, size_t ws_bytes,
                             void* stream_) {
  AF3_REQUIRE(M >= 0 && N >= 0 && N < (int64_t)1 << 30 && M < (int64_t)1 << 40, "linear_dz: bad sizes");
  AF3_REQUIRE(act >= kActNone && act <= kActGeluTanh, "linear_dz: activation %d", act);
  if (M == 0 || N == 0) return 0;
  AF3_REQUIRE(dy && (!act || z) && (dz || dbias), "linear_dz: null pointer");
  AF3_REQUIRE(!dz || ldz >= N, "linear_dz: bad leading dimension");
  const int blocks = lin_dz_blocks(M, N);
  AF3_REQUIRE(!dbias || (workspace && ws_bytes >= (size_t)blocks * N * 4), "linear_dz: workspace too small");
  DzArgs a = {dy, ldy, z, act, M, (int)N, dz, dz ? ldz : N, dbias ? (float*)workspace : nullptr};
  hipStream_t st = (hipStream_t)stream_;
  hipLaunchKernelGGL(lin_dz_kernel, dim3((unsigned)af3_cdiv(N, 256), (unsigned)blocks), dim3(256), 0, st, a);
  if (dbias)
    hipLaunchKernelGGL(lin_colsum_kernel, dim3((unsigned)af3_cdiv(N, kSumCols)), dim3(kSumCols * kSumRows), 0, st, a.part, blocks, (int)N,
                       dbias, bias_f32);
  return af3::check_launch("linear_dz");
}

extern "C" size_t af3_linear_bwd_workspace_bytes(int64_t T, int64_t N, int64_t K, int want_dx, int want_dw, int want_db) {
  size_t n = 0;  // (one after the other on one stream: they share it)
  const size_t each[3] = {want_dx ? af3_linear_workspace_bytes(T, K, N, 0, 1) : 0,
                          want_dw ? af3_linear_workspace_bytes(N, K, T, 1, 1) : 0,
                          want_db ? af3_linear_dz_workspace_bytes(T, N) : 0};
  for (size_t e : each) n = e > n ? e : n;
  return n;
}

extern "C" int af3_linear_bwd(const uint16_t* dy, int64_t ldy, const uint16_t* z, int act, const uint16_t* weight,
                              int64_t ldw, const uint16_t* x, int64_t ldx, int64_t T, int64_t N, int64_t K, uint16_t* dz,
                              int64_t ldz, uint16_t* dx, uint16_t* dweight, void* dbias, int bias_f32, void* workspace,
                              size_t ws_bytes, void* stream) {
  AF3_REQUIRE(T >= 0 && N > 0 && K > 0, "linear_bwd: bad sizes");
  AF3_REQUIRE(dy && (!dx || weight) && (!dweight || x), "linear_bwd: null pointer");
  AF3_REQUIRE(!act || dz || !(dx || dweight), "linear_bwd: the products behind an activation need dz");
  int rc = 0;
  if (dz || dbias) rc = af3_linear_dz(dy, ldy, z, act, T, N, dz, ldz, dbias, bias_f32, workspace, ws_bytes, stream);
  if (rc) return rc;
  const uint16_t* const g = dz ? dz : dy;
  const int64_t ldg = dz ? ldz : ldy;
  if (dx)
    rc = af3_linear(g, ldg, 0, weight, ldw, 1, T, K, N, nullptr, 0, 0, nullptr, 0, dx, nullptr, workspace, ws_bytes, stream);
  if (rc) return rc;
  if (dweight)
    rc = af3_linear(g, ldg, 1, x, ldx, 1, N, K, T, nullptr, 0, 0, nullptr, 0, dweight, nullptr, workspace, ws_bytes, stream);
  return rc;
}
