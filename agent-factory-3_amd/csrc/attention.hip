// Causal attention over a sliding window, with a sequence's first tokens kept
// visible and one learned sink logit per query head (gpt-oss attention), forward
// and backward.  No kernel of the reference: its models call the attention that
// transformers selects.
//
//   z_ij = scale q_i . k_j over the keys i sees:  lo_i <= j <= min(p_i, hi - 1)
//          and (no window, or j > p_i - window, or j < lo_i + first)
//   o_i  = sum_j e^{z_ij} v_j / (e^{sink} + sum_j e^{z_ij})      (0 where the denominator is 0)
//   delta_i = do_i . o_i,  p_ij = e^{z_ij - lse_i},  dz_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j dz_ij k_j,  dk_j = scale sum_i dz_ij q_i,  dv_j = sum_i p_ij do_i,
//   dsink = -sum_i e^{sink - lse_i} delta_i
//
// with p_i = i + (Sk - Sq) (the last query is the last key), lo / hi the batch
// row's key range, or lo_i the start of token i's sequence in a packed row.
//
// Rows.  The G query heads of a key/value head are rows of one tile: row r of a
// tile is (token r / G, head r % G), so a K / V tile in LDS serves every head
// that shares it, a 128-row tile spans only 128 / G tokens (a window of 128
// costs few keys beyond it), the gradients of a shared K / V row are one sum in
// registers, and a single token fills G rows.
//
// Layouts.  All products run on v_mfma_f32_32x32x16_bf16 with the tile's own
// row (query in forward and dq, key in dk / dv) in the lane and the other side
// in the 16 accumulator registers, register r of half h holding entry
// 8 (r / 4) + 4 h + r % 4.  Row statistics are then one value per lane, and the
// probabilities (rounded to bf16, as the operand needs) are the next product's
// B operand where they lie: a contraction may take its 16 entries in any order
// that both operands share, so the other operand's transposing LDS reads
// (ds_read_b64_tr_b16) fetch entries 4 h .. 4 h + 3 and 8 + 4 h .. in the
// accumulators' order.  Sums, statistics and the accumulators are fp32.
#include "af3_common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxLen = 1 << 29;   // tokens (positions and their sums with a window stay in 32 bits)
constexpr int kMaxStride = 1 << 23; // elements between heads or tokens (128 of them within 32-bit byte offsets)
constexpr float kLowest = -1e30f;  // running maximum of a row that has seen nothing (finite: -inf - it is -inf)

struct SaParams {
  const uint16_t *q, *k, *v;              // [B][H][S][D] by strides, D contiguous
  int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st;
  const void* sinks;                      // [Hq] or NULL
  int sinks_f32;
  const int32_t* starts;                  // [B][Sk] start of each token's sequence (packed rows), or NULL
  const int32_t* kv_range;                // [B][2] or NULL
  int B, Hq, Hkv, G, Sq, Sk, window, first;
  int g_mul;                              // x / G = x g_mul >> 16 for x < 256
  int tok;                                // tokens of a row tile
  int n_tiles, n_split;
  float scale, scale2;                    // scale2 = scale log2(e)
  uint16_t* out;                          // [B][Sq][Hq][D]
  float* lse;                             // [B][Hkv][Sq][G], log2 units; or NULL
  float* part;                            // n_split > 1: [n_split][B][Hkv][Sq][G][D] then (m, l) pairs
  // backward
  const uint16_t* dout;                   // [B][Sq][Hq][D] by strides
  int64_t do_sb, do_sh, do_st;
  float* delta;                           // -delta, as lse
  float* dsink_part;                      // [n_tiles][B][Hq]
  uint16_t *dq, *dk, *dv;                 // [B][S][H][D]
  void* dsinks;                           // [Hq], in the sinks' type
  int n_key_blocks;
};

__device__ __forceinline__ void a_dma16(const void* gptr, uint32_t lds_byte_addr) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(gptr), "{m0}"(lds_byte_addr) : "memory");
}
// the same from a wave-uniform base plus a 32-bit lane offset in bytes
__device__ __forceinline__ void a_dma16_s(const void* sbase, uint32_t voff, uint32_t lds_byte_addr) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "{m0}"(lds_byte_addr) : "memory");
}
// four bytes per lane
__device__ __forceinline__ void a_dma4(const void* gptr, uint32_t lds_byte_addr) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(gptr), "{m0}"(lds_byte_addr) : "memory");
}
__device__ __forceinline__ void a_dma4_s(const void* sbase, uint32_t voff, uint32_t lds_byte_addr) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(voff), "s"(sbase), "{m0}"(lds_byte_addr) : "memory");
}
#define A_WAIT_VM(n) asm volatile("s_waitcnt vmcnt(" #n ")" ::: "memory")
#define A_BARRIER() asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory")

__device__ __forceinline__ uint32_t a_lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// XOR of a row's 16-byte chunk index.  A 16-byte read takes 16 rows' equal chunks
// at a time, a transposing read 4 rows' 4 chunks per half wave; over 64 banks (256
// bytes: two rows of D = 64, one of 128) both then fall into distinct bank groups.
template <int D>
__device__ __forceinline__ int a_swz(int row) {
  if constexpr (D == 64)
    return ((row & 2) << 1) | ((row >> 1) & 2) | ((row >> 3) & 1);
  else
    return ((row & 3) << 2) | ((row >> 2) & 3);
}

template <int D>
__device__ __forceinline__ int a_off(int row, int chunk) { return row * (D * 2) + ((chunk ^ a_swz<D>(row)) << 4); }

// A lane's LDS offsets of the operands it reads from a [rows][D] tile.  The
// swizzle depends on a row's low four bits alone, so the same rows further down
// are a constant away.
template <int D>
struct Frag {
  uint32_t row[D / 16], tr[D / 32], tr8_[D / 32];
  // base: added to every address (the tile's own, where `tile` is then a constant
  // that fits the reads' offset field)
  __device__ __forceinline__ explicit Frag(int lane, uint32_t base = 0) {
    const int r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int x = 0; x < D / 16; ++x) row[x] = base + a_off<D>(r, 2 * x + h);
    const int tr_r = (h << 2) + ((lane & 15) >> 2);
    const int c = (((lane >> 4) & 1) << 4) + ((lane & 3) << 2);
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
      tr[d] = base + a_off<D>(tr_r, (d * 32 + c) >> 3) + ((c & 7) << 1);
      tr8_[d] = base + a_off<D>(tr_r + 8, (d * 32 + c) >> 3) + ((c & 7) << 1);
    }
  }
  // chunk 2 x + h of row r0 + lane % 32 of the tile at LDS address `tile` (r0 % 32 == 0)
  __device__ __forceinline__ af3_bf16x8 row8(uint32_t tile, int r0, int x) const {
    typedef const __attribute__((address_space(3))) af3_bf16x8 T;
    return *(T*)(uintptr_t)(tile + row[x] + (uint32_t)(r0 * D * 2));
  }
  // rows r0 + 4 h .. + 3 and r0 + 8 + 4 h .. + 3 of column 32 d + lane % 32 (r0 % 16 == 0)
  __device__ __forceinline__ af3_bf16x8 tr8(uint32_t tile, int r0, int d) const {
    const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(uintptr_t)(tile + tr[d] + (uint32_t)(r0 * D * 2)));
    const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(uintptr_t)(tile + tr8_[d] + (uint32_t)(r0 * D * 2)));
    return af3_bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
};

template <int V>
struct Int {
  static constexpr int value = V;
};

// The loads of these operands end here.  Left to their first use in the loop, the
// compiler's wait for them would stand there in every step and wait for the
// step's copies to LDS too, which it does not know of.
template <int N>
__device__ __forceinline__ void a_landed(af3_bf16x8 (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

__device__ __forceinline__ af3_f32x16 a_mfma(af3_bf16x8 a, af3_bf16x8 b, af3_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ af3_f32x16 a_zero() {
  af3_f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// registers 8 t .. 8 t + 7 of an accumulator as a bf16 operand
__device__ __forceinline__ af3_bf16x8 a_pack8(const af3_f32x16& p, int t) {
  af3_u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = af3_pack_bf16x2(p[8 * t + 2 * i], p[8 * t + 2 * i + 1]);
  return __builtin_bit_cast(af3_bf16x8, w);
}

// over a lane and its partner in the other half (lane ^ 32)
__device__ __forceinline__ float a_max_halves(float x) {
  const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float a_sum_halves(float x) {
  const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// a row number's distance, kept where 32 bits hold it (a step has 64 rows)
__device__ __forceinline__ int a_clamp64(int64_t x) { return (int)min(max(x, (int64_t)-1024), (int64_t)1024); }

__device__ __forceinline__ float a_sink2(const SaParams& p, int h) {
  const float s = (p.sinks_f32 ? ((const float*)p.sinks)[h] : af3_bf16_to_f32(((const uint16_t*)p.sinks)[h])) * kLog2e;
  return s > 3e38f ? 3e38f : s;  // (finite: nothing is left of any key either way; a NaN stays one)
}

// key range of a batch row, inside [0, Sk] whatever the tensor holds
__device__ __forceinline__ void a_kv_range(const SaParams& p, int b, int& lo, int& hi) {
  lo = 0;
  hi = p.Sk;
  if (p.kv_range) {
    lo = min(max(p.kv_range[2 * b], 0), p.Sk);
    hi = min(max(p.kv_range[2 * b + 1], lo), p.Sk);
  }
}

// the sequence starts of a batch row's tokens, or NULL
__device__ __forceinline__ const int32_t* a_starts(const SaParams& p, int b) {
  return p.starts ? p.starts + (int64_t)b * p.Sk : nullptr;
}

// What a row sees: keys [w, end) (the window, or all) and the fn keys from lo
// (the kept first tokens)
struct Vis {
  int w, end, lo, fn;
};

__device__ __forceinline__ Vis a_vis(const SaParams& p, int pos, int lo, int hi) {
  Vis v;
  v.lo = lo;
  v.end = min(pos + 1, hi);
  v.w = p.window > 0 ? max(lo, pos - p.window + 1) : lo;
  v.fn = max(0, min(p.first, v.end - lo));
  return v;
}

// The first and the last of tokens t0 .. t1 that lie in a sequence (k0 > k1 where none
// does): of a packed row, tokens before the first sequence or past the last have
// starts[t] = t + 1.  Their keys and rows are left out of every product, whatever they
// hold, as those outside a key range are; only a tile at an end of the row looks.
__device__ __forceinline__ void a_live(const int32_t* starts, int t0, int t1, int lane, int& k0, int& k1) {
  k0 = t1 + 1;
  k1 = t0 - 1;
  for (int t = t0; t <= t1; t += 64) {
    const uint64_t in = __ballot(t + lane <= t1 && starts[t + lane] <= t + lane);
    if (in == 0) continue;
    if (k0 > t1) k0 = t + __builtin_ctzll(in);
    k1 = t + 63 - __builtin_clzll(in);
  }
}

// scores of keys at or past `end` / before `from` to `to`; register r of s[c] is
// key j + 32 c + 8 (r / 4) + r % 4
template <int N>
__device__ __forceinline__ void a_mask_end(af3_f32x16 (&s)[N], int j, int end, float to) {
#pragma unroll
  for (int c = 0; c < N; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[c][r] = c * 32 + 8 * (r / 4) + r % 4 < end - j ? s[c][r] : to;
}
template <int N>
__device__ __forceinline__ void a_mask_from(af3_f32x16 (&s)[N], int j, int from, float to) {
#pragma unroll
  for (int c = 0; c < N; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[c][r] = c * 32 + 8 * (r / 4) + r % 4 >= from - j ? s[c][r] : to;
}
// keys outside both of a row's runs
template <int N>
__device__ __forceinline__ void a_mask_both(af3_f32x16 (&s)[N], int j, const Vis& v, float to) {
  const uint32_t n = max(0, v.end - v.w);
#pragma unroll
  for (int c = 0; c < N; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int x = j + c * 32 + 8 * (r / 4) + r % 4;
      s[c][r] = (uint32_t)(x - v.w) < n || (uint32_t)(x - v.lo) < (uint32_t)v.fn ? s[c][r] : to;
    }
}

// The keys a row tile runs over: [a0, a1) are first tokens before the window,
// [b0, b1) the rest; unions over the tile's rows.
struct Keys {
  int a0, a1, b0, b1;
};

__device__ __forceinline__ Keys a_keys(const SaParams& p, int pos0, int pos1, int lo, int hi) {
  Keys s;
  s.b1 = min(hi, pos1 + 1);
  s.b0 = p.window > 0 ? max(lo, pos0 - p.window + 1) : lo;
  s.a0 = lo;
  s.a1 = min(lo + p.first, min(s.b0, s.b1));
  return s;
}

// ---------------------------------------------------------------------------
// forward.  Block = 4 waves of 32 rows; 64-key tiles through LDS, K round two
// stages and V round three (global->LDS copies a tile ahead, one barrier per
// tile; 40 KB at D = 64, so four blocks share a CU).  S^T = K Q^T puts a row's
// scores into its lane; the running maximum moves only when it grows by more
// than 8 (log2 units: probabilities stay below 256), so most tiles need no
// rescaling of the output.  Probabilities are rounded to bf16 for the product
// with V, their sum is not: the output is 1.3 times one bf16 rounding off.  Scores
// are fp32: a probability is off by its score's rounding (2^-24 of it), and scores
// past 2^29 overflow in the exponential.
//
// Bound by the vector unit, not the matrix unit: an exponential issues over 16
// cycles, so 32 keys of 32 rows cost 256 cycles of them next to 256 of the two
// products; the counters give 87% of the cycles to the vector unit and 48% to
// the matrix unit.  8192 packed rows of 2144 keys on average, 64 heads over 8,
// D 64: 340 to 357 us by the card (845 to 805 TFLOP/s); a window of 128: 54 us; 2 x
// 4096 rows: 315 to 337 us.  Where a wave's rows are few the tiles are read at
// memory speed: one token over 131072 keys 43 us (6.2 TB/s), 32 tokens over 4099: 26.7 us (5.1).
// A window's block runs three to four tiles, so its start (first copies, q rows)
// is a third of it.  Stages as constants of six unrolled turns gain 3% on the
// long rows and lose 10% on the window (code fetched once per block), so the
// stages stay variables here.
// ---------------------------------------------------------------------------
constexpr int kRows = 128;  // rows of a tile
constexpr int kBN = 64;     // keys of a tile
constexpr int kMaxSplit = 256;

// K (or V) tiles of 64 rows into LDS by the block's 4 waves.  A whole tile's
// copies take the tile's address (scalar) and lane offsets that never change; a
// tile that ends early repeats its last row.
template <int D>
struct KvCopy {
  static constexpr int CH = D / 8;         // chunks per row
  static constexpr int RPI = 64 / CH;      // rows per copy
  static constexpr int N = kBN / RPI / 4;  // copies per wave
  const uint16_t* base;
  int64_t st;
  uint32_t off[N];
  int row0;  // the lane's row of copy x: row0 + x RPI
  __device__ __forceinline__ KvCopy(const uint16_t* base_, int64_t st_, int wave, int lane) : base(base_), st(st_) {
    row0 = wave * N * RPI + lane / CH;
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const int row = row0 + x * RPI;
      off[x] = (uint32_t)(row * (int)st + (((lane % CH) ^ a_swz<D>(row)) << 3)) * 2;
    }
  }
  __device__ __forceinline__ void operator()(int j0, int last, uint32_t lds, int wave) const {
    const uint16_t* t = base + j0 * st;
    const uint32_t at = lds + (uint32_t)(wave * N * 1024);
    if (j0 + kBN - 1 <= last) {
#pragma unroll
      for (int x = 0; x < N; ++x) a_dma16_s(t, off[x], at + x * 1024);
    } else {
#pragma unroll
      for (int x = 0; x < N; ++x) {
        const int over = max(0, row0 + x * RPI - (last - j0));
        a_dma16_s(t, off[x] - (uint32_t)(over * (int)st) * 2, at + x * 1024);
      }
    }
  }
};

template <int D>
__global__ __launch_bounds__(256, D == 64 ? 4 : 2) void sa_fwd_kernel(SaParams p) {
  constexpr int KS = D / 16, DB = D / 32;
  constexpr int kTile = kBN * D * 2;
  __shared__ __attribute__((aligned(16))) uint8_t lds[5 * kTile];
  const int bh = blockIdx.x % (p.B * p.Hkv);
  const int rest = blockIdx.x / (p.B * p.Hkv);
  const int split = p.n_split > 1 ? rest % p.n_split : 0;
  const int tile = p.n_tiles - 1 - (p.n_split > 1 ? rest / p.n_split : rest);  // the longest rows first
  const int b = p.B > 1 ? bh / p.Hkv : 0, hk = bh - b * p.Hkv;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 31, lh = lane >> 5;
  const int off = p.Sk - p.Sq;
  const int t0 = tile * p.tok, t1 = min(t0 + p.tok, p.Sq) - 1;  // tokens of the tile
  int lo, hi;
  a_kv_range(p, b, lo, hi);
  const int32_t* starts = a_starts(p, b);
  const int tile_lo = starts ? starts[t0] : lo;
  const int last_lo = starts ? starts[t1] : lo;  // the last sequence's start (the latest)
  Keys ks = a_keys(p, t0 + off, t1 + off, tile_lo, hi);
  int na, nb, i0, i1;  // tiles of first tokens, of the rest, and the block's own
  auto tiles = [&]() {
    na = max(0, (ks.a1 - ks.a0 + kBN - 1) / kBN), nb = max(0, (ks.b1 - ks.b0 + kBN - 1) / kBN);
    i0 = 0, i1 = na + nb;
    if (p.n_split > 1) {
      const int per = (na + nb + p.n_split - 1) / p.n_split;
      i0 = min(split * per, na + nb);
      i1 = min(i0 + per, na + nb);
    }
  };
  tiles();
  const KvCopy<D> kc(p.k + b * p.k_sb + hk * p.k_sh, p.k_st, wave, lane);
  const KvCopy<D> vc(p.v + b * p.v_sb + hk * p.v_sh, p.v_st, wave, lane);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(a_lds_addr(lds));
  auto first_key = [&](int i) { return i < na ? ks.a0 + i * kBN : ks.b0 + (i - na) * kBN; };
  // K and V of tile i; K goes round two stages, V round three
  auto load = [&](int i, int kst, int vst) {
    const int j0 = first_key(i), last = (i < na ? ks.a1 : ks.b1) - 1;
    kc(j0, last, lds0 + (uint32_t)(kst * kTile), wave);
    vc(j0, last, lds0 + (uint32_t)((2 + vst) * kTile), wave);
  };
  if (i0 < i1) load(i0, 0, 0);
  if (i0 + 1 < i1) load(i0 + 1, 1, 1);
  // Tokens in no sequence: the copies again, without them.  (Looked for before the
  // first copies, they cost a window's forward 3%: 56.0 us instead of 54.3.)
  if (__builtin_expect(starts && (tile_lo > t0 || last_lo > t1), 0)) {
    int k0, k1;
    a_live(starts, t0, t1, lane, k0, k1);
    ks = a_keys(p, k0 + off, k1 + off, k0 <= k1 ? starts[k0] : k0, hi);
    tiles();
    A_WAIT_VM(0);
    if (i0 < i1) load(i0, 0, 0);
    if (i0 + 1 < i1) load(i0 + 1, 1, 1);
  }

  const int row = wave * 32 + lr;
  const int tk = row * p.g_mul >> 16, g = row - tk * p.G;
  const bool valid = t0 + tk <= t1;
  const int t = valid ? t0 + tk : t0;
  const int head = hk * p.G + (valid ? g : 0);
  const Vis vis = a_vis(p, t + off, starts ? starts[t] : lo, hi);
  af3_bf16x8 qf[KS];
  {
    const uint16_t* qr = p.q + b * p.q_sb + head * p.q_sh + t * p.q_st;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *(const af3_bf16x8*)(qr + s * 16 + lh * 8);
  }
  float m = kLowest, l = 0.f;
  if (p.sinks && split == 0) {
    const float s2 = a_sink2(p, head);
    m = fmaxf(s2, kLowest);
    l = lh == 0 ? __builtin_amdgcn_exp2f(s2 - m) : 0.f;
  }
  a_landed(qf);
  af3_f32x16 o[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = a_zero();

  // The wave's positions; its tiles [own0, own1) (the others hold nothing that its
  // rows see) and among them [free0, free1), of which its rows see every key.
  const int wt0 = t0 + (wave * 32 * p.g_mul >> 16), wt1 = min(t1, t0 + ((wave * 32 + 31) * p.g_mul >> 16));
  const int wpos0 = wt0 + off, wpos1 = wt1 + off;
  const int from = p.window > 0 ? max(last_lo + p.first, wpos1 - p.window + 1) : last_lo;
  const int own1 = wt0 > t1 ? 0 : min(i1, na + max(0, wpos1 - ks.b0 + kBN) / kBN);
  const int own0 = p.window > 0 && p.first == 0 ? max(i0, na + max(0, wpos0 - p.window + 1 - ks.b0) / kBN) : i0;
  const int free0 = na + max(0, from - ks.b0 + kBN - 1) / kBN;
  const int free1 = na + max(0, min(wpos0 + 1, ks.b1) - ks.b0) / kBN;
  const Frag<D> fr(lane);

  // the softmax of 32 keys (half c of tile i) and their product with V; beside it the scores of the next 32
  auto step = [&](int i, int c, uint32_t vt, af3_f32x16 (&s)[1], uint32_t kt, af3_f32x16& next) {
    // (past the last tile these are what the ring holds, and nothing reads their scores)
    af3_bf16x8 kf[KS];
#pragma unroll
    for (int x = 0; x < KS; ++x) kf[x] = fr.row8(kt, (c ^ 1) * 32, x);
    if (i < free0 || i >= free1) {
      const int j = first_key(i) + c * 32;
      if (i < na) {  // first tokens before the window
        a_mask_end(s, j + 4 * lh, min(vis.lo + vis.fn, ks.a1), -INFINITY);
        a_mask_from(s, j + 4 * lh, vis.lo, -INFINITY);
      } else if (p.first > 0 && j < last_lo + p.first) {
        a_mask_both(s, j + 4 * lh, vis, -INFINITY);
      } else {
        if (j + 31 > wpos0 || j + 32 > ks.b1) a_mask_end(s, j + 4 * lh, vis.end, -INFINITY);
        if (j < from) a_mask_from(s, j + 4 * lh, vis.w, -INFINITY);
      }
    }
    float mx = s[0][0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[0][r]);
    mx = a_max_halves(mx) * p.scale2;
    if (__any(mx > m + 8.f)) {
      const float nm = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f(m - nm);
      m = nm;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
    }
    // Written in the order in which it has to issue (the barriers hold it): each
    // score product of the next keys has exponentials behind it, which run while
    // the matrix unit is busy, and the first half's product with V stands between
    // the second half's exponentials.
    af3_bf16x8 vf[DB], pf;
    next = a_zero();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      next = a_mfma(kf[x], qf[x], next);
      if (x == KS / 2 - 1)
#pragma unroll
        for (int d = 0; d < DB; ++d) vf[d] = fr.tr8(vt, c * 32, d);
      if (x == KS / 2) pf = a_pack8(s[0], 0);
      if (x >= KS / 2) o[x - KS / 2] = a_mfma(vf[x - KS / 2], pf, o[x - KS / 2]);
#pragma unroll
      for (int r = x * (16 / KS); r < (x + 1) * (16 / KS); ++r) {
        s[0][r] = __builtin_amdgcn_exp2f(fmaf(s[0][r], p.scale2, -m));
        l += s[0][r];
      }
      if (x == KS - 1)
#pragma unroll
        for (int d = 0; d < DB; ++d) vf[d] = fr.tr8(vt, c * 32 + 16, d);
      __builtin_amdgcn_sched_barrier(0);
    }
    pf = a_pack8(s[0], 1);
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = a_mfma(vf[d], pf, o[d]);
  };
  // K of tile i is done with after the scores of its second half (two stages), V
  // after its second half's product (three)
  af3_f32x16 sa[1], sb[1];
  A_WAIT_VM(0);
  A_BARRIER();
  if (own0 == i0 && i0 < own1) {
    sa[0] = a_zero();
#pragma unroll
    for (int x = 0; x < KS; ++x) sa[0] = a_mfma(fr.row8(lds0, 0, x), qf[x], sa[0]);
  }
  int kst = 0, vst = 0;
  for (int i = i0; i < i1; ++i) {
    const bool mine = i >= own0 && i < own1;
    const uint32_t vt = lds0 + (uint32_t)((2 + vst) * kTile);
    if (mine) step(i, 0, vt, sa, lds0 + (uint32_t)(kst * kTile), sb[0]);
    A_WAIT_VM(0);  // K and V of tile i + 1
    A_BARRIER();   // and every wave is past K of tile i and V of tile i - 1
    vst = vst == 2 ? 0 : vst + 1;
    if (i + 2 < i1) load(i + 2, kst, vst == 2 ? 0 : vst + 1);
    kst ^= 1;
    const uint32_t kt = lds0 + (uint32_t)(kst * kTile);
    if (mine) {
      step(i, 1, vt, sb, kt, sa[0]);
    } else if (i + 1 == own0) {
      sa[0] = a_zero();
#pragma unroll
      for (int x = 0; x < KS; ++x) sa[0] = a_mfma(fr.row8(kt, 0, x), qf[x], sa[0]);
    }
  }
  l = a_sum_halves(l);
  if (!valid) return;
  const int64_t prow = (((int64_t)b * p.Hkv + hk) * p.Sq + t) * p.G + g;
  if (p.n_split > 1) {
    const int64_t rows = (int64_t)p.B * p.Hkv * p.Sq * p.G;
    float* po = p.part + (split * rows + prow) * D;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *(float4*)(po + d * 32 + 2 * r + 4 * lh) = float4{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
    if (lh == 0) *(float2*)(p.part + p.n_split * rows * D + (split * rows + prow) * 2) = float2{m, l};
    return;
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // (a NaN stays one)
  const int64_t orow = (((int64_t)b * p.Sq + t) * p.Hq + head) * D;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      u32x2 w;
#pragma unroll
      for (int x = 0; x < 2; ++x) w[x] = af3_pack_bf16x2(o[d][r + 2 * x] * inv, o[d][r + 2 * x + 1] * inv);
      *(u32x2*)(p.out + orow + d * 32 + 2 * r + 4 * lh) = w;
    }
  if (p.lse && lh == 0) p.lse[prow] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// joins the splits of a row: one block per row, each wave a quarter of the splits
// (64 rows of 64 splits: 4.0 us, a launch's latency and two dependent loads)
template <int D>
__global__ __launch_bounds__(256) void sa_join_kernel(SaParams p) {
  __shared__ float sw[kMaxSplit], so[4][D], sl[4];
  const int64_t rows = (int64_t)p.B * p.Hkv * p.Sq * p.G;
  const int64_t prow = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float* ml = p.part + p.n_split * rows * D;
  const int s0 = threadIdx.x;
  const float2 x = s0 < p.n_split ? *(const float2*)(ml + (s0 * rows + prow) * 2) : float2{kLowest, 0.f};
  float m = x.x;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if (lane == 0) sl[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sl[0], sl[1]), fmaxf(sl[2], sl[3]));
  const float w = __builtin_amdgcn_exp2f(x.x - m);
  sw[s0] = w;
  float l = w * x.y;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  __syncthreads();
  if (lane == 0) sl[wave] = l;
  float o[D / 64] = {};
  const float* po = p.part + prow * D + lane;
#pragma unroll 8
  for (int s = wave; s < p.n_split; s += 4)
#pragma unroll
    for (int d = 0; d < D / 64; ++d) o[d] = fmaf(sw[s], po[s * rows * D + d * 64], o[d]);
#pragma unroll
  for (int d = 0; d < D / 64; ++d) so[wave][d * 64 + lane] = o[d];
  __syncthreads();
  l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const int g = (int)(prow % p.G);
  const int64_t u = prow / p.G;
  const int t = (int)(u % p.Sq);
  const int bh = (int)(u / p.Sq), b = bh / p.Hkv, hk = bh % p.Hkv;
  const int64_t orow = (((int64_t)b * p.Sq + t) * p.Hq + hk * p.G + g) * D;
  if ((int)threadIdx.x < D) {
    const int d = threadIdx.x;
    p.out[orow + d] = (uint16_t)af3_f32_to_bf16(((so[0][d] + so[1][d]) + (so[2][d] + so[3][d])) * inv);
  }
  if (p.lse && threadIdx.x == 0) p.lse[prow] = l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l);
}

// ---------------------------------------------------------------------------
// backward, queries: dq, delta and the sinks' partial sums.  The forward's
// tiles and layouts; p comes back from the saved log-sum.
//
// delta.  do . out of the rounded output is off by 2^-9 |do| |out|, which would
// be the largest error of the whole backward (the error of out is that of every
// key's probability and of its own rounding): dq 1.66, dk 1.58 times one bf16
// rounding.  So a tile uses that delta0, and the sums of dz and p k beside dz k
// give the true one at the end: sum dz = delta - delta0 sum p, sum p = 1 - p_sink,
// and dq = scale (sum dz k - (delta - delta0) sum p k).  dk, dv and the sinks take
// the true delta: dq 1.44, dk 1.41 times one rounding (of dz, and the result's),
// dsinks none.  (Means over 400 heads: single calls of eight heads and two tokens
// scatter between 1.1 and 1.9, since there one rounded dz scales a whole row.)  The
// bf16 remainder of out kept by the forward costs more (its writing alone 15 us of
// 70 with a window of 128) and corrects less (dq 1.53).
//
// Four products per step on the matrix unit; the second accumulator takes the
// registers of a third block per CU.  8192 packed rows, 64 heads over 8, D 64: 544
// to 577 us by the card (of 2144 keys on average; 4 products: 1060 to 1000 TFLOP/s),
// matrix unit busy 56%, vector unit 54%; 103 us with a window of 128, where half is
// a block's start: q, dout and out rows and the first tiles, 5 us for each of the
// two blocks a CU holds.
// ---------------------------------------------------------------------------
template <int D>
__global__ __launch_bounds__(256, D == 64 ? 2 : 1) void sa_dq_kernel(SaParams p) {
  constexpr int KS = D / 16, DB = D / 32;
  constexpr int kTile = kBN * D * 2;
  __shared__ __attribute__((aligned(16))) uint8_t lds[4 * kTile];
  __shared__ float ds_row[kRows];
  const int bh = blockIdx.x % (p.B * p.Hkv);
  const int tile = p.n_tiles - 1 - blockIdx.x / (p.B * p.Hkv);
  const int b = p.B > 1 ? bh / p.Hkv : 0, hk = bh - b * p.Hkv;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 31, lh = lane >> 5;
  const int off = p.Sk - p.Sq;
  const int t0 = tile * p.tok, t1 = min(t0 + p.tok, p.Sq) - 1;
  int lo, hi;
  a_kv_range(p, b, lo, hi);
  const int32_t* starts = a_starts(p, b);
  const int tile_lo = starts ? starts[t0] : lo;
  const int last_lo = starts ? starts[t1] : lo;  // the last sequence's start (the latest)
  Keys ks = a_keys(p, t0 + off, t1 + off, tile_lo, hi);
  int na, nb;
  auto tiles = [&]() {
    na = max(0, (ks.a1 - ks.a0 + kBN - 1) / kBN), nb = max(0, (ks.b1 - ks.b0 + kBN - 1) / kBN);
  };
  tiles();
  const KvCopy<D> kc(p.k + b * p.k_sb + hk * p.k_sh, p.k_st, wave, lane);
  const KvCopy<D> vc(p.v + b * p.v_sb + hk * p.v_sh, p.v_st, wave, lane);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(a_lds_addr(lds));
  auto first_key = [&](int i) { return i < na ? ks.a0 + i * kBN : ks.b0 + (i - na) * kBN; };
  auto issue = [&](int i, int stage) {
    const int j0 = first_key(i), last = (i < na ? ks.a1 : ks.b1) - 1;
    const uint32_t st = lds0 + (uint32_t)(stage * 2 * kTile);
    kc(j0, last, st, wave);
    vc(j0, last, st + kTile, wave);
  };
  if (na + nb > 0) issue(0, 0);  // (under way while the rows are read)
  if (__builtin_expect(starts && (tile_lo > t0 || last_lo > t1), 0)) {  // as in the forward
    int k0, k1;
    a_live(starts, t0, t1, lane, k0, k1);
    ks = a_keys(p, k0 + off, k1 + off, k0 <= k1 ? starts[k0] : k0, hi);
    tiles();
    A_WAIT_VM(0);
    if (na + nb > 0) issue(0, 0);
  }

  const int row = wave * 32 + lr;
  const int tk = row * p.g_mul >> 16, g = row - tk * p.G;
  const bool valid = t0 + tk <= t1;
  const int t = valid ? t0 + tk : t0;
  const int head = hk * p.G + (valid ? g : 0);
  const int64_t prow = (((int64_t)b * p.Hkv + hk) * p.Sq + t) * p.G + (valid ? g : 0);
  const Vis vis = a_vis(p, t + off, starts ? starts[t] : lo, hi);
  float lse = p.lse[prow];
  af3_bf16x8 qf[KS], df[KS];
  float delta = 0.f;
  {
    const uint16_t* qr = p.q + b * p.q_sb + head * p.q_sh + t * p.q_st;
    const uint16_t* dr = p.dout + b * p.do_sb + head * p.do_sh + t * p.do_st;
    const int64_t orow = (((int64_t)b * p.Sq + t) * p.Hq + head) * D;
    af3_bf16x8 of[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      qf[s] = *(const af3_bf16x8*)(qr + s * 16 + lh * 8);
      df[s] = *(const af3_bf16x8*)(dr + s * 16 + lh * 8);
      of[s] = *(const af3_bf16x8*)(p.out + orow + s * 16 + lh * 8);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 8; ++i) delta = fmaf((float)df[s][i], (float)of[s][i], delta);
    // (a row that sees nothing has no gradient, whatever its dout holds)
    delta = a_sum_halves(delta);
    delta = vis.w < vis.end || vis.fn > 0 ? delta : 0.f;
    a_landed(qf);
    a_landed(df);
  }
  asm volatile("" : "+v"(lse));  // landed, as the operands
  // the wave's own tiles and those of which its rows see every key, as in the forward
  const int wt0 = t0 + (wave * 32 * p.g_mul >> 16), wt1 = min(t1, t0 + ((wave * 32 + 31) * p.g_mul >> 16));
  const int wpos0 = wt0 + off, wpos1 = wt1 + off;
  const int from = p.window > 0 ? max(last_lo + p.first, wpos1 - p.window + 1) : last_lo;
  const int own1 = wt0 > t1 ? 0 : min(na + nb, na + max(0, wpos1 - ks.b0 + kBN) / kBN);
  const int own0 = p.window > 0 && p.first == 0 ? na + max(0, wpos0 - p.window + 1 - ks.b0) / kBN : 0;
  const int free0 = na + max(0, from - ks.b0 + kBN - 1) / kBN;
  const int free1 = na + max(0, min(wpos0 + 1, ks.b1) - ks.b0) / kBN;
  const Frag<D> fr(lane, lds0);
  af3_f32x16 acc[DB], pk[DB];  // sum dz k and sum p k
  float dsum = 0.f;            // sum dz
#pragma unroll
  for (int d = 0; d < DB; ++d) acc[d] = a_zero(), pk[d] = a_zero();
  auto turn = [&](int i, auto stage) {  // (the stage a constant: its addresses need no arithmetic)
    A_WAIT_VM(0);
    A_BARRIER();
    if (i + 1 < na + nb) issue(i + 1, 1 - stage.value);
    constexpr uint32_t kt = stage.value * 2 * kTile, vt = kt + kTile;
    if (i < own0 || i >= own1) return;
    // Written in the order in which it has to issue (the barriers hold it): reads ahead
    // of their use, the first half's exponentials beside the second's scores, its
    // products beside the second's exponentials (without: 572 us, with 548, on one card).
    af3_bf16x8 ka[KS], va[KS], kb[KS], vb[KS], tr[DB], ts[DB];
    af3_f32x16 s0[1] = {a_zero()}, s1[1] = {a_zero()}, d0[1], d1[1];
    const bool whole = i >= free0 && i < free1;
    // (dz is set to zero too, not p alone: whatever stands at a key that the row does not see)
    auto mask = [&](int j, af3_f32x16 (&x)[1]) {
      if (i < na) {
        a_mask_end(x, j + 4 * lh, min(vis.lo + vis.fn, ks.a1), 0.f);
        a_mask_from(x, j + 4 * lh, vis.lo, 0.f);
      } else if (p.first > 0 && j < last_lo + p.first) {
        a_mask_both(x, j + 4 * lh, vis, 0.f);
      } else {
        if (j + 31 > wpos0 || j + 32 > ks.b1) a_mask_end(x, j + 4 * lh, vis.end, 0.f);
        if (j < from) a_mask_from(x, j + 4 * lh, vis.w, 0.f);
      }
    };
    auto exps = [&](af3_f32x16& x, int r0, int n) {
#pragma unroll
      for (int r = r0; r < r0 + n; ++r) x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], p.scale2, -lse));
    };
#pragma unroll
    for (int x = 0; x < KS; ++x) ka[x] = fr.row8(kt, 0, x);
#pragma unroll
    for (int x = 0; x < KS; ++x) va[x] = fr.row8(vt, 0, x);
#pragma unroll
    for (int r = 0; r < 16; ++r) d0[0][r] = d1[0][r] = -delta;
#pragma unroll
    for (int x = 0; x < KS; ++x) s0[0] = a_mfma(ka[x], qf[x], s0[0]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < KS; ++x) kb[x] = fr.row8(kt, 32, x);
#pragma unroll
    for (int x = 0; x < KS; ++x) d0[0] = a_mfma(va[x], df[x], d0[0]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      s1[0] = a_mfma(kb[x], qf[x], s1[0]);
      vb[x] = fr.row8(vt, 32, x);
      exps(s0[0], x * (16 / KS), 16 / KS);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) tr[d] = fr.tr8(kt, 0, d);
    if (!whole) mask(first_key(i), s0);
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      d1[0] = a_mfma(vb[x], df[x], d1[0]);
#pragma unroll
      for (int r = x * (16 / KS); r < (x + 1) * (16 / KS); ++r) d0[0][r] *= s0[0][r];
      if (x >= KS / 2) {
        const int d = x - KS / 2;
        ts[d] = fr.tr8(kt, 16, d);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (!whole) mask(first_key(i), d0);
    {
      const af3_bf16x8 z0 = a_pack8(d0[0], 0), p0 = a_pack8(s0[0], 0), z1 = a_pack8(d0[0], 1), p1 = a_pack8(s0[0], 1);
      constexpr int E = 16 / (2 * DB);  // exponentials beside a pair of products
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        acc[d] = a_mfma(tr[d], z0, acc[d]);
        pk[d] = a_mfma(tr[d], p0, pk[d]);
        exps(s1[0], d * E, E);
        tr[d] = fr.tr8(kt, 32, d);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        acc[d] = a_mfma(ts[d], z1, acc[d]);
        pk[d] = a_mfma(ts[d], p1, pk[d]);
        exps(s1[0], (DB + d) * E, E);
        ts[d] = fr.tr8(kt, 48, d);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (!whole) mask(first_key(i) + 32, s1);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      dsum += d0[0][r];
      d1[0][r] *= s1[0][r];
    }
    if (!whole) mask(first_key(i) + 32, d1);
    const af3_bf16x8 z0 = a_pack8(d1[0], 0), p0 = a_pack8(s1[0], 0), z1 = a_pack8(d1[0], 1), p1 = a_pack8(s1[0], 1);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      acc[d] = a_mfma(tr[d], z0, acc[d]);
      pk[d] = a_mfma(tr[d], p0, pk[d]);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) dsum += d1[0][r];
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      acc[d] = a_mfma(ts[d], z1, acc[d]);
      pk[d] = a_mfma(ts[d], p1, pk[d]);
    }
  };
  for (int i = 0; i < na + nb; i += 2) {
    turn(i, Int<0>{});
    if (i + 1 < na + nb) turn(i + 1, Int<1>{});
  }
  // The row's true delta, sum p dp = sum dz + delta sum p with sum p = 1 - p_sink, and
  // what dq lacks for it: -(true delta - delta) sum p k.
  const float p_sink = p.sinks ? __builtin_amdgcn_exp2f(a_sink2(p, head) - lse) : 0.f;
  const float c = a_sum_halves(dsum) - delta * p_sink;
  delta += c;
  if (valid && lh == 0) p.delta[prow] = -delta;
  if (p.sinks) {
    if (lh == 0) ds_row[row] = valid ? -p_sink * delta : 0.f;
    __syncthreads();
    if ((int)threadIdx.x < p.G) {  // the tile's sum for each of the shared heads, in token order
      float sum = 0.f;
      for (int x = 0; x < p.tok; ++x) sum += ds_row[x * p.G + threadIdx.x];
      p.dsink_part[((int64_t)tile * p.B + b) * p.Hq + hk * p.G + threadIdx.x] = sum;
    }
  }
  if (!valid) return;
  uint16_t* qrow = p.dq + (((int64_t)b * p.Sq + t) * p.Hq + head) * D;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      u32x2 w;
#pragma unroll
      for (int x = 0; x < 2; ++x)
        w[x] = af3_pack_bf16x2(fmaf(-c, pk[d][r + 2 * x], acc[d][r + 2 * x]) * p.scale,
                               fmaf(-c, pk[d][r + 2 * x + 1], acc[d][r + 2 * x + 1]) * p.scale);
      *(u32x2*)(qrow + d * 32 + 2 * r + 4 * lh) = w;
    }
}

// the sinks' gradient of head h from the tiles' sums, in a fixed order (256 threads)
__device__ __forceinline__ void a_dsink(const SaParams& p, int h, float* sh) {
  const int n = p.n_tiles * p.B;
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += 256) s += p.dsink_part[(int64_t)i * p.Hq + h];
  sh[threadIdx.x] = s;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    if (p.sinks_f32)
      ((float*)p.dsinks)[h] = sh[0];
    else
      ((uint16_t*)p.dsinks)[h] = (uint16_t)af3_f32_to_bf16(sh[0]);
  }
}

// ---------------------------------------------------------------------------
// backward, keys: dk and dv.  Block = 64 keys of one key/value head, K and V rows
// in registers; the (token, head) rows that see them go through a four-stage LDS
// ring, 64 at a time (q, dout, and their lse and -delta), from the last rows back.
// Waves 0 and 1 (32 keys each) take the first 32 rows of a step, waves 2 and 3 the
// others, and their sums are joined at the end.  S = Q K^T puts a key's column
// into its lane; the sum over the heads that share the key is the sum over rows,
// and the rows that see a key are one run of row numbers per lane.  A step's
// exponentials stand between the products of the next step's scores and of its
// own first half, held in that order, so that the matrix unit works beside them.
//
// Two passes over the scores (this and dq's) instead of one with atomic sums of
// dq: five products become seven (eight with dq's p k), but every sum has a fixed
// order and no fp32 copy of dq is written and read.  8192 packed rows, 64 heads over
// 8, D 64: 668 to 707 us by the card (of 2144 keys on average; 4 products: 860 to 815
// TFLOP/s), matrix unit busy 50%, the rest LDS reads and the exponentials that do not
// fit beside products; 82 us with a window of 128, where a block's start and its
// partly visible steps count.
// ---------------------------------------------------------------------------
// first token after t0, whose sequence starts at s0, of a later sequence (starts does
// not decrease), or n > t0: 64 probes a round, the answer stays in (lo, hi]
__device__ __forceinline__ int a_sequence_end(const int32_t* starts, int s0, int t0, int n, int lane) {
  int lo = t0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int at = lo + step * (lane + 1);
    const int same = __popcll(__ballot(at < hi && starts[at] == s0));
    hi = min(hi, lo + step * (same + 1));
    lo += step * same;
  }
  return hi;
}

constexpr int kKeys = 64;  // keys of a block
constexpr int kRT = 64;    // rows of a step
constexpr int kStages = 4;

template <int D>
__global__ __launch_bounds__(256, D == 64 ? 2 : 1) void sa_dkv_kernel(SaParams p) {
  constexpr int KS = D / 16, DB = D / 32;
  constexpr int kTile = kRT * D * 2;
  constexpr int CH = D / 8, RPI = 64 / CH, N = kRT / RPI / 4;  // chunks per row, rows per copy, copies per wave
  constexpr int EPS = 16 / (2 * KS);                           // exponentials per product slot
  __shared__ __attribute__((aligned(16))) uint8_t lds[kStages * 2 * kTile];
  // rows' lse, -delta and (where the block holds a sequence's first key) sequence start
  __shared__ __attribute__((aligned(16))) float rowv[kStages][4][kRT];
  if ((int)blockIdx.x >= p.n_key_blocks) {  // the last blocks: the sinks
    a_dsink(p, blockIdx.x - p.n_key_blocks, (float*)lds);
    return;
  }
  const int bh = blockIdx.x % (p.B * p.Hkv);
  const int j0 = (int)(blockIdx.x / (p.B * p.Hkv)) * kKeys;  // the longest columns first
  const int b = p.B > 1 ? bh / p.Hkv : 0, hk = bh - b * p.Hkv;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = wave >> 1;  // rows 32 part .. + 31 of a step
  const int lr = lane & 31, lh = lane >> 5;
  const int off = p.Sk - p.Sq;
  int lo, hi;
  a_kv_range(p, b, lo, hi);
  const int32_t* starts = a_starts(p, b);
  const int jl = min(j0 + kKeys, p.Sk) - 1;  // last key of the block
  const int jw = j0 + (wave & 1) * 32;       // first key of the wave
  const int j = jw + lr;
  const bool kvalid = j <= jl;

  // tokens that may see a key of the block
  int tb = p.Sq, s_last = lo;  // [ta, tb); s_last: the latest start among their sequences
  int j_last = jl;
  if (starts) {
    const int s_first = starts[j0];
    s_last = starts[jl];
    if (__builtin_expect((s_last > jl) | (s_first > j0), 0)) {  // keys in no sequence
      a_live(starts, j0, jl, lane, lo, j_last);
      hi = j_last + 1;
      s_last = lo <= j_last ? starts[j_last] : lo;
    }
  }
  const int ta = max(0, max(j0, lo) - off);
  // (the last key's sequence may have first tokens in the block; an earlier one ends in it)
  if (p.window > 0 && (p.first == 0 || s_last + p.first <= j0)) tb = min(tb, min(jl, hi - 1) + p.window - off);
  if (starts) tb = a_sequence_end(starts, s_last, j_last, tb, lane);
  tb = jl < lo || j0 >= hi ? ta : max(ta, min(tb, p.Sq));
  const int64_t n_rows = (int64_t)(tb - ta) * p.G;
  const int n_steps = (int)((n_rows + kRT - 1) / kRT);
  // Where a sequence starts inside the block (its last at s_last), steps [0, mixed)
  // hold rows of earlier ones, which ask each row for its own start.  The steps
  // before them (they run from the last back) are s_last's alone: keys before it
  // gather anything there, and start again from zero at step mixed - 1.
  const int mixed = starts && s_last > j0 ? ((min(s_last, tb) - ta) * p.G + kRT - 1) / kRT : 0;

  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(a_lds_addr(lds));
  const uint32_t rowv0 = __builtin_amdgcn_readfirstlane(a_lds_addr(rowv));
  const uint16_t* qb = p.q + b * p.q_sb + (int64_t)hk * p.G * p.q_sh;
  const uint16_t* db = p.dout + b * p.do_sb + (int64_t)hk * p.G * p.do_sh;
  const int64_t sb = ((int64_t)b * p.Hkv + hk) * p.Sq * p.G + (int64_t)ta * p.G;
  // Steps run from the last rows back, so that the blocks of a head, which end at
  // the same rows, read them at about the same time.  Copies: where a step's rows
  // are whole tokens, lane offsets never change and the scalar bases move on; else,
  // and in the last rows' step, each row is looked up.  ns: the step to be copied
  // next; nt, ng: token and head of its first row.
  const int back = (int)((n_rows - 1) & (kRT - 1)), back_t = back * p.g_mul >> 16;
  const int adv_t = kRT / p.G, adv_g = kRT - adv_t * p.G;
  const bool even = adv_g == 0;
  int nt = tb - 1 - back_t, ng = p.G - 1 - (back - back_t * p.G), ns = n_steps - 1;
  uint32_t qo[N], od[N];
#pragma unroll
  for (int x = 0; x < N; ++x) {
    const int row = (wave * N + x) * RPI + lane / CH, t = row * p.g_mul >> 16, g = row - t * p.G;
    const int col = ((lane % CH) ^ a_swz<D>(row)) << 3;
    qo[x] = (uint32_t)(t * (int)p.q_st + g * (int)p.q_sh + col) * 2;
    od[x] = (uint32_t)(t * (int)p.do_st + g * (int)p.do_sh + col) * 2;
  }
  const uint16_t *qp = qb + (int64_t)nt * p.q_st, *dp_ = db + (int64_t)nt * p.do_st;  // (even: ng is 0)
  const float* rp = (wave == 1 ? p.delta : p.lse) + sb + (int64_t)ns * kRT;
  // 2 N + 1 copies per wave and step, always: past the first rows' step that one again,
  // into a stage nobody reads, so that every wait is a constant
  auto issue = [&](int stage) {
    const uint32_t st = lds0 + (uint32_t)(stage * 2 * kTile + wave * N * 1024);
    const uint32_t rv = rowv0 + (uint32_t)((stage * 4 + wave) * kRT * 4);
    if (even && ns < n_steps - 1 && ns >= mixed) {
#pragma unroll
      for (int x = 0; x < N; ++x) {
        a_dma16_s(qp, qo[x], st + x * 1024);
        a_dma16_s(dp_, od[x], st + kTile + x * 1024);
      }
      a_dma4_s(rp, (uint32_t)lane * 4, rv);
    } else {
#pragma unroll
      for (int x = 0; x < N; ++x) {
        const int row = (wave * N + x) * RPI + lane / CH, y = ng + row, yt = y * p.g_mul >> 16;
        const int64_t t = min(nt + yt, tb - 1), g = y - yt * p.G;
        const int col = ((lane % CH) ^ a_swz<D>(row)) << 3;
        a_dma16(qb + t * p.q_st + g * p.q_sh + col, st + x * 1024);
        a_dma16(db + t * p.do_st + g * p.do_sh + col, st + kTile + x * 1024);
      }
      const void* src = rp + (ns == n_steps - 1 ? min(lane, back) : lane);
      if (wave == 2 && ns < mixed) src = starts + min(nt + ((ng + lane) * p.g_mul >> 16), tb - 1);
      a_dma4(src, rv);
    }
    if (ns > 0) {
      --ns;
      nt -= adv_t;
      ng -= adv_g;
      if (ng < 0) ng += p.G, --nt;
      qp -= adv_t * p.q_st;
      dp_ -= adv_t * p.do_st;
      rp -= kRT;
    }
  };
  if (n_steps > 0) {
    issue(0);
    issue(1);
    issue(2);
  }

  af3_bf16x8 kf[KS], vf[KS];
  {
    const int64_t jj = kvalid ? j : jl;
    const uint16_t* kr = p.k + b * p.k_sb + hk * p.k_sh + jj * p.k_st;
    const uint16_t* vr = p.v + b * p.v_sb + hk * p.v_sh + jj * p.v_st;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      kf[s] = *(const af3_bf16x8*)(kr + s * 16 + lh * 8);
      vf[s] = *(const af3_bf16x8*)(vr + s * 16 + lh * 8);
    }
    a_landed(kf);
    a_landed(vf);
  }
  const bool jin = kvalid && j >= lo && j < hi;
  const bool wave_in = jw >= lo && jw + 31 < hi && jw + 31 <= jl;
  const bool kept = j < s_last + p.first;  // a first token: its rows end with the sequence
  const Frag<D> fr(lane, lds0 + (uint32_t)(part * 32 * D * 2));
  const uint32_t rv0 = rowv0 + (uint32_t)(part * 128 + lh * 16);

  // The wave's steps [own0, own1), whose rows see some of its keys, and among them
  // [free0, free1), whose rows see all of them.  In rows of the block: those that
  // see key x are (x - off - ta) G up to (x - off - ta + window) G.
  int own0, own1, free0, free1;
  {
    const int64_t k0 = jw - off - ta, k1 = k0 + 31, r0 = part * 32;
    const int64_t nk = max(k0, (int64_t)s_last + p.first - off - ta);  // the first key that a window ends for
    const int64_t e1 = p.window > 0 && nk <= k1 ? min(n_rows, (k1 + p.window) * p.G) : n_rows;
    const int64_t e0 = p.window > 0 && nk <= k1 ? min(n_rows, (nk + p.window) * p.G) : n_rows;
    const bool some_kept = p.first > 0 && s_last + p.first > jw;
    own0 = (int)max((int64_t)0, (k0 * p.G - r0 + 32) >> 6);
    own1 = (int)(((some_kept ? n_rows : e1) - r0 + 63) >> 6);
    free0 = max((int)max((int64_t)0, (k1 * p.G - r0 + 63) >> 6), mixed);
    free1 = wave_in ? (int)((e0 - r0 + 32) >> 6) : 0;
  }
  typedef const __attribute__((address_space(3))) f32x4 lds_f4;
  auto row4 = [&](int stage, int which, int q) {
    return *(lds_f4*)(uintptr_t)(rv0 + (uint32_t)(((stage * 4 + which) * kRT + 8 * q) * 4));
  };

  af3_f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dk[d] = a_zero(), dv[d] = a_zero();

  // scores and dp - delta of the wave's rows of a step, by themselves
  auto scores = [&](auto st, af3_f32x16& s, af3_f32x16& dp) {
    constexpr int stage = st.value;
    constexpr uint32_t qt = stage * 2 * kTile, dt = qt + kTile;
    s = a_zero();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 de = row4(stage, 1, q);
      dp[4 * q] = de.x; dp[4 * q + 1] = de.y; dp[4 * q + 2] = de.z; dp[4 * q + 3] = de.w;
    }
#pragma unroll
    for (int x = 0; x < KS; ++x) s = a_mfma(fr.row8(qt, 0, x), kf[x], s);
#pragma unroll
    for (int x = 0; x < KS; ++x) dp = a_mfma(fr.row8(dt, 0, x), vf[x], dp);
  };
  // a step's probabilities, dz and products, beside the next step's scores
  auto run = [&](int i, auto st, af3_f32x16& s, af3_f32x16& dp, af3_f32x16& s1, af3_f32x16& dp1) {
    constexpr int stage = st.value, nstage = (stage + 1) & 3;
    constexpr uint32_t qt = stage * 2 * kTile, dt = qt + kTile, qn = nstage * 2 * kTile, dn = qn + kTile;
    f32x4 ls[4];
    af3_bf16x8 qr[KS], dr[KS], td[DB], tq[DB], pf, sf;
#pragma unroll
    for (int q = 0; q < 4; ++q) ls[q] = row4(stage, 0, q);
#pragma unroll
    for (int x = 0; x < KS; ++x) qr[x] = fr.row8(qn, 0, x);
    if (i < free0 || i >= free1) {
      const int64_t row = (int64_t)i * kRT + part * 32 + 4 * lh;  // register r: row + 8 (r / 4) + r % 4
      const int64_t d = j - off - ta;
      const int rlo = jin ? a_clamp64(d * p.G - row) : kRT;
      const int rw = p.window > 0 ? a_clamp64((d + p.window) * p.G - row) : kRT;
      const int rhi = min(kept || i < mixed ? kRT : rw, a_clamp64(n_rows - row));
      if (i < free0 || !wave_in) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool on = 8 * (r / 4) + r % 4 >= rlo;
          s[r] = on ? s[r] : -INFINITY;
          dp[r] = on ? dp[r] : 0.f;
        }
      }
      if (i >= free1) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool on = 8 * (r / 4) + r % 4 < rhi;
          s[r] = on ? s[r] : -INFINITY;
          dp[r] = on ? dp[r] : 0.f;
        }
      }
      if (i < mixed) {  // each row's own sequence
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 s4 = row4(stage, 2, q);
          const float sv[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int st = __float_as_int(sv[y]);
            const bool on = j >= st && (8 * q + y < rw || j < st + p.first);
            s[4 * q + y] = on ? s[4 * q + y] : -INFINITY;
            dp[4 * q + y] = on ? dp[4 * q + y] : 0.f;
          }
        }
      }
    }
    s1 = a_zero();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < 2 * KS; ++x) {
      if (x < KS)
        s1 = a_mfma(qr[x], kf[x], s1);
      else
        dp1 = a_mfma(dr[x - KS], vf[x - KS], dp1);
      if (x < KS) dr[x] = fr.row8(dn, 0, x);
      if (x == 0) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 de = row4(nstage, 1, q);
          dp1[4 * q] = de.x; dp1[4 * q + 1] = de.y; dp1[4 * q + 2] = de.z; dp1[4 * q + 3] = de.w;
        }
      }
      if (x == KS / 2) {
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          td[d] = fr.tr8(dt, 0, d);
          tq[d] = fr.tr8(qt, 0, d);
        }
      }
      if (x == KS) {
        pf = a_pack8(s, 0);
        sf = a_pack8(dp, 0);
      }
      if (x >= KS) {  // the first half's products, one after each of the next step's
        const int y = x - KS, d = y / 2;
        if (y & 1)
          dk[d] = a_mfma(tq[d], sf, dk[d]);
        else
          dv[d] = a_mfma(td[d], pf, dv[d]);
      }
#pragma unroll
      for (int r = x * EPS; r < (x + 1) * EPS; ++r) {
        const f32x4 l4 = ls[r / 4];
        const float lv = r % 4 == 0 ? l4.x : r % 4 == 1 ? l4.y : r % 4 == 2 ? l4.z : l4.w;
        s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], p.scale2, -lv));
        dp[r] *= s[r];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      td[d] = fr.tr8(dt, 16, d);
      tq[d] = fr.tr8(qt, 16, d);
    }
    pf = a_pack8(s, 1);
    sf = a_pack8(dp, 1);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      dv[d] = a_mfma(td[d], pf, dv[d]);
      dk[d] = a_mfma(tq[d], sf, dk[d]);
    }
  };
  static_assert(N == 2 || N == 4, "wait counts");
  // (2 N + 1 copies a step: the step after next may be under way)
  auto wait_next = [&]() {
    if constexpr (N == 2) A_WAIT_VM(5); else A_WAIT_VM(9);
  };
  af3_f32x16 s0, dp0, s1, dp1;
  if (n_steps > 0) {
    if constexpr (N == 2) A_WAIT_VM(10); else A_WAIT_VM(18);
    A_BARRIER();
    if (n_steps <= own1) scores(Int<0>{}, s0, dp0);
  }
  // one step: (s, dp) hold its scores; (sn, dpn) get the next one's.  (The stage is a
  // constant of each of four turns: its LDS addresses need no arithmetic.)
  auto turn = [&](int i, auto st, af3_f32x16& s, af3_f32x16& dp, af3_f32x16& sn, af3_f32x16& dpn) {
    wait_next();  // the next step's copies
    A_BARRIER();  // and every wave is past the step before this one
    issue((st.value + 3) & 3);
    if (i == mixed - 1) {
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          dk[d][r] = j < s_last ? 0.f : dk[d][r];
          dv[d][r] = j < s_last ? 0.f : dv[d][r];
        }
    }
    if (i >= own0 && i < own1)
      run(i, st, s, dp, sn, dpn);
    else if (i == own1)
      scores(Int<(st.value + 1) & 3>{}, sn, dpn);
  };
  for (int i = n_steps - 1; i >= 0; i -= 4) {
    turn(i, Int<0>{}, s0, dp0, s1, dp1);
    if (i > 0) turn(i - 1, Int<1>{}, s1, dp1, s0, dp0);
    if (i > 1) turn(i - 2, Int<2>{}, s0, dp0, s1, dp1);
    if (i > 2) turn(i - 3, Int<3>{}, s1, dp1, s0, dp0);
  }
  A_WAIT_VM(0);  // the repeated copies
  // waves 2 and 3 hand their sums to waves 0 and 1 through the ring's LDS
  A_BARRIER();
  float* sum = (float*)lds + ((wave & 1) * 64 + lane) * 4;  // four values of a lane, then the next four 2 KB on
  if (part == 1) {
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        *(float4*)(sum + (d * 8 + r / 4) * 512) = float4{dk[d][r], dk[d][r + 1], dk[d][r + 2], dk[d][r + 3]};
        *(float4*)(sum + (d * 8 + 4 + r / 4) * 512) = float4{dv[d][r], dv[d][r + 1], dv[d][r + 2], dv[d][r + 3]};
      }
  }
  A_BARRIER();
  if (part == 1 || !kvalid) return;
  const int64_t o = (((int64_t)b * p.Sk + j) * p.Hkv + hk) * D;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const float4 k4 = *(const float4*)(sum + (d * 8 + r / 4) * 512);
      const float4 v4 = *(const float4*)(sum + (d * 8 + 4 + r / 4) * 512);
      const int64_t c = o + d * 32 + 2 * r + 4 * lh;
      *(u32x2*)(p.dv + c) = u32x2{af3_pack_bf16x2(dv[d][r] + v4.x, dv[d][r + 1] + v4.y),
                                  af3_pack_bf16x2(dv[d][r + 2] + v4.z, dv[d][r + 3] + v4.w)};
      *(u32x2*)(p.dk + c) = u32x2{af3_pack_bf16x2((dk[d][r] + k4.x) * p.scale, (dk[d][r + 1] + k4.y) * p.scale),
                                  af3_pack_bf16x2((dk[d][r + 2] + k4.z) * p.scale, (dk[d][r + 3] + k4.w) * p.scale)};
    }
}

// ---------------------------------------------------------------------------
// where each token's sequence starts: tokens in no sequence get t + 1 (they see
// nothing).  Every value lies in [0, t + 1] whatever the input holds.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void sa_starts_kernel(const int32_t* __restrict__ cu, int n, int T,
                                                        int32_t* __restrict__ starts) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= T) return;
  int a = 0, b = n;  // the last s with cu[s] <= t lies in [a - 1, b)
  while (a < b) {
    const int mid = (a + b) >> 1;
    if (cu[mid] <= t) a = mid + 1; else b = mid;
  }
  starts[t] = a > 0 && t < cu[a] ? max(cu[a - 1], 0) : t + 1;
}

// A sequence starts where a position is not its predecessor's plus one, and at the
// first token of the row's range; tokens outside the range get t + 1, as those in no
// sequence above.  A block takes kPosTokens of a row, 1024 side by side at a time; the
// last start before them it finds by going back over as many tokens at once, to the
// row's first if need be.  Latency-bound: 6.2 us for 8192 tokens, 11 for 128000 of
// eleven sequences, 34 for 128000 of one.  (One block per row with a run of tokens to
// each thread took 11 and 275 us, the latter more than a third of a windowed layer's
// forward; every layer makes its starts, now those of a batch with ids [B, S] too.)
constexpr int kPosTokens = 4096;

__global__ __launch_bounds__(1024) void sa_starts_pos_kernel(const int64_t* __restrict__ pos, int64_t ld, int T,
                                                             int n_chunks, const int32_t* __restrict__ range,
                                                             int32_t* __restrict__ starts) {
  constexpr int N = kPosTokens / 1024;
  __shared__ int sh[16];
  const int row = blockIdx.x / n_chunks, c0 = (blockIdx.x - row * n_chunks) * kPosTokens;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  pos += row * ld;
  starts += (int64_t)row * T;
  int lo = 0, hi = T;
  if (range) {
    lo = min(max(range[2 * row], 0), T);
    hi = min(max(range[2 * row + 1], lo), T);
  }
  auto starts_at = [&](int t) { return t < T && (t == 0 || (uint64_t)pos[t] - (uint64_t)pos[t - 1] != 1); };
  bool on[N];
#pragma unroll
  for (int i = 0; i < N; ++i) on[i] = starts_at(c0 + i * 1024 + (int)threadIdx.x);
  int before = -1;  // the last start before the tokens at hand
  for (int e = c0; e > 0 && before < 0; e -= kPosTokens) {
    int last = -1;
    bool b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = starts_at(e - kPosTokens + i * 1024 + (int)threadIdx.x);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint64_t m = __ballot(b[i]);
      if (m) last = e - kPosTokens + i * 1024 + wave * 64 + 63 - __builtin_clzll(m);
    }
    if (lane == 0) sh[wave] = last;
    __syncthreads();
    for (int w = 0; w < 16; ++w) before = max(before, sh[w]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int t0 = c0 + i * 1024 + wave * 64, t = t0 + lane;
    const uint64_t m = __ballot(on[i]), upto = m & (~0ull >> (63 - lane));
    if (lane == 0) sh[wave] = m ? t0 + 63 - __builtin_clzll(m) : -1;
    __syncthreads();
    int s = before;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) s = max(s, sh[w]);
      before = max(before, sh[w]);
    }
    if (upto) s = t0 + 63 - __builtin_clzll(upto);
    if (t < T) starts[t] = t >= lo && t < hi ? max(s, lo) : t + 1;
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Splits of a row tile's keys over blocks.  One block per (batch row, key/value
// head, row tile) leaves most of the 256 CUs idle when there are few of them.  A
// block whose rows fill one wave at most (a few new tokens) is bound by reading K
// and V.  Where every batch row has all keys, two such blocks per CU read fastest
// (one token over 131072 keys, 8 key/value heads: 512 blocks 43 us, 768 45, 1024
// 46, 2048 47); with ranges of their own the rows end unevenly and smaller pieces
// level them (32 rows of 90 to 4099 keys: 512 blocks 35 us, 1024 29, 2048 26.5).
// Fuller tiles are split only below a block per CU (the join reads their rows too).
int sa_splits(int B, int Hkv, int64_t n_tiles, int64_t rows, int64_t keys, bool ranges) {
  const int64_t blocks = (int64_t)B * Hkv * n_tiles;
  const bool few = rows <= 32;
  const int64_t target = few && ranges ? 2048 : 512;
  if (blocks == 0 || blocks > (few ? target / 2 : 255)) return 1;
  const int64_t most = keys / 256;  // at least four key tiles each
  int64_t n = target / blocks;
  if (n > most) n = most;
  return n < 1 ? 1 : n > kMaxSplit ? kMaxSplit : (int)n;
}

struct SaShape {
  int tok, n_tiles, n_split, window, first;
};

SaShape sa_shape(int B, int Hq, int Hkv, int Sq, int Sk, int window, int first, bool ranges) {
  SaShape s;
  const int G = Hq / Hkv;
  s.window = window >= Sk ? 0 : window;  // it covers every key
  s.first = s.window > 0 ? (first < Sk ? first : Sk) : 0;
  s.tok = kRows / G;
  s.n_tiles = (int)af3_cdiv(Sq, s.tok);
  int64_t keys = s.window > 0 ? (int64_t)s.window + s.tok + s.first : Sk;
  if (keys > Sk) keys = Sk;
  s.n_split = sa_splits(B, Hkv, s.n_tiles, (int64_t)Sq * G, keys, ranges);
  return s;
}

int sa_check(const char* who, int B, int Hq, int Hkv, int Sq, int Sk, int D, int window, int first, float scale,
             const int64_t* strides, int n_strides, const int32_t* starts, int n_starts, const int32_t* kv_range) {
  AF3_REQUIRE(B >= 0 && Sq >= 0 && Sk >= 0 && Sq < kMaxLen && Sk < kMaxLen, "%s: bad batch or length", who);
  AF3_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "%s: %d query heads do not share %d key/value heads", who, Hq, Hkv);
  AF3_REQUIRE(Hq / Hkv <= kRows, "%s: more than %d query heads per key/value head", who, kRows);
  AF3_REQUIRE(D == 64 || D == 128, "%s: head dimension %d is not 64 or 128", who, D);
  AF3_REQUIRE(window >= 0 && first >= 0, "%s: negative window or first", who);
  AF3_REQUIRE(scale > 0.f && scale * kLog2e < INFINITY, "%s: scale must be positive and finite", who);
  AF3_REQUIRE(strides, "%s: null strides", who);
  for (int i = 0; i < n_strides; ++i) {
    AF3_REQUIRE(strides[i] % 8 == 0, "%s: strides must be multiples of 8", who);
    // (a tile's tokens, and a token's heads, are reached by 32-bit offsets from the tile's address)
    AF3_REQUIRE((i % 3 != 2 && i != 1 && i != 10) || (strides[i] >= 0 && strides[i] < kMaxStride),
                "%s: token strides, and head strides of q and dout, must be below %d", who, kMaxStride);
  }
  AF3_REQUIRE(!starts || ((B <= 1 || B == n_starts) && Sq == Sk && !kv_range),
              "%s: packed rows have starts of their own, Sq == Sk and no kv_range", who);
  // (a launch holds less than 2^32 threads; row numbers of dk / dv stay in 32 bits)
  const int64_t tiles = af3_cdiv(Sq, kRows / (Hq / Hkv)), key_blocks = af3_cdiv(Sk, kKeys);
  AF3_REQUIRE((int64_t)B * Hkv * (Sq + Sk + 1) < 0x7fffffffLL &&
                  (int64_t)B * Hkv * (tiles > key_blocks ? tiles : key_blocks) + Hq < (1LL << 24),
              "%s: too many rows", who);
  return 0;
}

SaParams sa_params(const SaShape& s, const uint16_t* q, const uint16_t* k, const uint16_t* v, const int64_t* st,
                   const void* sinks, int sinks_f32, const int32_t* starts, const int32_t* kv_range, int B, int Hq,
                   int Hkv, int Sq, int Sk, float scale) {
  SaParams p = {};
  p.q = q; p.k = k; p.v = v;
  p.q_sb = st[0]; p.q_sh = st[1]; p.q_st = st[2];
  p.k_sb = st[3]; p.k_sh = st[4]; p.k_st = st[5];
  p.v_sb = st[6]; p.v_sh = st[7]; p.v_st = st[8];
  p.sinks = sinks; p.sinks_f32 = sinks_f32;
  p.starts = starts; p.kv_range = kv_range;
  p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv; p.Sq = Sq; p.Sk = Sk;
  p.window = s.window; p.first = s.first; p.tok = s.tok; p.n_tiles = s.n_tiles; p.n_split = 1;
  p.g_mul = (65536 + p.G - 1) / p.G;
  p.scale = scale; p.scale2 = scale * kLog2e;
  return p;
}

size_t sa_up(size_t n) { return (n + 255) / 256 * 256; }

bool sa_al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int af3_seq_starts(const int32_t* cu_seqlens, int n_seqs, int n_tokens, int32_t* starts, void* stream_) {
  AF3_REQUIRE(n_seqs >= 0 && n_tokens >= 0 && n_tokens < kMaxLen, "seq_starts: bad sizes");
  if (n_tokens == 0) return 0;
  AF3_REQUIRE(cu_seqlens && starts, "seq_starts: null pointer");
  hipLaunchKernelGGL(sa_starts_kernel, dim3((n_tokens + 255) / 256), dim3(256), 0, (hipStream_t)stream_, cu_seqlens,
                     n_seqs, n_tokens, starts);
  return af3::check_launch("seq_starts");
}

extern "C" int af3_seq_starts_rows(const int64_t* position_ids, int64_t ld, int n_rows, int n_tokens,
                                   const int32_t* kv_range, int32_t* starts, void* stream_) {
  const int64_t n_chunks = af3_cdiv(n_tokens, kPosTokens);  // (a launch holds less than 2^32 threads)
  AF3_REQUIRE(n_rows >= 0 && n_tokens >= 0 && n_tokens < kMaxLen && n_rows * n_chunks < (1 << 22) &&
                  (ld == 0 || ld >= n_tokens),
              "seq_starts_rows: bad sizes");
  if (n_rows == 0 || n_tokens == 0) return 0;
  AF3_REQUIRE(position_ids && starts, "seq_starts_rows: null pointer");
  hipLaunchKernelGGL(sa_starts_pos_kernel, dim3((unsigned)(n_rows * n_chunks)), dim3(1024), 0, (hipStream_t)stream_,
                     position_ids, ld, n_tokens, (int)n_chunks, kv_range, starts);
  return af3::check_launch("seq_starts_rows");
}

extern "C" int af3_seq_starts_positions(const int64_t* position_ids, int n_tokens, int32_t* starts, void* stream_) {
  AF3_REQUIRE(n_tokens >= 0 && n_tokens < kMaxLen, "seq_starts_positions: bad size");
  return af3_seq_starts_rows(position_ids, n_tokens, 1, n_tokens, nullptr, starts, stream_);
}

extern "C" size_t af3_sink_attention_workspace_bytes(int B, int Hq, int Hkv, int Sq, int Sk, int D, int window,
                                                     int first, int ranges) {
  if (B <= 0 || Hkv <= 0 || Hq < Hkv || Hq / Hkv > kRows || Sq <= 0 || Sk < 0) return 0;
  const SaShape s = sa_shape(B, Hq, Hkv, Sq, Sk, window, first, ranges != 0);
  return s.n_split > 1 ? (size_t)s.n_split * B * Hq * Sq * (D + 2) * 4 : 0;
}

extern "C" int af3_sink_attention_fwd(const uint16_t* q, const uint16_t* k, const uint16_t* v, const int64_t* strides,
                                      const void* sinks, int sinks_f32, const int32_t* cu_seqlens, int n_seqs,
                                      int32_t* starts, const int32_t* kv_range, int B, int Hq, int Hkv, int Sq, int Sk,
                                      int D, int window, int first, float scale, uint16_t* out, float* lse, void* workspace,
                                      size_t ws_bytes, void* stream_) {
  const char* who = "sink_attention_fwd";
  if (int rc = sa_check(who, B, Hq, Hkv, Sq, Sk, D, window, first, scale, strides, 9, starts,
                        cu_seqlens || n_seqs < 1 ? 1 : n_seqs, kv_range))
    return rc;
  if (B == 0 || Sq == 0) return 0;
  AF3_REQUIRE(q && out && (Sk == 0 || (k && v)), "%s: null pointer", who);
  AF3_REQUIRE(sa_al16(q) && sa_al16(k) && sa_al16(v) && sa_al16(out),
              "%s: rows must be 16-byte aligned", who);
  hipStream_t stream = (hipStream_t)stream_;
  AF3_REQUIRE(!cu_seqlens || starts, "%s: cu_seqlens without starts", who);
  if (cu_seqlens)
    if (int rc = af3_seq_starts(cu_seqlens, n_seqs, Sk, starts, stream_)) return rc;
  const SaShape s = sa_shape(B, Hq, Hkv, Sq, Sk, window, first, kv_range != nullptr);
  SaParams p = sa_params(s, q, k, v, strides, sinks, sinks_f32, starts, kv_range, B, Hq, Hkv, Sq, Sk, scale);
  p.out = out;
  p.lse = lse;
  p.n_split = s.n_split;
  const int64_t grid = (int64_t)s.n_tiles * B * Hkv * s.n_split;
  if (s.n_split > 1) {
    AF3_REQUIRE(workspace && sa_al16(workspace) &&
                    ws_bytes >= af3_sink_attention_workspace_bytes(B, Hq, Hkv, Sq, Sk, D, window, first, kv_range != nullptr),
                "%s: workspace too small", who);
    p.part = (float*)workspace;
  }
  if (D == 64)
    hipLaunchKernelGGL(sa_fwd_kernel<64>, dim3((unsigned)grid), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL(sa_fwd_kernel<128>, dim3((unsigned)grid), dim3(256), 0, stream, p);
  if (s.n_split > 1) {
    const unsigned g = (unsigned)((int64_t)B * Hq * Sq);
    if (D == 64)
      hipLaunchKernelGGL(sa_join_kernel<64>, dim3(g), dim3(256), 0, stream, p);
    else
      hipLaunchKernelGGL(sa_join_kernel<128>, dim3(g), dim3(256), 0, stream, p);
  }
  return af3::check_launch(who);
}

extern "C" size_t af3_sink_attention_bwd_workspace_bytes(int B, int Hq, int Hkv, int Sq) {
  if (B <= 0 || Hkv <= 0 || Hq < Hkv || Hq / Hkv > kRows || Sq <= 0) return 0;
  const int64_t n_tiles = af3_cdiv(Sq, kRows / (Hq / Hkv));
  return sa_up((size_t)B * Hq * Sq * 4) + (size_t)n_tiles * B * Hq * 4;
}

extern "C" int af3_sink_attention_bwd(const uint16_t* q, const uint16_t* k, const uint16_t* v, const uint16_t* dout,
                                      const int64_t* strides, const void* sinks, int sinks_f32, const int32_t* starts,
                                      const int32_t* kv_range, int B, int Hq, int Hkv, int Sq, int Sk, int D,
                                      int window, int first, float scale, const uint16_t* out, const float* lse,
                                      uint16_t* dq, uint16_t* dk, uint16_t* dv, void* dsinks, void* workspace,
                                      size_t ws_bytes, void* stream_) {
  const char* who = "sink_attention_bwd";
  if (int rc = sa_check(who, B, Hq, Hkv, Sq, Sk, D, window, first, scale, strides, 12, starts, B, kv_range))
    return rc;
  const bool nq = B > 0 && Sq > 0, nk = B > 0 && Sk > 0;
  AF3_REQUIRE((!nq || (q && dout && out && lse && dq && workspace)) && (!nk || (k && v && dk && dv)) &&
                  (!sinks || dsinks),
              "%s: null pointer", who);
  AF3_REQUIRE(sa_al16(q) && sa_al16(k) && sa_al16(v) && sa_al16(dout) && sa_al16(out) && sa_al16(dq) && sa_al16(dk) &&
                  sa_al16(dv) && sa_al16(workspace),
              "%s: rows must be 16-byte aligned", who);
  AF3_REQUIRE(ws_bytes >= af3_sink_attention_bwd_workspace_bytes(B, Hq, Hkv, Sq), "%s: workspace too small", who);
  hipStream_t stream = (hipStream_t)stream_;
  const SaShape s = sa_shape(B, Hq, Hkv, Sq, Sk, window, first, kv_range != nullptr);
  SaParams p = sa_params(s, q, k, v, strides, sinks, sinks_f32, starts, kv_range, B, Hq, Hkv, Sq, Sk, scale);
  p.dout = dout;
  p.do_sb = strides[9]; p.do_sh = strides[10]; p.do_st = strides[11];
  p.out = (uint16_t*)out;
  p.lse = (float*)lse;
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.delta = (float*)workspace;
  p.dsink_part = (float*)((uint8_t*)workspace + sa_up((size_t)B * Hq * Sq * 4));
  const unsigned gq = (unsigned)((int64_t)s.n_tiles * B * Hkv);
  if (gq) {
    if (D == 64)
      hipLaunchKernelGGL(sa_dq_kernel<64>, dim3(gq), dim3(256), 0, stream, p);
    else
      hipLaunchKernelGGL(sa_dq_kernel<128>, dim3(gq), dim3(256), 0, stream, p);
  }
  // (dk, dv, and the sinks' sums over the tiles: over nothing where there are no query rows)
  p.dsinks = dsinks;
  p.n_key_blocks = nk ? (int)(af3_cdiv(Sk, kKeys) * B * Hkv) : 0;
  const dim3 grid((unsigned)(p.n_key_blocks + (sinks ? Hq : 0))), block(256);
  if (grid.x) {
    if (D == 64)
      hipLaunchKernelGGL(sa_dkv_kernel<64>, grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL(sa_dkv_kernel<128>, grid, block, 0, stream, p);
  }
  return af3::check_launch(who);
}
