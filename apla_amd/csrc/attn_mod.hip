// Attention (head_dim 64) whose scores are modified and masked on the way to the softmax, forward and deterministic backward:
//   s_ij = scale q_i.k_j ;  s = cap tanh(s / cap) ;  s -= slope_h dist(i, j) ;  masked places = -inf ;  o_i = sum_j softmax(s)_ij v_j
// Queries and keys have their own lengths per sequence (packed by offsets, or uniform with used lengths: a cache); several query
// heads may share one key / value head.  Query i of a sequence stands at key position i + (nk - nq).
//
// Everything positional about the mask is ONE number per query row: lim_i = min(nk, causal ? max(i + nk - nq + 1, prefix) : nk), 0
// for rows of no document; key j is visible iff j < lim_i and the two document ids are equal.  So a workgroup visits the key tiles below its
// largest lim; with documents it first lists those of them whose [min, max] of ids meets its rows'.  A wave runs a tile without a mask
// where lim and the ids say that all of it is visible.
//
// The products are those of attention.hip (S^T = K Q^T with the query row on the lane, P^T from the accumulator as the next operand).
// In a masked tile a weight of zero times a non-finite value is zero (poison_bits): what stands in masked places never matters.
// P and dS are rounded to 16 bits as MFMA operands (half a step of values <= 256 resp. of dS, relative; fp16 over many keys: see LIFT); scores, softmax
// statistics, sums and accumulators are fp32.  A row's dS add up to 0, so over few keys their roundings weigh more than the result's own: sequences of up to
// 64 tokens, a single tile, multiply what the rounding left of dS too (in all masked tiles that costs 5 to 13 % of the long cases' backward).
//
// What bounds the tile kernels is the vector unit: a score costs a multiply-add, an exponential, an addition and half a maximum in the forward (the cap
// a further exponential and a reciprocal).  Counters of the forward over 16384 causal rows: vector unit 79 % busy, matrix unit 45 %, no LDS conflicts; capped fp16 forward 84 / 23 %, its dQ 80 / 30 %, dK/dV 61 / 26 %.
#include "attn_tiles.h"
#include "common.h"

namespace {

constexpr float NEG_BIG = -1e30f;       // running maximum before the first visible key: finite, so that masked scores give exp2(-inf) = 0
constexpr float LAZY = 8.f;             // the running maximum follows only when a score exceeds it by 2^8: weights stay <= 256 (times 2^FWD_LIFT)
// fp16: weights of the forward are 2^FWD_LIFT times larger (at most 2^15), so that many small ones next to a large one, of 2^-14 .. 2^-21 of it, are normal numbers
// too: 2^18 keys of weight 2^-20.6 beside one of weight 1 gave an output off by 5 %.  Statistics count in the same unit.
#if defined(APLA_FP16)
constexpr float FWD_LIFT = 7.f;
#else
constexpr float FWD_LIFT = 0.f;
#endif
constexpr int LIST = 256;               // tiles listed per pass (one per thread)

struct ModArgs {
  const bf16 *q, *k, *v;
  long ldq, ldk, ldv;
  bf16* o;
  long ldo;
  float* lse;
  const int32_t *cu_q, *cu_k, *len_k, *prefix, *doc_q, *doc_k;
  const float *slopes, *pos_q, *pos_k;
  int S, Tq, Tk, max_q, max_k, Hq, G, causal;
  float scale, c, k1, kx, A;            // c = scale log2e; cap: 2 scale log2e / cap, scale / cap, cap log2e
  int fine;                             // every tile counts as masked (see cap_fine)
  const int2 *rng_q, *rng_k;            // [S][tiles of 64]: smallest and largest document id
  int nt_q, nt_k, nblk, np;             // tiles per sequence in those; 128-row blocks per sequence; see where()
  const bf16* d_o;
  long lddo;
  bf16 *dq, *dk, *dv;
  long lddq, lddk, lddv;
  float* delta;
  float *part_o, *part_ml;              // few-row kernel: partial sums
  float *part_q, *part_k;               // backward: partial dQ [sq][Tq][Hq * 64]; dK, then dV [sk][Tk][Hkv * 64]
  int sq, sk;                           // workgroups that share a block's tiles
  int nsplit, chunk, nrt;
};

// fp16: P of n keys is about 1 / n, below its normal range (2^-14) from some thousand keys on, where operands would lose bits (errors of 1.4e-3 at 50 000 equal
// weights, 1e-2 at 2^20).  The backward lifts P, and dS with it, by 2^lift through the exponent's subtrahend and takes it out of the stored results: weights down to
// 1 / (4 n) keep the type's precision.  What is then too large for a dS in fp16 shows as a result that is not finite, and the workgroup starts again without.
#if defined(APLA_FP16)
constexpr bool LIFT = true;
#else
constexpr bool LIFT = false;
#endif
constexpr int LIFT_FROM = 4096;         // up to here 1 / (4 n) is a normal number
__device__ __forceinline__ int lift_of(int nk) { return LIFT && nk > LIFT_FROM ? 20 - __builtin_clz((unsigned)nk - 1u) : 0; }     // ceil(log2(nk / 4096))

struct MSeq { long q0, k0; int nq, nk, off, pre; };
// Offsets that do not fit the tensors are cut to them, so no access leaves the tensors whatever the device-side arrays hold.
__device__ __forceinline__ MSeq mseq(const ModArgs& a, int s) {
  MSeq m;
  if (a.cu_q) {
    const int b = min(max(a.cu_q[s], 0), a.Tq), e = min(max(a.cu_q[s + 1], b), a.Tq);
    m.q0 = b; m.nq = min(e - b, a.max_q);
  } else { m.q0 = (long)s * a.max_q; m.nq = a.max_q; }
  if (a.cu_k) {
    const int b = min(max(a.cu_k[s], 0), a.Tk), e = min(max(a.cu_k[s + 1], b), a.Tk);
    m.k0 = b; m.nk = min(e - b, a.max_k);
  } else { m.k0 = (long)s * a.max_k; m.nk = a.max_k; }
  if (a.len_k) m.nk = min(max(a.len_k[s], 0), m.nk);
  m.off = m.nk - m.nq;
  m.pre = a.prefix ? a.prefix[s] : 0;
  return m;
}
__device__ __forceinline__ int row_lim(const ModArgs& a, const MSeq& m, int i) {
  return a.causal ? max(0, min(m.nk, max(i + m.off + 1, m.pre))) : m.nk;
}

__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

// ---- a product with weights that may be zero next to values that may be infinite or NaN
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
#if defined(APLA_FP16)
constexpr unsigned EXP_LO = 0x7c00u, EXP_STEP = 0x04000400u;
#else
constexpr unsigned EXP_LO = 0x7f80u, EXP_STEP = 0x00800080u;
#endif
constexpr unsigned EXP_HI = EXP_LO << 16;
// bits 15 / 31 of the result: an exponent of all ones among the fragment's values (magnitude + one exponent step carries into the sign's place)
__device__ __forceinline__ unsigned nonfinite_bits(const bf16x8& f) {
  const u32x4 w = __builtin_bit_cast(u32x4, f);
  unsigned r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= (w[i] & 0x7fff7fffu) + EXP_STEP;
  return r & 0x80008000u;
}
// ---- fragments by lane constants.  tile_off XORs the 16-byte chunk with bits 1-3 of the row, so next to a first row that is a multiple of 16 every
// fragment's address is that row * 128 plus one constant of the lane, up to an XOR of bits 5 and 6: k-step ks of a row fragment ^ (ks << 5), column
// half dt of a transposed one ^ (dt << 6), its rows + 8 ^ 32 (tiles start at multiples of 128 bytes).  Left to itself hipcc keeps 40 addresses.
struct Frag { unsigned rf, tr; };
__device__ __forceinline__ Frag frag_consts(int lane) {
  const int g = lane >> 4, i = lane & 15, r = 4 * (g >> 1) + (i >> 2), col = 16 * (g & 1) + 4 * (i & 3);
  return {(unsigned)tile_off(lane & 31, lane >> 5), (unsigned)(tile_off(r, col >> 3) + ((col & 4) << 1))};
}
__device__ __forceinline__ unsigned lds_of(const char* p) { return (unsigned)(size_t)(__attribute__((address_space(3))) const char*)p; }
__device__ __forceinline__ bf16x8 row_at(unsigned base, int row, int ks) {      // base = tile + rf
  return *(const __attribute__((address_space(3))) bf16x8*)(size_t)((base ^ (unsigned)(ks << 5)) + row * 128);
}
__device__ __forceinline__ bf16x8 tr_at(unsigned base, int row, int dt) {      // base = tile + tr
  const bf16x4 lo = DS_READ_TR16_B64_H16((__attribute__((address_space(3))) char*)(size_t)((base ^ (unsigned)(dt << 6)) + row * 128));
  const bf16x4 hi = DS_READ_TR16_B64_H16((__attribute__((address_space(3))) char*)(size_t)((base ^ (unsigned)(dt << 6) ^ 32u) + (row + 8) * 128));
  return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// The 32 transposed fragments' product acc[2] += tile^T w: rows rbase .. rbase + 31 of an LDS tile times the weights that the accumulator w holds for them.
struct TrFrags { bf16x8 f[4]; };      // [dt][sk]
__device__ __forceinline__ void tr_load(TrFrags& t, unsigned base, int rbase) {       // base = tile + tr
#pragma unroll
  for (int sk = 0; sk < 2; ++sk)
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) t.f[2 * dt + sk] = tr_at(base, rbase + 16 * sk, dt);
}
__device__ __forceinline__ void tr_product(f32x16 (&acc)[2], const TrFrags& t, const f32x16& w) {
#pragma unroll
  for (int sk = 0; sk < 2; ++sk) {
    const bf16x8 wb = acc_to_operand(w, sk);
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) acc[dt] = MFMA_F32_32x32x16_H16(t.f[2 * dt + sk], wb, acc[dt]);
  }
}

// what is left of w once it is rounded to 16 bits (none of what overflows there)
__device__ __forceinline__ void rounding_rest(f32x16& w) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float hi = (float)(bf16)w[i];
    w[i] = fabsf(hi) < INFINITY ? w[i] - hi : 0.f;
  }
}

// Zero times a non-finite value is zero: where a tile that holds such values meets a mask, the product runs over a copy of the tile with those values
// taken out (clean_tile), and the results that a weight other than zero would lead one to are remembered as bits (poison_bits; bit 16 dt + i
// for accumulator element [dt][i]) and become NaN at the end (apply_poison).
__device__ __forceinline__ bf16x8 finite_part(const bf16x8& f) {
  u32x4 w = __builtin_bit_cast(u32x4, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = ((w[i] & EXP_LO) == EXP_LO ? 0u : w[i] & 0xffffu) | ((w[i] & EXP_HI) == EXP_HI ? 0u : w[i] & 0xffff0000u);
  return __builtin_bit_cast(bf16x8, w);
}
// (nearly no registers, however slow: the path must not set the kernel's register count.)  w: weights of rows rbase .. rbase + 31 of the tile `raw`.
__device__ __forceinline__ unsigned poison_bits(const char* raw, int rbase, const f32x16& w, int lane) {
  unsigned own = 0, m = 0;             // bit i: this lane's weight i is not zero; the other 16 rows' weights are in the other half of the wave
  unsigned one = 1;
  asm volatile("" : "+s"(one));        // (hipcc would keep the sixteen bits in registers over the whole tile loop)
#pragma unroll
  for (int i = 0; i < 16; ++i) own |= w[i] != 0.f ? one << i : 0u;
  const auto sw = __builtin_amdgcn_permlane32_swap(own, own, false, false);
  const unsigned nz[2] = {(unsigned)sw[0], (unsigned)sw[1]};
  const int h = lane >> 5;
#pragma unroll 1
  for (int r = 0; r < 32; ++r) {       // row r = acc_row(i, half)
    const unsigned short x = *(const unsigned short*)(raw + tile_off(rbase + r, lane >> 3) + (lane & 7) * 2);
    const unsigned long long bad = __ballot((x & EXP_LO) == EXP_LO);       // bit d
    if (bad == 0) continue;
    const unsigned lo = ((unsigned)bad >> (4 * h)) & 0x0f0f0f0fu, hi = ((unsigned)(bad >> 32) >> (4 * h)) & 0x0f0f0f0fu;
    const unsigned mine = (lo & 0xf) | (lo >> 4 & 0xf0) | (lo >> 8 & 0xf00) | (lo >> 12 & 0xf000) |
                          ((hi & 0xf) | (hi >> 4 & 0xf0) | (hi >> 8 & 0xf00) | (hi >> 12 & 0xf000)) << 16;
    const unsigned z = (r >> 2) & 1 ? nz[1] : nz[0];
    m |= (z >> ((r & 3) + 4 * (r >> 3))) & 1 ? mine : 0u;
  }
  return m;
}
// a single key has weight 1 and its score no gradient: what dP - delta leaves of it is rounding (infinities and NaN stay NaN)
__device__ __forceinline__ void no_gradient(f32x16 (&acc)[2]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) acc[i >> 4][i & 15] *= 0.f;
}
__device__ __forceinline__ void apply_poison(f32x16 (&acc)[2], unsigned m) {
  if (__ballot(m != 0) == 0) return;
#pragma unroll
  for (int i = 0; i < 32; ++i) acc[i >> 4][i & 15] = (m >> i) & 1 ? __builtin_nanf("") : acc[i >> 4][i & 15];
}

// a condition that is the same for the whole wave, as a scalar: branches on it need no execution mask
__device__ __forceinline__ bool uniform(bool c) { return __builtin_amdgcn_readfirstlane((int)c) != 0; }

// ---- staging (byte offsets within a tile: at most 63 rows of 2^25 bytes, below 2^31): 64 rows x 64 columns by 256 threads (two 16-byte pieces each) through registers; rows past nrows read row nrows - 1
struct Stage { bf16x8 v[2]; };
__device__ __forceinline__ bool stage_odd(const Stage& t) { return __ballot((nonfinite_bits(t.v[0]) | nonfinite_bits(t.v[1])) != 0) != 0; }
// byte offset of a thread's first piece from the tile's first row (its second lies 32 rows further)
__device__ __forceinline__ unsigned stage_off(long ld, int tid) { return (unsigned)((tid >> 3) * (int)ld * 2 + (tid & 7) * 16); }
__device__ __forceinline__ void stage_load(Stage& t, const bf16* base, long ld, unsigned off, int row0, int nrows, int tid) {
  const char* p = (const char*)(base + (long)row0 * ld);
  if (row0 + 64 <= nrows) {       // whole tile: scalar addresses next to the lane's constant
    t.v[0] = *(const bf16x8*)(p + off);
    t.v[1] = *(const bf16x8*)(p + ld * 64 + off);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) t.v[i] = *(const bf16x8*)(p + (long)min((tid >> 3) + 32 * i, nrows - 1 - row0) * ld * 2 + (tid & 7) * 16);
  }
}
__device__ __forceinline__ void stage_store(const Stage& t, char* lds, int tid) {
  const int o = tile_off(tid >> 3, tid & 7);
  *(bf16x8*)(lds + o) = t.v[0];
  *(bf16x8*)(lds + o + 32 * 128) = t.v[1];
}
// The same tile straight into LDS (16 bytes a lane, no registers between): LDS takes a wave's lanes side by side, so the tile's swizzle is in the addresses read.
// Done when the wave's vector loads are (tile_ready).
__device__ __forceinline__ unsigned dma_off(long ld, int tid) { return (unsigned)((tid >> 3) * (int)ld * 2 + (tile_off(tid >> 3, tid & 7) & 127)); }
__device__ __forceinline__ void dma16(unsigned lds, const char* base, unsigned off) {      // (the builtin makes hipcc wait for it before any read of LDS)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0", "memory");
}
__device__ __forceinline__ void dma4(unsigned lds, const void* base, unsigned off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0", "memory");
}
__device__ __forceinline__ void dma_tile(char* tile, const bf16* base, long ld, unsigned off, int row0, int nrows, int tid, int wave) {
  const char* p = (const char*)(base + (long)row0 * ld);
  const unsigned d = lds_of(tile) + wave * 1024;
  if (row0 + 64 <= nrows) {
    dma16(d, p, off);
    dma16(d + 4096, p + ld * 64, off);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) dma16(d + i * 4096, p, (unsigned)min((tid >> 3) + 32 * i, nrows - 1 - row0) * (unsigned)ld * 2 + (tile_off(tid >> 3, tid & 7) & 127));
  }
}
__device__ __forceinline__ void tile_ready() { __builtin_amdgcn_s_waitcnt(0x0f70); __syncthreads(); }      // vmcnt(0)
// non-finite values in an 8 KB LDS tile (every wave looks at all of it)
__device__ __forceinline__ bool tile_odd(const char* tile, int lane) {
  unsigned b = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) b |= nonfinite_bits(*(const bf16x8*)(tile + (i * 64 + lane) * 16));
  return __ballot(b != 0) != 0;
}
// copy of an 8 KB LDS tile without its non-finite values, by the whole workgroup (a barrier before it is used)
__device__ __forceinline__ void clean_tile(const char* raw, char* clean, int tid) {
#pragma unroll
  for (int i = 0; i < 2; ++i) *(bf16x8*)(clean + (tid + i * 256) * 16) = finite_part(*(const bf16x8*)(raw + (tid + i * 256) * 16));
}

// position of a row: its own coordinates, or its place in the sequence (BIAS 1 without positions)
template <int BIAS>
__device__ __forceinline__ void row_pos(float (&p)[2], const float* pos, long row, int place) {
  if constexpr (BIAS == 1) p[0] = pos ? pos[row] : (float)place;
  if constexpr (BIAS == 2) { p[0] = pos[2 * row]; p[1] = pos[2 * row + 1]; }
}
template <int BIAS>
__device__ __forceinline__ float dist(const float (&p)[2], float x, float y) {
  if constexpr (BIAS == 1) return fabsf(x - p[0]);
  const float dx = x - p[0], dy = y - p[1];
  return __builtin_amdgcn_sqrtf(dx * dx + dy * dy);
}

// ------------------------------------------------------------------------------------------------ forward, one 64-key tile
// LDS of a key tile: K, V (8 KB each), positions [2][64], document ids [64]
constexpr int KT_POS = 16384, KT_DOC = KT_POS + 512, KT_BYTES = KT_DOC + 256;

struct RowState { float m, l; };       // m: the maximum that weights refer to, less FWD_LIFT
// log of the sum l of weights that refer to m (log2 units); the lift is taken out before the logarithm, whose rounding would grow with it
__device__ __forceinline__ float log_sum(float m, float l) {
  if constexpr (FWD_LIFT > 0.f) return (m + FWD_LIFT + __builtin_amdgcn_logf(l * (1.f / 128.f))) * LN2;
  return (m + __builtin_amdgcn_logf(l)) * LN2;
}
__device__ __forceinline__ float reference(float mx, float zm) {       // of scores up to mx, zm: their unit in log2 units
  if constexpr (FWD_LIFT > 0.f) return mx - FWD_LIFT / zm;
  return mx;
}
struct RowCtx { int lim, doc; float pos[2], slope; };       // slope in log2 units

// cap tanh(s / cap) in log2 units: A (1 - 2 r), r = 1 / (1 + e^(2 s / cap)).  That is exact to 2^-23 A, which small scores feel relatively; cap_fine
// takes the odd series below |s / cap| = 1/4 (its next term is 2^-27 there).  Masked tiles do so — every key of a short sequence is in one —,
// full tiles hold 64 keys or more of a row, over which the difference averages out, as long as A is small: they do so too with caps above 64 (2^-23 A is
// 1.1e-5 there, and would be 0.15 at a cap of 9e5).
__device__ __forceinline__ float cap_score(float s, const ModArgs& a, float& r, float sub = 0.f) {      // less `sub`
  r = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * a.k1));
  return fmaf(-2.f * a.A, r, a.A - sub);
}
__device__ __forceinline__ float cap_fine(float s, const ModArgs& a, float& r) {
  const float z = cap_score(s, a, r), x = s * a.kx, y = x * x;
  const float series = a.A * x * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
  return y < 0.0625f ? series : z;
}
__device__ __forceinline__ int pick(const int4& v, int e) { return e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w; }
// x[16] of one row and 32 keys, first key jr0, hidden ones replaced: by the row's limit, then by the documents (ids of the 32 at LDS `ids`).  One read at a
// time: this path must not set the kernel's register count.
__device__ __forceinline__ void hide_keys(f32x16& x, float hidden, int lim, int doc, int jr0, const char* ids, int h2, bool docs) {
  const int left = lim - jr0 - 4 * h2;
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = (i & 3) + 8 * (i >> 2) < left ? x[i] : hidden;
  if (docs) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int4 d = *(const int4*)(ids + (8 * g + 4 * h2) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * g + e] = pick(d, e) == doc ? x[4 * g + e] : hidden;
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}
// x and y [16] of one key j and 32 rows (their limits and ids in LDS): hidden ones become 0
__device__ __forceinline__ void hide_rows(f32x16& x, f32x16& y, int j, int doc, const char* lims, const char* ids, int h2, bool docs) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int4 l = *(const int4*)(lims + (8 * g + 4 * h2) * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool vis = j < pick(l, e);
      x[4 * g + e] = vis ? x[4 * g + e] : 0.f;
      y[4 * g + e] = vis ? y[4 * g + e] : 0.f;
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  if (docs) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int4 d = *(const int4*)(ids + (8 * g + 4 * h2) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool vis = pick(d, e) == doc;
        x[4 * g + e] = vis ? x[4 * g + e] : 0.f;
        y[4 * g + e] = vis ? y[4 * g + e] : 0.f;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// Scores s[16] of one row (on the lane) and 32 keys, or of one key and 32 rows, in log2 units; with neither cap nor bias they stay raw
// and the caller multiplies by c.  `side`: LDS address of the positions of the other 32 (x, then y 256 bytes behind), r: cap_score's r of every
// score.  masked (the same for the wave) chooses the finer cap here, and nothing else.
template <bool CAP, int BIAS>
__device__ __forceinline__ void modify(f32x16& s, f32x16& r, const ModArgs& a, const float (&pos)[2], float slope, const char* side, int h2, bool masked) {
  if constexpr (CAP) {
    if (masked) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float t;
        s[i] = cap_fine(s[i], a, t);
        r[i] = t;
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);      // (this path must not set the kernel's register count)
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) { float t; s[i] = cap_score(s[i], a, t); r[i] = t; }
    }
  }
  if constexpr (BIAS > 0) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 px = *(const f32x4*)(side + (8 * g + 4 * h2) * 4);
      f32x4 py;
      if constexpr (BIAS > 1) py = *(const f32x4*)(side + 256 + (8 * g + 4 * h2) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float d = dist<BIAS>(pos, px[e], BIAS > 1 ? py[e] : 0.f);
        const int i = 4 * g + e;
        s[i] = CAP ? fmaf(-slope, d, s[i]) : fmaf(s[i], a.c, -slope * d);
      }
    }
  }
}

// both halves of a wave hold the same rows: their larger value, in both
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}

// One wave's 32 rows against 64 keys in two halves: while the matrix unit multiplies Q with the second half's keys the wave exponentiates the first half,
// and the first half's product with V runs under the second half's exponentials.
// masked: some of the 64 keys are hidden from some of the wave's rows.  odd: V holds non-finite values; `clean` is then its copy without them.
template <bool CAP, int BIAS>
__device__ __forceinline__ void fwd_tile(f32x16 (&acc)[2], RowState& st, unsigned& poison, const bf16x8 (&qf)[4], const ModArgs& a, const RowCtx& r,
                                         const char* tile, const char* clean, int j0, int lane, const Frag& fr, bool masked, bool docs, bool odd) {
  const int h2 = lane >> 5;
  const float zm = (CAP || BIAS) ? 1.f : a.c;
  const unsigned Ks = lds_of(tile) + fr.rf, Vs = (odd ? lds_of(clean) : lds_of(tile) + 8192) + fr.tr;
  f32x16 s[2], unused;
  auto finish = [&](int kt) {       // cap, bias, mask, running maximum
    modify<CAP, BIAS>(s[kt], unused, a, r.pos, r.slope, tile + KT_POS + kt * 128, h2, masked);
    if (masked) hide_keys(s[kt], -INFINITY, r.lim, r.doc, j0 + kt * 32, tile + KT_DOC + kt * 128, h2, docs);
    float mx = s[kt][0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[kt][i]);
    mx = half_max(mx);
    if (__ballot((mx - st.m) * zm > LAZY + FWD_LIFT)) {
      const float m_new = fmaxf(st.m, reference(mx, zm)), alpha = __builtin_amdgcn_exp2f((st.m - m_new) * zm);
      st.m = m_new;
      st.l *= alpha;
#pragma unroll
      for (int i = 0; i < 16; ++i) { acc[0][i] *= alpha; acc[1][i] *= alpha; }
      if (kt == 1) {         // the first half's weights are not in acc yet
#pragma unroll
        for (int i = 0; i < 16; ++i) s[0][i] *= alpha;
      }
    }
  };
  float mc;
  auto weights = [&](int kt, int g) {      // four of the sixteen
#pragma unroll
    for (int i = 4 * g; i < 4 * g + 4; ++i) {
      s[kt][i] = __builtin_amdgcn_exp2f((CAP || BIAS) ? s[kt][i] - mc : fmaf(s[kt][i], zm, -mc));
      st.l += s[kt][i];
    }
  };
  {
    bf16x8 kf[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) kf[ks] = row_at(Ks, 0, ks);
    __builtin_amdgcn_sched_barrier(0);     // the four reads are under way before the first product waits for one
#pragma unroll
    for (int i = 0; i < 16; ++i) s[0][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) s[0] = MFMA_F32_32x32x16_H16(kf[ks], qf[ks], s[0]);
  }
  finish(0);
  mc = st.m * zm;
  {
    bf16x8 kf[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) kf[ks] = row_at(Ks, 32, ks);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[1][i] = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      weights(0, g);
      s[1] = MFMA_F32_32x32x16_H16(kf[g], qf[g], s[1]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  asm volatile("" : "+v"(s[0]));           // (hipcc would move the exponentials behind the branches that follow)
  TrFrags vf;
  tr_load(vf, Vs, 0);
  finish(1);
  if (__builtin_expect(odd, 0)) poison |= poison_bits(tile + 8192, 0, s[0], lane);
  mc = st.m * zm;
  {
    const bf16x8 w0 = acc_to_operand(s[0], 0), w1 = acc_to_operand(s[0], 1);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      acc[g & 1] = MFMA_F32_32x32x16_H16(vf.f[2 * (g & 1) + (g >> 1)], g < 2 ? w0 : w1, acc[g & 1]);
      weights(1, g);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  tr_load(vf, Vs, 32);
  if (__builtin_expect(odd, 0)) poison |= poison_bits(tile + 8192, 32, s[1], lane);
  tr_product(acc, vf, s[1]);
}

// ---- the list of key tiles that rows with (lim_max, documents dmin..dmax) can see, one pass of up to LIST tiles from t0
struct TileRef { int t, lo, hi, whole; };      // whole: all of it is visible to all rows of the workgroup
// n entries in list[]; all threads call it, ends with a barrier.  Tiles w0 .. w1 - 1 lie within the limits of all rows.
__device__ __forceinline__ int build_list(TileRef* list, int* cnt, int t0, int ntiles, int w0, int w1, const int2* rng, int dmin, int dmax, int tid) {
  const int t = t0 + tid;
  bool vis = t < ntiles;
  int2 r = {0, 0};
  if (vis) {
    r = rng[t];
    vis = r.y >= max(dmin, 0) && r.x <= dmax;
  }
  const unsigned long long b = __ballot(vis);
  if ((tid & 63) == 0) cnt[tid >> 6] = __popcll(b);
  __syncthreads();
  int base = 0, n = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) { const int c = cnt[w]; base += w < (tid >> 6) ? c : 0; n += c; }
  if (vis) {
    const int at = base + __popcll(b & ((1ull << (tid & 63)) - 1));
    list[at] = {t, r.x, r.y, t >= w0 && t < w1 && r.x >= 0 && r.x == r.y && dmin == r.x && dmax == r.x};
  }
  __syncthreads();
  return n;
}

// document range and limits (smallest, largest) of the rows a workgroup holds, for its list (LDS exchange of the waves' own)
__device__ __forceinline__ void group_range(int& lo, int& hi, int& lim0, int& lim, int* buf, int wave, int lane) {
  if (lane == 0) { buf[wave] = lo; buf[4 + wave] = hi; buf[8 + wave] = lim; buf[12 + wave] = lim0; }
  __syncthreads();
  lo = __builtin_amdgcn_readfirstlane(min(min(buf[0], buf[1]), min(buf[2], buf[3])));
  hi = __builtin_amdgcn_readfirstlane(max(max(buf[4], buf[5]), max(buf[6], buf[7])));
  lim = __builtin_amdgcn_readfirstlane(max(max(buf[8], buf[9]), max(buf[10], buf[11])));
  lim0 = __builtin_amdgcn_readfirstlane(min(min(buf[12], buf[13]), min(buf[14], buf[15])));
  __syncthreads();
}

// a list entry as scalars
__device__ __forceinline__ TileRef scalar_ref(const TileRef& r) {
  return {__builtin_amdgcn_readfirstlane(r.t), __builtin_amdgcn_readfirstlane(r.lo), __builtin_amdgcn_readfirstlane(r.hi), __builtin_amdgcn_readfirstlane(r.whole)};
}

// any of the four waves' verdicts (dK/dV)
__device__ __forceinline__ bool any_odd(const char* p) {
  const int4 f = *(const int4*)p;
  return __builtin_amdgcn_readfirstlane(f.x | f.y | f.z | f.w) != 0;
}

// per-key side data of a tile: positions and document (threads 0..63)
struct KeySide { float x, y; int d; };
template <int BIAS>
__device__ __forceinline__ void side_load(KeySide& ks, const ModArgs& a, const MSeq& m, int j0, int tid) {
  if (tid < 64) {
    const int j = min(j0 + tid, m.nk - 1);
    float p[2] = {0.f, 0.f};
    row_pos<BIAS>(p, a.pos_k, m.k0 + j, j);
    ks.x = p[0]; ks.y = p[1];
    ks.d = a.doc_k ? a.doc_k[m.k0 + j] : 0;
  }
}
// the same into a tile's LDS, one wave each for x, y and the documents
template <int BIAS, bool DOCS>
__device__ __forceinline__ void dma_side(char* tile, const ModArgs& a, const MSeq& m, int j0, int lane, int wave) {
  const unsigned j = min(j0 + lane, m.nk - 1), d = lds_of(tile) + KT_POS;
  if constexpr (BIAS == 1) {
    if (wave == 0) {
      if (a.pos_k) dma4(d, a.pos_k + m.k0, j * 4);
      else *(float*)(tile + KT_POS + lane * 4) = (float)j;
    }
  }
  if constexpr (BIAS == 2) {
    if (wave < 2) dma4(d + wave * 256, a.pos_k + 2 * m.k0 + wave, j * 8);
  }
  if constexpr (DOCS) {
    if (wave == 2) dma4(d + KT_DOC - KT_POS, a.doc_k + m.k0, j * 4);
  }
}

// Workgroup -> (sequence, head, block of 128 rows).  Blocks go to the 8 XCDs in turn (blockIdx & 7), each with an L2 of its own: the workgroups that read
// the same rows (one key head of one sequence: `per` of them) stay on one XCD, in `np` parts on np of them where the number of such units is
// no multiple of 8, and the units go round the XCDs, so that long and short sequences mix.  j counts the unit's workgroups, long causal blocks first.
struct Where { int unit, j; };
__device__ __forceinline__ Where where(const ModArgs& a, int per) {
  const int xcd = blockIdx.x & 7, idx = blockIdx.x >> 3, each = (per + a.np - 1) / a.np;
  const int u = idx / each * 8 + xcd;      // (unit, part)
  return {u / a.np, idx % each * a.np + u % a.np};
}
// parts per unit, and the grid's size
static inline int unit_parts(long units) { return units % 8 == 0 ? 1 : units % 4 == 0 ? 2 : units % 2 == 0 ? 4 : 8; }
static inline long unit_grid(long units, int np, long per) { return units * np * ((per + np - 1) / np); }

// a transposed accumulator pair (store_acc_T's layout) as fp32 partial sums of one split
template <bool MUL>
__device__ __forceinline__ void store_part(const f32x16 (&acc)[2], float* rowptr, int h, float mul) {
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 v = {acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
      if constexpr (MUL) v *= mul;
      *(f32x4*)(rowptr + 32 * dt + 8 * g + 4 * h) = v;
    }
}
// does any wave of the workgroup hold infinities or NaN?  (all threads call it; buf: 4 ints that nobody else uses meanwhile)
__device__ __forceinline__ bool overflowed(const f32x16 (&a)[2], const f32x16 (&b)[2], int* buf, int wave, int lane) {
  unsigned r = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i)
    r |= (unsigned)!(fabsf(a[i >> 4][i & 15]) < INFINITY) | (unsigned)!(fabsf(b[i >> 4][i & 15]) < INFINITY);
  const bool any = __ballot(r != 0) != 0;
  if (lane == 0) buf[wave] = any;
  __syncthreads();
  const int all = buf[0] | buf[1] | buf[2] | buf[3];
  __syncthreads();
  return uniform(all != 0);
}

// what a lane knows of its query row
template <int BIAS>
__device__ __forceinline__ RowCtx row_ctx(const ModArgs& a, const MSeq& m, int i, int h) {
  RowCtx r;
  r.doc = a.doc_q ? a.doc_q[m.q0 + i] : 0;
  r.lim = r.doc < 0 ? 0 : row_lim(a, m, i);
  r.pos[0] = r.pos[1] = 0.f;
  row_pos<BIAS>(r.pos, a.pos_q, m.q0 + i, i + m.off);
  r.slope = BIAS ? a.slopes[h] * LOG2E : 0.f;
  return r;
}

// ------------------------------------------------------------------------------------------------ forward
// 128 rows of a head per workgroup, 32 per wave; key tiles of 64 (K, V, positions, ids) go straight into one half of LDS while the other is worked on.
// Three workgroups share a CU where 168 registers hold a wave's state, or nearly (the capped forward without a bias keeps 7 registers in scratch, bf16 documents
// with a 2-D bias one); capped scores next to a bias or documents would keep many (8 x 12 heads of 1370 rows with both: 148 us with two, 169
// with three).  Three take 10 % (cap) to 19 % (ragged, 2-D bias) less time than two.  Forward on a warm card: 64 x 12 heads of 257 rows 38 us, 12 heads
// of 16384 causal rows 487 us (847 TFLOP/s of the visible half), 48 ragged sequences with a 2-D bias 125 us, capped 8 x 24 heads of 1370
// rows in fp16 191 us (484 TFLOP/s).
template <bool CAP, int BIAS, bool DOCS>
__global__ __launch_bounds__(256, CAP && (DOCS || BIAS) ? 2 : 3) void attn_mod_fwd_kernel(ModArgs a) {
  __shared__ __attribute__((aligned(128))) char smem[2 * KT_BYTES], clean[8192];
  __shared__ TileRef list[DOCS ? LIST : 1];
  __shared__ int buf[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h2 = lane >> 5;
  const Frag fr = frag_consts(lane);
  const Where w = where(a, a.G * a.nblk);
  if (w.j >= a.G * a.nblk) return;
  const int Hkv = a.Hq / a.G, hk = w.unit % Hkv, h = hk * a.G + w.j % a.G, blk = w.j / a.G;
  const MSeq m = mseq(a, w.unit / Hkv);
  const int q0 = (a.causal ? a.nblk - 1 - blk : blk) * 128;
  if (q0 >= m.nq) return;
  const int qr = q0 + wave * 32 + (lane & 31);
  const bool active = q0 + wave * 32 < m.nq;
  const int qi = min(qr, m.nq - 1);
  bf16x8 qf[4];
  load_row_frags(qf, a.q + (m.q0 + qi) * a.ldq + h * 64, lane);
  const RowCtx r = row_ctx<BIAS>(a, m, qi, h);
  constexpr bool docs = DOCS;
  // limits (smallest, largest) and documents of the wave's and of the workgroup's rows; without documents the limits grow with the row
  int wlo = 0, whi = 0, dlo = 0, dhi = 0, wlim0, wlim1, lim0, lim;
  if constexpr (DOCS) {
    wlo = wave_min_i(r.doc); whi = wave_max_i(r.doc); wlim0 = wave_min_i(r.lim); wlim1 = wave_max_i(r.lim);
    dlo = wlo; dhi = whi; lim0 = wlim0; lim = wlim1;
    group_range(dlo, dhi, lim0, lim, buf, wave, lane);
  } else {
    const int wq = min(q0 + wave * 32, m.nq - 1);
    wlim0 = row_lim(a, m, wq); wlim1 = row_lim(a, m, min(wq + 31, m.nq - 1));
    lim0 = row_lim(a, m, q0); lim = row_lim(a, m, min(q0 + 127, m.nq - 1));
  }
  if (CAP && a.fine) lim0 = wlim0 = 0;

  f32x16 acc[2];
#pragma unroll
  for (int i = 0; i < 16; ++i) { acc[0][i] = 0.f; acc[1][i] = 0.f; }
  RowState st = {NEG_BIG, 0.f};
  unsigned poison = 0;
  const bf16 *kb = a.k + m.k0 * a.ldk + (hk) * 64, *vb = a.v + m.k0 * a.ldv + (hk) * 64;
  const unsigned offk = dma_off(a.ldk, tid), offv = dma_off(a.ldv, tid);
  const int ntiles = (lim + 63) / 64;
  for (int t0 = 0; t0 < ntiles; t0 = DOCS ? t0 + LIST : ntiles) {
    int n = __builtin_amdgcn_readfirstlane(ntiles);
    if constexpr (DOCS) n = build_list(list, buf, t0, ntiles, 0, lim0 / 64, a.rng_k + (long)(w.unit / Hkv) * a.nt_k, dlo, dhi, tid);
    // entry e of the tiles to visit (past the last: the last): from the list, or simply tile e
    auto entry = [&](int e) -> TileRef {
      e = min(e, n - 1);
      if constexpr (DOCS) return list[e];
      else return TileRef{e, 0, 0, e < lim0 / 64};
    };
    auto known = [&](const TileRef& x) -> TileRef { return DOCS ? scalar_ref(x) : x; };
    auto fetch = [&](char* tile, int t) {
      dma_tile(tile, kb, a.ldk, offk, t * 64, m.nk, tid, wave);
      dma_tile(tile + 8192, vb, a.ldv, offv, t * 64, m.nk, tid, wave);
      dma_side<BIAS, DOCS>(tile, a, m, t * 64, lane, wave);
    };
    TileRef cur, next;
    if (n > 0) {
      cur = known(entry(0)); next = known(entry(0 + 1));
      fetch(smem, cur.t);
    }
    tile_ready();
    for (int e = 0; e < n; ++e) {      // tile e is in LDS, e + 1 on its way to the other half
      char *tile = smem + (e & 1) * KT_BYTES, *other = smem + ((e + 1) & 1) * KT_BYTES;
      const TileRef ahead = entry(e + 2);
      if (e + 1 < n) fetch(other, next.t);
      const int j0 = cur.t * 64;
      const bool odd = !cur.whole && tile_odd(tile + 8192, lane);
      if (__builtin_expect(odd, 0)) {
        clean_tile(tile + 8192, clean, tid);
        __syncthreads();
      }
      if (active && j0 < wlim1 && (!docs || (cur.hi >= max(wlo, 0) && cur.lo <= whi))) {
        const bool masked = !cur.whole && !(j0 + 64 <= wlim0 && (!docs || (cur.lo == cur.hi && wlo == cur.lo && whi == cur.lo)));
        fwd_tile<CAP, BIAS>(acc, st, poison, qf, a, r, tile, clean, j0, lane, fr, masked, docs, masked && odd);
      }
      cur = next;
      next = known(ahead);
      tile_ready();
    }
  }
  apply_poison(acc, poison);
  const float l = st.l + __shfl_xor(st.l, 32, 64);
  if (qr < m.nq) {
    store_acc_T(acc, a.o + (m.q0 + qr) * a.ldo + h * 64, h2, l != 0.f ? 1.f / l : 0.f);
    if (h2 == 0)
      a.lse[(long)h * a.Tq + m.q0 + qr] = l != 0.f ? log_sum(st.m * ((CAP || BIAS) ? 1.f : a.c), l) : -INFINITY;
  }
}

// ------------------------------------------------------------------------------------------------ forward, few rows: keys split over waves and workgroups
// The G * nq rows of the query heads that share a key head fill tiles of 16 columns (v_mfma_f32_16x16x32: a single token of 1 .. 16 heads is one
// tile).  Every wave walks its own 64-key tiles (every fourth of the workgroup's chunk) without a barrier: K straight into operand registers, V through the wave's own LDS for the
// transposed read, both a tile ahead.  The four waves' (maximum, sum, output) are joined in LDS, those of several workgroups by
// attn_mod_join_kernel, both in a fixed order.  Bound by the keys' way from memory and by uneven chunks: single tokens of 24 heads on 32 ragged caches of up to 8192
// keys with 8 heads (188 MB) 54 us = 3.5 TB/s (39 us where they lie in the last-level cache), the join 5 us; about 500 workgroups start at
// once on 512 places, and the busiest CU has 1.4 times the mean number of keys.
constexpr int RT_POS = 8192, RT_DOC = RT_POS + 512, RT_BYTES = RT_DOC + 256;      // LDS of a wave: V, positions [2][64], document ids
constexpr int ROWS = 16;

// Scores [4][4] of row (lane & 15) and keys 16 kb + 4 (lane >> 4) + i, as modify() for the wide tiles
template <bool CAP, int BIAS>
__device__ __forceinline__ void modify_few(f32x4 (&s)[4], const ModArgs& a, const RowCtx& r, const char* side, int g, bool masked) {
#pragma unroll
  for (int kb = 0; kb < 4; ++kb) {
    f32x4 px, py;
    if constexpr (BIAS > 0) px = *(const f32x4*)(side + (16 * kb + 4 * g) * 4);
    if constexpr (BIAS > 1) py = *(const f32x4*)(side + 256 + (16 * kb + 4 * g) * 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float z = s[kb][e], rc;
      if constexpr (CAP) z = masked ? cap_fine(z, a, rc) : cap_score(z, a, rc);
      if constexpr (BIAS > 0) {
        const float d = dist<BIAS>(r.pos, px[e], BIAS > 1 ? py[e] : 0.f);
        z = CAP ? z - r.slope * d : fmaf(z, a.c, -r.slope * d);
      }
      s[kb][e] = z;
    }
  }
}
// the four lane groups of a wave hold the same 16 rows: largest value / sum of the four, in all of them
__device__ __forceinline__ float quad_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  return half_max(fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1])));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

template <bool CAP, int BIAS>
__global__ __launch_bounds__(256, 2) void attn_mod_rows_kernel(ModArgs a) {
  __shared__ __attribute__((aligned(128))) char smem[4 * RT_BYTES];
  __shared__ float ml[4][2][ROWS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c16 = lane & 15;
  const int Hkv = a.Hq / a.G;
  // sequences and heads fastest: the XCDs (blockIdx & 7) then share every chunk number, of which the last hold keys in the longest sequences only
  const int pairs = a.S * Hkv, pair = blockIdx.x % pairs, part = blockIdx.x / pairs;
  const int hk = pair % Hkv, s = pair / Hkv, rt = part % a.nrt, sp = part / a.nrt;
  const MSeq m = mseq(a, s);
  const int rows = a.G * m.nq, rr = rt * ROWS + c16;
  if (rt * ROWS >= rows) return;
  const int jb = sp * a.chunk, jw = jb + wave * 64;
  if (sp > 0 && jb >= m.nk) return;      // (the join reads no chunk past the keys)
  const bool docs = a.doc_k != nullptr;
  char* tile = smem + wave * RT_BYTES;
  const bf16 *kb = a.k + m.k0 * a.ldk + hk * 64, *vb = a.v + m.k0 * a.ldv + hk * 64;
  bf16x8 kf[4][2], vs[8];
  KeySide sd;
  auto fetch = [&](int j0) {       // keys past the last read it again
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) kf[b][ks] = *(const bf16x8*)(kb + (long)min(j0 + 16 * b + c16, m.nk - 1) * a.ldk + 32 * ks + 8 * g);
#pragma unroll
    for (int i = 0; i < 8; ++i) vs[i] = *(const bf16x8*)(vb + (long)min(j0 + 8 * i + (lane >> 3), m.nk - 1) * a.ldv + (lane & 7) * 8);
    side_load<BIAS>(sd, a, m, j0, lane);
  };
  if (jw < m.nk) fetch(jw);        // before anything is known of the rows: the first tile's way from memory is half of a short call
  const int rc = min(rr, rows - 1), h = hk * a.G + rc % a.G, qi = rc / a.G;
  bf16x8 qf[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) qf[ks] = *(const bf16x8*)(a.q + (m.q0 + qi) * a.ldq + h * 64 + 32 * ks + 8 * g);
  const RowCtx r = row_ctx<BIAS>(a, m, qi, h);
  const int wlo = wave_min_i(r.doc), whi = wave_max_i(r.doc), wlim0 = CAP && a.fine ? 0 : wave_min_i(r.lim), wlim1 = wave_max_i(r.lim);
  f32x4 acc[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  RowState st = {NEG_BIG, 0.f};
  unsigned poison = 0;             // bit 4 db + i
  const float zm = (CAP || BIAS) ? 1.f : a.c;
  const int je = min(wlim1, jb + a.chunk);
  const int vo = 4 * g + (c16 >> 2), vcol = 4 * (c16 & 3);
  const unsigned tr = lds_of(tile) + (unsigned)(tile_off(vo, vcol >> 3) + ((vcol & 4) << 1));
  for (int j0 = jw; j0 < je; j0 += 256) {
    bool odd = false, any = true, full = j0 + 64 <= wlim0;
    if (docs) {
      const int2 x = a.rng_k[(long)s * a.nt_k + j0 / 64];
      any = uniform(x.y >= max(wlo, 0) && x.x <= whi);
      full = full && uniform(x.x == x.y && wlo == x.x && whi == x.x);
    }
    f32x4 sc[4];
    if (any) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        sc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) sc[b] = MFMA_F32_16x16x32_H16(kf[b][ks], qf[ks], sc[b]);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) *(bf16x8*)(tile + tile_off(8 * i + (lane >> 3), lane & 7)) = vs[i];
    if constexpr (BIAS > 0) *(float*)(tile + RT_POS + lane * 4) = sd.x;
    if constexpr (BIAS > 1) *(float*)(tile + RT_POS + 256 + lane * 4) = sd.y;
    if (docs) *(int*)(tile + RT_DOC + lane * 4) = sd.d;
    if (!full) {
      unsigned bits = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) bits |= nonfinite_bits(vs[i]);
      odd = __ballot(bits != 0) != 0;
    }
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
    if (j0 + 256 < je) fetch(j0 + 256);
    if (any) {
      modify_few<CAP, BIAS>(sc, a, r, tile + RT_POS, g, !full);
      if (!full) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int4 d = docs ? *(const int4*)(tile + RT_DOC + (16 * b + 4 * g) * 4) : int4{0, 0, 0, 0};
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[b][e] = j0 + 16 * b + 4 * g + e < r.lim && (!docs || pick(d, e) == r.doc) ? sc[b][e] : -INFINITY;
        }
      }
      float mx = sc[0][0];
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[b][e]);
      mx = quad_max(mx);
      if (__ballot((mx - st.m) * zm > LAZY + FWD_LIFT)) {
        const float m_new = fmaxf(st.m, reference(mx, zm)), alpha = __builtin_amdgcn_exp2f((st.m - m_new) * zm);
        st.m = m_new;
        st.l *= alpha;
#pragma unroll
        for (int d = 0; d < 4; ++d) acc[d] *= alpha;
      }
      const float mc = st.m * zm;
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[b][e] = __builtin_amdgcn_exp2f((CAP || BIAS) ? sc[b][e] - mc : fmaf(sc[b][e], zm, -mc));
          st.l += sc[b][e];
        }
      if (__builtin_expect(odd, 0)) {      // as poison_bits, then the wave's own tile is cleaned in place
        unsigned own = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) own |= sc[i >> 2][i & 3] != 0.f ? 1u << i : 0u;
#pragma unroll 1
        for (int k = 0; k < 64; ++k) {
          const unsigned short x = *(const unsigned short*)(tile + tile_off(k, lane >> 3) + (lane & 7) * 2);
          const unsigned long long bad = __ballot((x & EXP_LO) == EXP_LO);
          const unsigned nz = (unsigned)__shfl((int)own, c16 + 16 * ((k >> 2) & 3), 64);
          unsigned mine = 0;
#pragma unroll
          for (int d = 0; d < 4; ++d) mine |= ((unsigned)(bad >> (16 * d + 4 * g)) & 0xfu) << (4 * d);
          poison |= (nz >> (4 * (k >> 4) + (k & 3))) & 1 ? mine : 0u;
        }
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
#pragma unroll 1
        for (int i = 0; i < 8; ++i) *(bf16x8*)(tile + (i * 64 + lane) * 16) = finite_part(*(const bf16x8*)(tile + (i * 64 + lane) * 16));
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {        // 32 keys: operand element j is key 32 t + 16 (j >> 2) + 4 g + (j & 3), on both sides
        bf16x8 p;
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = (bf16)sc[2 * t + (j >> 2)][j & 3];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const bf16x4 lo = DS_READ_TR16_B64_H16((__attribute__((address_space(3))) char*)(size_t)((tr ^ (unsigned)(d << 5)) + 32 * t * 128));
          const bf16x4 hi = DS_READ_TR16_B64_H16((__attribute__((address_space(3))) char*)(size_t)((tr ^ (unsigned)(d << 5)) + (32 * t + 16) * 128));
          acc[d] = MFMA_F32_16x16x32_H16((bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}), p, acc[d]);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i >> 2][i & 3] = (poison >> i) & 1 ? __builtin_nanf("") : acc[i >> 2][i & 3];
  // join the four waves: [16 rows][64] fp32 each in 4 KB of its own LDS, 16-byte chunks spread over the banks by their row
  const float l = quad_sum(st.l);
  float* mine = (float*)tile;
#pragma unroll
  for (int d = 0; d < 4; ++d) *(f32x4*)(mine + c16 * 64 + (((4 * d + g) ^ c16) << 2)) = acc[d];
  if (g == 0) { ml[wave][0][c16] = st.m * zm; ml[wave][1][c16] = l; }
  __syncthreads();
  const int row = tid >> 4, ch = tid & 15, ro = rt * ROWS + row;
  const float M = fmaxf(fmaxf(ml[0][0][row], ml[1][0][row]), fmaxf(ml[2][0][row], ml[3][0][row]));
  float L = 0.f;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const float f = ml[u][1][row] != 0.f ? __builtin_amdgcn_exp2f(ml[u][0][row] - M) : 0.f;
    L += f * ml[u][1][row];
    const f32x4 t = *(const f32x4*)((const float*)(smem + u * RT_BYTES) + row * 64 + ((ch ^ row) << 2));
    if (f != 0.f) x += f * t;
  }
  if (ro >= rows) return;
  const int ho = hk * a.G + ro % a.G;
  const long qo = m.q0 + ro / a.G;
  if (a.nsplit == 1) {
    const float inv = L != 0.f ? 1.f / L : 0.f;
    *(bf16x4*)(a.o + qo * a.ldo + ho * 64 + ch * 4) = pack4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    if (ch == 0) a.lse[(long)ho * a.Tq + qo] = L != 0.f ? log_sum(M, L) : -INFINITY;
  } else {
    const long p = ((((long)s * Hkv + hk) * a.nrt + rt) * a.nsplit + sp) * ROWS + row;
    *(f32x4*)(a.part_o + p * 64 + ch * 4) = x;
    if (ch == 0) { a.part_ml[p * 2] = M; a.part_ml[p * 2 + 1] = L; }
  }
}

__global__ __launch_bounds__(256) void attn_mod_join_kernel(ModArgs a) {
  const int tid = threadIdx.x, row = tid >> 4, ch = tid & 15, rt = blockIdx.x, hk = blockIdx.y, s = blockIdx.z;
  const MSeq m = mseq(a, s);
  const int rows = a.G * m.nq, ro = rt * ROWS + row;
  if (ro >= rows) return;
  const long p0 = (((long)s * (a.Hq / a.G) + hk) * a.nrt + rt) * a.nsplit;
  float M = NEG_BIG, L = 0.f;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  const int n = min(a.nsplit, (m.nk + a.chunk - 1) / a.chunk);      // chunks past the sequence's keys hold nothing
  for (int sp = 0; sp < n; ++sp) M = fmaxf(M, a.part_ml[((p0 + sp) * ROWS + row) * 2]);
  for (int sp = 0; sp < n; ++sp) {
    const long p = (p0 + sp) * ROWS + row;
    const float l = a.part_ml[p * 2 + 1], f = l != 0.f ? __builtin_amdgcn_exp2f(a.part_ml[p * 2] - M) : 0.f;
    L += f * l;
    if (f != 0.f) x += f * *(const f32x4*)(a.part_o + p * 64 + ch * 4);
  }
  const int ho = hk * a.G + ro % a.G;
  const long qo = m.q0 + ro / a.G;
  const float inv = L != 0.f ? 1.f / L : 0.f;
  *(bf16x4*)(a.o + qo * a.ldo + ho * 64 + ch * 4) = pack4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
  if (ch == 0) a.lse[(long)ho * a.Tq + qo] = L != 0.f ? log_sum(M, L) : -INFINITY;
}

// ------------------------------------------------------------------------------------------------ backward
// Four scores s[4 g .. 4 g + 3] of a row to weights exp2(z - L2); the rest as modify().  Between matrix instructions: while the unit works on the next
// product the wave works on these.
template <bool CAP, int BIAS>
__device__ __forceinline__ void weigh4(f32x16& s, f32x16& r, int g, float L2, const ModArgs& a, const float (&pos)[2], float slope, const char* side, int h2, bool masked) {
  f32x4 px, py;
  if constexpr (BIAS > 0) px = *(const f32x4*)(side + (8 * g + 4 * h2) * 4);
  if constexpr (BIAS > 1) py = *(const f32x4*)(side + 256 + (8 * g + 4 * h2) * 4);
  float z[4];
  if constexpr (CAP) {
    if (masked) {
#pragma unroll
      for (int e = 0; e < 4; ++e) { float t; z[e] = cap_fine(s[4 * g + e], a, t) - L2; r[4 * g + e] = t; }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) { float t; z[e] = cap_score(s[4 * g + e], a, t, L2); r[4 * g + e] = t; }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float d = 0.f;
    if constexpr (BIAS > 0) d = dist<BIAS>(pos, px[e], BIAS > 1 ? py[e] : 0.f);
    if constexpr (CAP) z[e] = BIAS ? fmaf(-slope, d, z[e]) : z[e];
    else z[e] = fmaf(s[4 * g + e], a.c, BIAS ? fmaf(-slope, d, -L2) : -L2);
    s[4 * g + e] = __builtin_amdgcn_exp2f(z[e]);
  }
}
// P = exp2(z - L2) from the forward's lse, dS = P (dP - delta), with the cap times 1 - tanh^2 = 4 (r - r^2), r = 1 / (1 + e^(2 s / cap)).
// With the cap `delta` is 4 delta, so that the factor 4 costs nothing (dQ of 8 x 24 heads of 1370 capped rows 308 -> 280 us).
// Two kernels, each writing its gradient once: dQ by query rows, dK and dV by keys over the queries of all heads that share them.  The scores are computed
// twice, but nothing is added across workgroups in an order that changes.
template <bool CAP>
__device__ __forceinline__ float dscore(float p, float dp, float delta, float r) {
  if constexpr (CAP) return p * fmaf(4.f, dp, -delta) * fmaf(-r, r, r);
  else return p * (dp - delta);
}
template <bool CAP, int BIAS>
__device__ __forceinline__ void dq_tile(f32x16 (&acc)[2], unsigned& poison, const bf16x8 (&qf)[4], const bf16x8 (&df)[4], float L2, float delta, const ModArgs& a,
                                        const RowCtx& r, const char* tile, const char* clean, int j0, int lane, const Frag& fr, bool masked, bool docs, bool odd, bool few) {
  const int h2 = lane >> 5;
  const unsigned Ks = lds_of(tile), Vs = Ks + 8192, Kt = odd ? lds_of(clean) : Ks;
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) {
    f32x16 s, p, rc;
    bf16x8 kf[4], vf[4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) { kf[ks] = row_at(Ks + fr.rf, kt * 32, ks); vf[ks] = row_at(Vs + fr.rf, kt * 32, ks); }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) { s[i] = 0.f; p[i] = 0.f; }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) s = MFMA_F32_32x32x16_H16(kf[ks], qf[ks], s);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      p = MFMA_F32_32x32x16_H16(vf[g], df[g], p);
      weigh4<CAP, BIAS>(s, rc, g, L2, a, r.pos, r.slope, tile + KT_POS + kt * 128, h2, masked);
      __builtin_amdgcn_sched_barrier(0);
    }
    TrFrags tk;
    tr_load(tk, Kt + fr.tr, kt * 32);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = dscore<CAP>(s[i], p[i], delta, rc[i]);
    if (masked) {
      hide_keys(s, 0.f, r.lim, r.doc, j0 + kt * 32, tile + KT_DOC + kt * 128, h2, docs);
      if (__builtin_expect(odd, 0)) poison |= poison_bits(tile, kt * 32, s, lane);
    }
    tr_product(acc, tk, s);
    if (few) { rounding_rest(s); tr_product(acc, tk, s); }
  }
}

// dQ of 128 rows per workgroup, staged as in the forward; three workgroups per CU where 168 registers hold a wave's state, as there: 15 % less time than two at
// 64 x 12 heads of 257 rows (51 us), 9 % at 8 x 24 capped ones of 1370 (230 us).  (fp16 documents with a 1-D bias keep 4 registers in scratch.)
template <bool CAP, int BIAS, bool DOCS>
__global__ __launch_bounds__(256, CAP && (DOCS || BIAS) ? 2 : 3) void attn_mod_dq_kernel(ModArgs a) {
  __shared__ __attribute__((aligned(128))) char smem[2 * KT_BYTES], clean[8192];
  __shared__ TileRef list[DOCS ? LIST : 1];
  __shared__ int buf[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h2 = lane >> 5;
  const Frag fr = frag_consts(lane);
  const Where w = where(a, a.G * a.nblk * a.sq);
  if (w.j >= a.G * a.nblk * a.sq) return;
  const int Hkv = a.Hq / a.G, hk = w.unit % Hkv, h = hk * a.G + w.j % a.G, sp = w.j / a.G % a.sq, blk = w.j / (a.G * a.sq);
  const MSeq m = mseq(a, w.unit / Hkv);
  const int q0 = (a.causal ? a.nblk - 1 - blk : blk) * 128;
  if (q0 >= m.nq) return;
  const int qr = q0 + wave * 32 + (lane & 31);
  const bool active = q0 + wave * 32 < m.nq;
  const int qi = min(qr, m.nq - 1);
  bf16x8 qf[4], df[4];
  load_row_frags(qf, a.q + (m.q0 + qi) * a.ldq + h * 64, lane);
  load_row_frags(df, a.d_o + (m.q0 + qi) * a.lddo + h * 64, lane);
  const long stat = (long)h * a.Tq + m.q0 + qi;
  float delta = 0.f;      // rowsum(dO o O): this lane's half of the row, then the other half
  {
    bf16x8 of[4];
    load_row_frags(of, a.o + (m.q0 + qi) * a.ldo + h * 64, lane);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf((float)df[ks][e], (float)of[ks][e], delta);
    delta += __shfl_xor(delta, 32, 64);
  }
  const float ls = a.lse[stat];
  float L2 = ls == -INFINITY ? -NEG_BIG : ls * LOG2E;
  if constexpr (CAP) delta *= 4.f;         // (as dscore takes it; the dK/dV kernel reads it so)
  if (sp == 0 && qr < m.nq && h2 == 0) a.delta[stat] = delta;
  const RowCtx r = row_ctx<BIAS>(a, m, qi, h);
  constexpr bool docs = DOCS;
  // limits (smallest, largest) and documents of the wave's and of the workgroup's rows; without documents the limits grow with the row
  int wlo = 0, whi = 0, dlo = 0, dhi = 0, wlim0, wlim1, lim0, lim;
  if constexpr (DOCS) {
    wlo = wave_min_i(r.doc); whi = wave_max_i(r.doc); wlim0 = wave_min_i(r.lim); wlim1 = wave_max_i(r.lim);
    dlo = wlo; dhi = whi; lim0 = wlim0; lim = wlim1;
    group_range(dlo, dhi, lim0, lim, buf, wave, lane);
  } else {
    const int wq = min(q0 + wave * 32, m.nq - 1);
    wlim0 = row_lim(a, m, wq); wlim1 = row_lim(a, m, min(wq + 31, m.nq - 1));
    lim0 = row_lim(a, m, q0); lim = row_lim(a, m, min(q0 + 127, m.nq - 1));
  }
  if (CAP && a.fine) lim0 = wlim0 = 0;
  f32x16 acc[2];
  unsigned poison;
  const bf16 *kb = a.k + m.k0 * a.ldk + (hk) * 64, *vb = a.v + m.k0 * a.ldv + (hk) * 64;
  const unsigned offk = dma_off(a.ldk, tid), offv = dma_off(a.ldv, tid);
  const int ntiles = (lim + 63) / 64;
  int lift = lift_of(m.nk);
  L2 -= lift;
  for (;; L2 += lift, lift = 0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) { acc[0][i] = 0.f; acc[1][i] = 0.f; }
    poison = 0;
    for (int t0 = 0; t0 < ntiles; t0 = DOCS ? t0 + LIST : ntiles) {
      int n = __builtin_amdgcn_readfirstlane(ntiles);
      if constexpr (DOCS) n = build_list(list, buf, t0, ntiles, 0, lim0 / 64, a.rng_k + (long)(w.unit / Hkv) * a.nt_k, dlo, dhi, tid);
      // entry e of the tiles to visit (past the last: the last): from the list, or simply tile e
      auto entry = [&](int e) -> TileRef {
        e = min(e, n - 1);
        if constexpr (DOCS) return list[e];
        else return TileRef{e, 0, 0, e < lim0 / 64};
      };
      auto known = [&](const TileRef& x) -> TileRef { return DOCS ? scalar_ref(x) : x; };
      auto fetch = [&](char* tile, int t) {
        dma_tile(tile, kb, a.ldk, offk, t * 64, m.nk, tid, wave);
        dma_tile(tile + 8192, vb, a.ldv, offv, t * 64, m.nk, tid, wave);
        dma_side<BIAS, DOCS>(tile, a, m, t * 64, lane, wave);
      };
      const int each = (n + a.sq - 1) / a.sq, e0 = min(n, sp * each), e1 = min(n, e0 + each);      // this split's part of the list
      TileRef cur, next;
      if (e0 < e1) {
        cur = known(entry(e0)); next = known(entry(e0 + 1));
        fetch(smem, cur.t);
      }
      tile_ready();
      for (int e = e0; e < e1; ++e) {      // tile e is in LDS, e + 1 on its way to the other half
        char *tile = smem + ((e - e0) & 1) * KT_BYTES, *other = smem + ((e + 1 - e0) & 1) * KT_BYTES;
        const TileRef ahead = entry(e + 2);
        if (e + 1 < e1) fetch(other, next.t);
        const int j0 = cur.t * 64;
        const bool odd = !cur.whole && tile_odd(tile + 0, lane);
        if (__builtin_expect(odd, 0)) {
          clean_tile(tile + 0, clean, tid);
          __syncthreads();
        }
        if (active && j0 < wlim1 && (!docs || (cur.hi >= max(wlo, 0) && cur.lo <= whi))) {
          const bool masked = !cur.whole && !(j0 + 64 <= wlim0 && (!docs || (cur.lo == cur.hi && wlo == cur.lo && whi == cur.lo)));
          dq_tile<CAP, BIAS>(acc, poison, qf, df, L2, delta, a, r, tile, clean, j0, lane, fr, masked, docs, masked && odd, m.nk <= 64);
        }
        cur = next;
        next = known(ahead);
        tile_ready();
      }
    }
    if (!LIFT || lift == 0 || !overflowed(acc, acc, buf, wave, lane)) break;
  }
  const float unlift = LIFT ? __builtin_ldexpf(1.f, -lift) : 1.f;
  apply_poison(acc, poison);
  if (m.nk == 1) no_gradient(acc);
  if (qr < m.nq) {
    if (a.sq == 1) store_acc_T(acc, a.dq + (m.q0 + qr) * a.lddq + h * 64, h2, a.scale * unlift);
    else store_part<LIFT>(acc, a.part_q + (((long)sp * a.Tq + m.q0 + qr) * a.Hq + h) * 64, h2, unlift);
  }
}

// dK, dV of 128 keys: every wave holds 32 keys (the key on the lane) and the workgroup walks the 64-row query tiles of all heads that share them.
// Two workgroups per CU: K, V, dK and dV of a wave's keys take 96 registers, so tiles may come through registers as well (64 x 12 heads of 257 rows 67 us, 8 x 24
// capped ones of 1370 335 us, 12 heads of 8192 rows in documents 91 us).  Caps next to documents keep 1 to 8 registers in scratch, 15 to 20 with LONG.
// LDS of a query tile: Q, dO (8 KB each), then per row: lse (log2 units), delta, position x / y, lim, document, verdicts
constexpr int QT_L = 16384, QT_D = QT_L + 256, QT_X = QT_D + 256, QT_Y = QT_X + 256, QT_LIM = QT_Y + 256, QT_DOC = QT_LIM + 256, QT_ODD = QT_DOC + 256, QT_BYTES = QT_ODD + 128;
struct QuerySide { float L2, delta, x, y; int lim, doc; };

template <bool CAP, int BIAS>
__device__ __forceinline__ void dkdv_tile(f32x16 (&dk)[2], f32x16 (&dv)[2], unsigned& pk, unsigned& pv, const bf16x8 (&kf)[4], const bf16x8 (&vf)[4], const ModArgs& a, int j, int docj,
                                          const float (&pj)[2], float slope, const char* tile, const char* clean, int lane, const Frag& fr, bool masked, bool docs, bool odd, bool few) {
  const int h2 = lane >> 5;
  const unsigned Qs = lds_of(tile), Ds = Qs + 8192, Qt = odd ? lds_of(clean) : Qs;
#pragma unroll
  for (int qt = 0; qt < 2; ++qt) {
    f32x16 s, p, rc;
    {
      bf16x8 qf[4], df[4];
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) { qf[ks] = row_at(Qs + fr.rf, qt * 32, ks); df[ks] = row_at(Ds + fr.rf, qt * 32, ks); }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 16; ++i) { s[i] = 0.f; p[i] = 0.f; }
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) { s = MFMA_F32_32x32x16_H16(qf[ks], kf[ks], s); p = MFMA_F32_32x32x16_H16(df[ks], vf[ks], p); }
    }
    TrFrags td;
    tr_load(td, Qt + 8192 + fr.tr, qt * 32);
    __builtin_amdgcn_sched_barrier(0);
    modify<CAP, BIAS>(s, rc, a, pj, slope, tile + QT_X + qt * 128, h2, masked);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int ir = qt * 32 + 8 * g + 4 * h2;
      const f32x4 L2 = *(const f32x4*)(tile + QT_L + ir * 4), dl = *(const f32x4*)(tile + QT_D + ir * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * g + e;
        const float pr = __builtin_amdgcn_exp2f((CAP || BIAS) ? s[i] - L2[e] : fmaf(s[i], a.c, -L2[e]));
        s[i] = dscore<CAP>(pr, p[i], dl[e], rc[i]);
        p[i] = pr;
      }
    }
    if (masked) {
      hide_rows(p, s, j, docj, tile + QT_LIM + qt * 128, tile + QT_DOC + qt * 128, h2, docs);
      if (__builtin_expect(odd, 0)) {
        pv |= poison_bits(tile + 8192, qt * 32, p, lane);
        pk |= poison_bits(tile, qt * 32, s, lane);
      }
    }
    TrFrags tq;
    tr_load(tq, Qt + fr.tr, qt * 32);
    tr_product(dv, td, p);
    tr_product(dk, tq, s);
    if (few) { rounding_rest(s); tr_product(dk, tq, s); }
  }
}

// LONG (fp16 only): sequences whose weights are lifted.  Its second pass costs registers and the order of the products: 12 heads of 8192 causal rows 304 us against 290
// without, so shorter sequences run without it.
template <bool CAP, int BIAS, bool DOCS, bool LONG = false>
__global__ __launch_bounds__(256, 2) void attn_mod_dkdv_kernel(ModArgs a) {
  __shared__ __attribute__((aligned(128))) char smem[2 * QT_BYTES], clean[16384];
  __shared__ TileRef list[DOCS ? LIST : 1];
  __shared__ int buf[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h2 = lane >> 5;
  const Where w = where(a, a.nblk * a.sk);
  if (w.j >= a.nblk * a.sk) return;
  const int Hkv = a.Hq / a.G, hk = w.unit % Hkv, sp = w.j % a.sk;
  const MSeq m = mseq(a, w.unit / Hkv);
  const int jb = w.j / a.sk * 128;
  if (jb >= m.nk) return;
  const int jr = jb + wave * 32 + (lane & 31), j = min(jr, m.nk - 1);
  const bool active = jb + wave * 32 < m.nk;
  bf16x8 kf[4], vf[4];
  load_row_frags(kf, a.k + (m.k0 + j) * a.ldk + hk * 64, lane);
  load_row_frags(vf, a.v + (m.k0 + j) * a.ldv + hk * 64, lane);
  constexpr bool docs = DOCS;
  const int docj = docs ? a.doc_k[m.k0 + j] : 0;
  float pj[2] = {0.f, 0.f};
  row_pos<BIAS>(pj, a.pos_k, m.k0 + j, j);
  int wlo = 0, whi = 0, dlo = 0, dhi = 0;
  if constexpr (DOCS) {
    int none0 = 0, none1 = 0;
    wlo = wave_min_i(docj); whi = wave_max_i(docj);
    dlo = wlo; dhi = whi;
    group_range(dlo, dhi, none0, none1, buf, wave, lane);
  }
  unsigned pk, pv;
  f32x16 dk[2], dv[2];
  // query tiles that can see key jb: rows i with lim_i > jb, a suffix of the rows (all of them if the prefix reaches jb)
  const int first = m.nq == 0 ? 0 : (!a.causal || m.pre > jb) ? 0 : max(0, jb - m.off) / 64;
  const int ntiles = (m.nq + 63) / 64;
  // whole tiles: every row of theirs sees all 128 keys, all of them rows and keys of the sequence
  const int jlast = jb + 127;
  const int w0 = jlast >= m.nk ? ntiles : (!a.causal || m.pre > jlast) ? 0 : (max(0, jlast - m.off) + 63) / 64, w1 = CAP && a.fine ? 0 : m.nq / 64;
  int lift = LONG ? lift_of(m.nk) : 0;
  int tid_ = tid;
  for (;; lift = 0) {
    if constexpr (LONG) asm volatile("" : "+v"(tid_));       // (what follows from the lane is formed again: hipcc would keep it in registers over both passes)
    const int tid = tid_, lane = tid & 63;
    const Frag fr = frag_consts(lane);
    const unsigned offq = stage_off(a.ldq, tid), offd = stage_off(a.lddo, tid);
#pragma unroll
    for (int i = 0; i < 16; ++i) { dk[0][i] = dk[1][i] = 0.f; dv[0][i] = dv[1][i] = 0.f; }
    pk = pv = 0;
    for (int t0 = first; t0 < ntiles; t0 = DOCS ? t0 + LIST : ntiles) {
      int n = ntiles - first;
      if constexpr (DOCS) n = build_list(list, buf, t0, ntiles, w0, w1, a.rng_q + (long)(w.unit / Hkv) * a.nt_q, dlo, dhi, tid);
      auto entry = [&](int e) -> TileRef {       // e < n
        if constexpr (DOCS) return list[e];
        else return TileRef{first + e, 0, 0, first + e >= w0 && first + e < w1};
      };
      auto known = [&](const TileRef& x) -> TileRef { return DOCS ? scalar_ref(x) : x; };
      const int each = (n * a.G + a.sk - 1) / a.sk, x0 = min(n * a.G, sp * each), total = min(n * a.G, x0 + each) - x0;      // this split's part
      Stage qs, os;
      QuerySide sd;
      auto fetch = [&](int t, int g) {      // a query tile of head g of the group
        const int h = hk * a.G + g, i0 = t * 64;
        stage_load(qs, a.q + m.q0 * a.ldq + h * 64, a.ldq, offq, i0, m.nq, tid);
        stage_load(os, a.d_o + m.q0 * a.lddo + h * 64, a.lddo, offd, i0, m.nq, tid);
        if (tid < 64) {
          const int i = min(i0 + tid, m.nq - 1);
          const long stat = (long)h * a.Tq + m.q0 + i;
          const float ls = a.lse[stat];
          sd.L2 = ls == -INFINITY ? -NEG_BIG : LONG ? ls * LOG2E - lift : ls * LOG2E;
          sd.delta = a.delta[stat];
          float p[2] = {0.f, 0.f};
          row_pos<BIAS>(p, a.pos_q, m.q0 + i, i + m.off);
          sd.x = p[0]; sd.y = p[1];
          sd.doc = a.doc_q ? a.doc_q[m.q0 + i] : 0;
          sd.lim = i0 + tid < m.nq && sd.doc >= 0 ? row_lim(a, m, i) : 0;
        }
      };
      auto put = [&](char* tile, bool whole) {
        stage_store(qs, tile, tid);
        stage_store(os, tile + 8192, tid);
        if (tid < 64) {
          *(float*)(tile + QT_L + tid * 4) = sd.L2;
          *(float*)(tile + QT_D + tid * 4) = sd.delta;
          if constexpr (BIAS > 0) *(float*)(tile + QT_X + tid * 4) = sd.x;
          if constexpr (BIAS > 1) *(float*)(tile + QT_Y + tid * 4) = sd.y;
          *(int*)(tile + QT_LIM + tid * 4) = sd.lim;
          *(int*)(tile + QT_DOC + tid * 4) = sd.doc;
        }
        if (!whole) {
          const bool odd = stage_odd(qs) || stage_odd(os);
          if (lane == 0) *(int*)(tile + QT_ODD + wave * 4) = odd;
        }
      };
      // entry e of head g is in LDS, the next in registers; the one behind that, e2 of head g2, is requested when those are free
      TileRef cur, next;
      int e = n ? x0 % n : 0, g = n ? x0 / n : 0, e2 = e, g2 = g, t2 = 0;
      auto step = [&](int& e_, int& g_) { if (++e_ == n) { e_ = 0; ++g_; } };
      if (total > 0) {
        cur = known(entry(e2));
        step(e2, g2);
        next = known(entry(e2));
        fetch(cur.t, g);
        put(smem, cur.whole);
        if (total > 1) fetch(next.t, g2);
        step(e2, g2);
        t2 = known(entry(e2)).t;
      }
      __syncthreads();
      for (int x = 0; x < total; ++x) {
        char* tile = smem + (x & 1) * QT_BYTES;
        const TileRef ahead = entry(e2);
        const int gn = g2;
        step(e2, g2);
        const int t3 = entry(e2).t;
        const int i0 = cur.t * 64, jw = jb + wave * 32, last = min(i0 + 63, m.nq - 1);
        const bool odd = !cur.whole && any_odd(tile + QT_ODD);
        if (__builtin_expect(odd, 0)) {
          clean_tile(tile, clean, tid);
          clean_tile(tile + 8192, clean + 8192, tid);
          __syncthreads();
        }
        if (active && row_lim(a, m, last) > jw && (!docs || (cur.hi >= max(wlo, 0) && cur.lo <= whi))) {
          const float slope = BIAS ? a.slopes[hk * a.G + g] * LOG2E : 0.f;
          const bool masked = !cur.whole && !(!(CAP && a.fine) && i0 + 64 <= m.nq && jw + 32 <= m.nk && row_lim(a, m, i0) >= jw + 32 &&
                                                     (!docs || (cur.lo >= 0 && cur.lo == cur.hi && wlo == cur.lo && whi == cur.lo)));
          dkdv_tile<CAP, BIAS>(dk, dv, pk, pv, kf, vf, a, j, docj, pj, slope, tile, clean, lane, fr, masked, docs, masked && odd, m.nq <= 64);
        }
        if (x + 1 < total) put(smem + ((x + 1) & 1) * QT_BYTES, next.whole);
        if (x + 2 < total) fetch(t2, gn);
        step(e, g);
        cur = next;
        next = known(ahead);
        t2 = DOCS ? __builtin_amdgcn_readfirstlane(t3) : t3;
        __syncthreads();
      }
    }
    if (!LONG || lift == 0 || !overflowed(dk, dv, buf, wave, lane)) break;
  }
  const float unlift = LONG ? __builtin_ldexpf(1.f, -lift) : 1.f;
  apply_poison(dk, pk);
  if (m.nk == 1) no_gradient(dk);
  apply_poison(dv, pv);
  if (jr < m.nk) {
    if (a.sk == 1) {
      store_acc_T(dk, a.dk + (m.k0 + jr) * a.lddk + hk * 64, h2, a.scale * unlift);
      store_acc_T(dv, a.dv + (m.k0 + jr) * a.lddv + hk * 64, h2, unlift);
    } else {
      float* p = a.part_k + (((long)sp * a.Tk + m.k0 + jr) * Hkv + hk) * 64;
      store_part<LONG>(dk, p, h2, unlift);
      store_part<LONG>(dv, p + (long)a.sk * a.Tk * Hkv * 64, h2, unlift);
    }
  }
}

// Rows = mul * the sum of n fp32 partial sums [n][T][heads * 64], in their order; rows that no sequence holds are left.  One output, or two of them with
// their partial sums one behind the other.  blockIdx: (32-row group of a sequence, output and head, sequence)
struct SumOut { bf16* out; long ld; float mul; };
__global__ __launch_bounds__(256) void attn_mod_sum_kernel(ModArgs a, const float* part, int n, int queries, int heads, SumOut o0, SumOut o1) {
  const int row = blockIdx.x * 32 + (threadIdx.x >> 3), second = blockIdx.y >= heads, h = blockIdx.y - (second ? heads : 0), c = (threadIdx.x & 7) * 8;
  const MSeq m = mseq(a, blockIdx.z);
  if (row >= (queries ? m.nq : m.nk)) return;
  const SumOut o = second ? o1 : o0;
  const long r = (queries ? m.q0 : m.k0) + row, T = queries ? a.Tq : a.Tk;
  f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
  for (int i = second ? n : 0, end = i + n; i < end; ++i) {
    const float* p = part + ((i * T + r) * heads + h) * 64 + c;
    x += *(const f32x4*)p;
    y += *(const f32x4*)(p + 4);
  }
  bf16x8 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) { v[e] = (bf16)(x[e] * o.mul); v[4 + e] = (bf16)(y[e] * o.mul); }
  *(bf16x8*)(o.out + r * o.ld + h * 64 + c) = v;
}

// The rows that no sequence holds (before the first, behind the last, past a sequence's used or cut length) of the outputs named in `fill`: 0, -inf in lse.
// blockIdx.x: the rows behind sequence blockIdx.x - 1 (0: before the first), blockIdx.y: a share of them.
__global__ __launch_bounds__(256) void attn_mod_fill_kernel(ModArgs a, int fill) {
  const int s = (int)blockIdx.x - 1, Hkv = a.Hq / a.G;
  const MSeq m = mseq(a, s < 0 ? 0 : s), n = mseq(a, s + 1 < a.S ? s + 1 : a.S - 1);
  const long q0 = s < 0 ? 0 : m.q0 + m.nq, q1 = s + 1 < a.S ? n.q0 : a.Tq, k0 = s < 0 ? 0 : m.k0 + m.nk, k1 = s + 1 < a.S ? n.k0 : a.Tk;
  const long step = (long)gridDim.y * 32, lane8 = (threadIdx.x & 7) * 8;
  const bf16x8 zero = {};
  for (long r = q0 + blockIdx.y * 32 + (threadIdx.x >> 3); r < q1; r += step)
    for (int h = 0; h < a.Hq; ++h) {
      if (fill & APLA_FILL_O) *(bf16x8*)(a.o + r * a.ldo + h * 64 + lane8) = zero;
      if (fill & APLA_FILL_DQ) *(bf16x8*)(a.dq + r * a.lddq + h * 64 + lane8) = zero;
      if ((fill & APLA_FILL_LSE) && lane8 == 0) a.lse[(long)h * a.Tq + r] = -INFINITY;
    }
  if (fill & (APLA_FILL_DK | APLA_FILL_DV))
    for (long r = k0 + blockIdx.y * 32 + (threadIdx.x >> 3); r < k1; r += step)
      for (int h = 0; h < Hkv; ++h) {
        if (fill & APLA_FILL_DK) *(bf16x8*)(a.dk + r * a.lddk + h * 64 + lane8) = zero;
        if (fill & APLA_FILL_DV) *(bf16x8*)(a.dv + r * a.lddv + h * 64 + lane8) = zero;
      }
}

// smallest and largest document id of every 64-row tile of every sequence: one wave per tile
__global__ __launch_bounds__(256) void attn_mod_ranges_kernel(ModArgs a, int queries, int2* out, int nt) {
  const long id = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int s = (int)(id / nt), t = (int)(id % nt), lane = threadIdx.x & 63;
  if (s >= a.S) return;
  const MSeq m = mseq(a, s);
  const int n = queries ? m.nq : m.nk;
  const int32_t* doc = queries ? a.doc_q + m.q0 : a.doc_k + m.k0;
  if (t * 64 >= n) return;
  const int d = doc[min(t * 64 + lane, n - 1)];
  const int lo = wave_min_i(d), hi = wave_max_i(d);
  if (lane == 0) out[(long)s * nt + t] = {lo, hi};
}

// ------------------------------------------------------------------------------------------------ host side
struct Plan { bool rows; int nsplit, chunk, nrt, sq, sk; long rng_q, rng_k, part, part_q, part_k, bytes; };

// Backward: workgroups that share the tiles of one 128-row block, where the blocks alone would leave the card idle (fewer than 512 of them: two per CU),
// each with at least four 64-row tiles; their fp32 partial sums are added by attn_mod_sum_kernel.
int split_of(long blocks, long tiles) {
  const long want = (768 + blocks - 1) / blocks, most = tiles / 4;
  const long n = blocks >= 512 ? 1 : want < most ? want : most;
  return (int)(n < 1 ? 1 : n > 8 ? 8 : n);
}

// Few rows (attn_mod_rows_kernel): up to two tiles of 16 rows of a head group, or at most 64 blocks of 128 rows in all (a quarter of the CUs; measured with
// 39 blocks of 1654 keys 26 us against 45, 64 of 4096 keys 42 against 75, but 144 of 257 keys 22 against 12).  Keys are split so that about
// 1024 workgroups run, 256 keys at least each (32 ragged caches of up to 8192 keys: 48 us with chunks of 2048, 80 with 4096, 52 with 1024).
Plan plan_of(const apla_attn_mod_t& p, bool backward) {
  Plan pl = {};
  const int G = p.Hq / p.Hkv;
  const long rows = (long)G * p.max_q, wgs = (long)p.S * p.Hq * ((p.max_q + 127) / 128);
  pl.nrt = (int)((rows + ROWS - 1) / ROWS);
  pl.rows = !backward && (rows <= 2 * ROWS || wgs <= 64);
  pl.nsplit = 1;
  pl.chunk = (p.max_k + 255) / 256 * 256;
  if (pl.rows) {
    const long have = (long)p.S * p.Hkv * pl.nrt;
    long want = (1024 + have - 1) / have;
    const long most = (p.max_k + 255) / 256;
    want = want < 1 ? 1 : want > most ? most : want;
    if (want < 1) want = 1;
    pl.chunk = (int)(((p.max_k + want - 1) / want + 255) / 256 * 256);
    if (pl.chunk < 256) pl.chunk = 256;
    pl.nsplit = (p.max_k + pl.chunk - 1) / pl.chunk;
    if (pl.nsplit < 1) pl.nsplit = 1;
  }
  long b = 0;
  if (p.doc_k) {
    pl.rng_k = b; b += ((long)p.S * ((p.max_k + 63) / 64) * 8 + 15) / 16 * 16;
    if (backward) { pl.rng_q = b; b += ((long)p.S * ((p.max_q + 63) / 64) * 8 + 15) / 16 * 16; }
  }
  if (pl.rows && pl.nsplit > 1) { pl.part = b; b += (long)p.S * p.Hkv * pl.nrt * pl.nsplit * ROWS * (64 + 2) * 4; }
  pl.sq = pl.sk = 1;
  if (backward) {
    pl.sq = split_of((long)p.S * p.Hq * ((p.max_q + 127) / 128), (p.max_k + 63) / 64);
    pl.sk = split_of((long)p.S * p.Hkv * ((p.max_k + 127) / 128), (long)G * ((p.max_q + 63) / 64));
    if (pl.sq > 1) { pl.part_q = b; b += (long)pl.sq * p.Tq * p.Hq * 256; }
    if (pl.sk > 1) { pl.part_k = b; b += 2L * pl.sk * p.Tk * p.Hkv * 256; }
  }
  pl.bytes = b;
  return pl;
}

// workgroups of the largest launch of a call
long most_blocks(const apla_attn_mod_t& p, const Plan& pl, bool backward) {
  const long units = (long)p.S * p.Hkv, G = p.Hq / p.Hkv, nq = (p.max_q + 127L) / 128, nk = (p.max_k + 127L) / 128;
  const int np = unit_parts(units);
  long n = (p.S + 1L) * 64;                                                        // fill
  auto also = [&](long m) { n = m > n ? m : n; };
  if (p.doc_k) also((p.S * (((p.max_q > p.max_k ? p.max_q : p.max_k) + 63L) / 64) + 3) / 4);        // ranges
  if (!backward) also(pl.rows ? units * pl.nrt * pl.nsplit : unit_grid(units, np, G * nq));
  else also(unit_grid(units, np, G * nq * pl.sq)), also(unit_grid(units, np, nk * pl.sk));
  return n;
}

int mod_check(const char* who, const apla_attn_mod_t* p, bool backward) {
  APLA_REQUIRE(p, "%s: no arguments", who);
  APLA_REQUIRE(p->S > 0 && p->S <= 65535 && p->Hq > 0 && p->Hq <= 65535 && p->Hkv > 0 && p->Hq % p->Hkv == 0, "%s: need 1..65535 sequences and Hq a multiple of Hkv (S=%d Hq=%d Hkv=%d)", who, p->S, p->Hq, p->Hkv);
  APLA_REQUIRE(p->Tq > 0 && p->Tk > 0 && p->max_q > 0 && p->max_k > 0 && p->max_q <= p->Tq && p->max_k <= p->Tk, "%s: need 0 < max_q <= Tq and 0 < max_k <= Tk (%d/%d, %d/%d)", who, p->max_q, p->Tq, p->max_k, p->Tk);
  APLA_REQUIRE((p->cu_q || (long)p->S * p->max_q == p->Tq) && (p->cu_k || (long)p->S * p->max_k == p->Tk), "%s: without offsets the rows must be S x max", who);
  APLA_REQUIRE(p->max_q <= (1 << 24) && p->max_k <= (1 << 24), "%s: sequences of at most 2^24 tokens", who);
  APLA_REQUIRE(p->scale > 0.f && p->scale < 1e30f && (p->softcap == 0.f || (p->softcap >= 1e-6f && p->softcap < 1e6f)), "%s: need scale > 0 and a softcap of 0 or 1e-6 .. 1e6", who);
  APLA_REQUIRE(p->q && p->k && p->v && p->o && p->lse, "%s: a pointer is missing", who);
  APLA_REQUIRE(apla_aligned16(p->q) && apla_aligned16(p->k) && apla_aligned16(p->v) && apla_aligned16(p->o), "%s: q, k, v, o must be 16-byte aligned", who);
  APLA_REQUIRE(p->ldq >= p->Hq * 64L && p->ldo >= p->Hq * 64L && p->ldk >= p->Hkv * 64L && p->ldv >= p->Hkv * 64L, "%s: a row stride is shorter than its heads", who);
  APLA_REQUIRE(((p->ldq | p->ldk | p->ldv | p->ldo) & 7) == 0 && p->ldq < (1L << 24) && p->ldk < (1L << 24) && p->ldv < (1L << 24), "%s: row strides must be multiples of 8, below 2^24", who);
  APLA_REQUIRE((!p->doc_q) == (!p->doc_k), "%s: document ids are needed for queries and keys", who);
  APLA_REQUIRE(p->pos_dim >= 0 && p->pos_dim <= 2 && (p->pos_dim == 0 ? !p->pos_q && !p->pos_k : p->pos_q && p->pos_k && p->slopes), "%s: positions need slopes, both sides and 1 or 2 coordinates", who);
  APLA_REQUIRE(!p->prefix || p->causal, "%s: a prefix needs the causal mask", who);
  if (backward) {
    APLA_REQUIRE(p->d_o && p->dq && p->dk && p->dv && p->delta, "%s: a pointer is missing", who);
    APLA_REQUIRE(apla_aligned16(p->d_o) && apla_aligned16(p->dq) && apla_aligned16(p->dk) && apla_aligned16(p->dv), "%s: d_o, dq, dk, dv must be 16-byte aligned", who);
    APLA_REQUIRE(p->lddo >= p->Hq * 64L && p->lddq >= p->Hq * 64L && p->lddk >= p->Hkv * 64L && p->lddv >= p->Hkv * 64L && ((p->lddo | p->lddq | p->lddk | p->lddv) & 7) == 0 && p->lddo < (1L << 24),
                 "%s: gradient row strides must cover their heads and be multiples of 8, that of d_o below 2^24", who);
  }
  const Plan pl = plan_of(*p, backward);
  APLA_REQUIRE(pl.bytes == 0 || (p->workspace && apla_aligned16(p->workspace) && p->workspace_bytes >= pl.bytes), "%s: needs %ld bytes of 16-byte aligned workspace (got %ld)", who, pl.bytes, p->workspace_bytes);
  const long blocks = most_blocks(*p, pl, backward);
  APLA_REQUIRE(blocks < (1L << 24), "%s: %ld workgroups in one launch (below 2^24 are possible: 2^32 work items)", who, blocks);
  return APLA_OK;
}

ModArgs mod_args(const apla_attn_mod_t& p, const Plan& pl) {
  ModArgs a = {};
  a.q = (const bf16*)p.q; a.k = (const bf16*)p.k; a.v = (const bf16*)p.v; a.ldq = p.ldq; a.ldk = p.ldk; a.ldv = p.ldv;
  a.o = (bf16*)p.o; a.ldo = p.ldo; a.lse = p.lse;
  a.cu_q = p.cu_q; a.cu_k = p.cu_k; a.len_k = p.len_k; a.prefix = p.prefix; a.doc_q = p.doc_q; a.doc_k = p.doc_k;
  a.slopes = p.slopes; a.pos_q = p.pos_q; a.pos_k = p.pos_k;
  a.S = p.S; a.Tq = p.Tq; a.Tk = p.Tk; a.max_q = p.max_q; a.max_k = p.max_k; a.Hq = p.Hq; a.G = p.Hq / p.Hkv; a.causal = p.causal;
  a.scale = p.scale; a.c = p.scale * LOG2E;
  if (p.softcap > 0.f) { a.k1 = 2.f * p.scale * LOG2E / p.softcap; a.kx = p.scale / p.softcap; a.A = p.softcap * LOG2E; a.fine = p.softcap > 64.f; }
  a.nt_q = (p.max_q + 63) / 64; a.nt_k = (p.max_k + 63) / 64;
  char* ws = (char*)p.workspace;
  if (p.doc_k) { a.rng_k = (const int2*)(ws + pl.rng_k); a.rng_q = (const int2*)(ws + pl.rng_q); }
  a.np = unit_parts((long)p.S * p.Hkv);
  a.nsplit = pl.nsplit; a.chunk = pl.chunk; a.nrt = pl.nrt;
  a.part_o = (float*)(ws + pl.part);
  a.part_ml = a.part_o + (long)p.S * p.Hkv * pl.nrt * pl.nsplit * ROWS * 64;
  a.sq = pl.sq; a.sk = pl.sk; a.part_q = (float*)(ws + pl.part_q); a.part_k = (float*)(ws + pl.part_k);
  a.d_o = (const bf16*)p.d_o; a.lddo = p.lddo; a.dq = (bf16*)p.dq; a.dk = (bf16*)p.dk; a.dv = (bf16*)p.dv;
  a.lddq = p.lddq; a.lddk = p.lddk; a.lddv = p.lddv; a.delta = p.delta;
  return a;
}

void launch_fill(const ModArgs& a, int fill, hipStream_t stream) {
  const long rows = (long)a.Tq + a.Tk, each = rows / (a.S * 256L) + 1;
  hipLaunchKernelGGL(attn_mod_fill_kernel, dim3((unsigned)a.S + 1, (unsigned)(each < 64 ? each : 64)), dim3(256), 0, stream, a, fill);
}

void launch_ranges(const ModArgs& a, bool queries, hipStream_t stream) {
  const int nt = queries ? a.nt_q : a.nt_k;
  hipLaunchKernelGGL(attn_mod_ranges_kernel, dim3((unsigned)(((long)a.S * nt + 3) / 4)), dim3(256), 0, stream, a, queries ? 1 : 0, (int2*)(queries ? a.rng_q : a.rng_k), nt);
}

// KERNEL<cap?, 0 no bias | 1 distance on a line | 2 on a plane, more...>
#define APLA_MOD_LAUNCH(KERNEL, grid, ...)                                                                        \
  do {                                                                                                            \
    const int bias_ = !p->slopes ? 0 : p->pos_dim == 2 ? 2 : 1;                                                   \
    if (p->softcap > 0.f) {                                                                                       \
      if (bias_ == 0) hipLaunchKernelGGL((KERNEL<true, 0 __VA_ARGS__>), grid, dim3(256), 0, stream, a);           \
      else if (bias_ == 1) hipLaunchKernelGGL((KERNEL<true, 1 __VA_ARGS__>), grid, dim3(256), 0, stream, a);      \
      else hipLaunchKernelGGL((KERNEL<true, 2 __VA_ARGS__>), grid, dim3(256), 0, stream, a);                      \
    } else {                                                                                                      \
      if (bias_ == 0) hipLaunchKernelGGL((KERNEL<false, 0 __VA_ARGS__>), grid, dim3(256), 0, stream, a);          \
      else if (bias_ == 1) hipLaunchKernelGGL((KERNEL<false, 1 __VA_ARGS__>), grid, dim3(256), 0, stream, a);     \
      else hipLaunchKernelGGL((KERNEL<false, 2 __VA_ARGS__>), grid, dim3(256), 0, stream, a);                     \
    }                                                                                                             \
  } while (0)
#define APLA_MOD_LAUNCH_DOCS(KERNEL, grid, ...)                                                                   \
  do {                                                                                                            \
    if (a.doc_k) APLA_MOD_LAUNCH(KERNEL, grid, , true __VA_ARGS__);                                               \
    else APLA_MOD_LAUNCH(KERNEL, grid, , false __VA_ARGS__);                                                      \
  } while (0)

}  // namespace

extern "C" long apla_attn_mod_workspace_bytes(const apla_attn_mod_t* p, int backward) {
  if (!p || p->S <= 0 || p->Hq <= 0 || p->Hkv <= 0 || p->Hq % p->Hkv || p->max_q <= 0 || p->max_k <= 0) return -1;
  return plan_of(*p, backward != 0).bytes;
}

extern "C" int apla_attn_mod_few_rows(const apla_attn_mod_t* p) {
  if (apla_attn_mod_workspace_bytes(p, 0) < 0) return -1;
  return plan_of(*p, false).rows ? 1 : 0;
}

extern "C" int apla_attn_mod_fwd(const apla_attn_mod_t* p, hipStream_t stream) {
  const int rc = mod_check("apla_attn_mod_fwd", p, false);
  if (rc != APLA_OK) return rc;
  const Plan pl = plan_of(*p, false);
  ModArgs a = mod_args(*p, pl);
  const long units = (long)p->S * p->Hkv;
  if ((p->fill & (APLA_FILL_O | APLA_FILL_LSE)) && a.cu_q) launch_fill(a, p->fill & (APLA_FILL_O | APLA_FILL_LSE), stream);
  if (a.doc_k) launch_ranges(a, false, stream);
  if (pl.rows) {
    const dim3 grid((unsigned)(units * pl.nrt * pl.nsplit));
    APLA_MOD_LAUNCH(attn_mod_rows_kernel, grid, );
    if (pl.nsplit > 1) hipLaunchKernelGGL(attn_mod_join_kernel, dim3((unsigned)pl.nrt, (unsigned)p->Hkv, (unsigned)p->S), dim3(256), 0, stream, a);
  } else {
    a.nblk = (p->max_q + 127) / 128;
    const dim3 grid((unsigned)unit_grid(units, a.np, (long)a.G * a.nblk));
    APLA_MOD_LAUNCH_DOCS(attn_mod_fwd_kernel, grid, );
  }
  APLA_CHECK_LAUNCH("apla_attn_mod_fwd");
  return APLA_OK;
}

extern "C" int apla_attn_mod_bwd(const apla_attn_mod_t* p, hipStream_t stream) {
  const int rc = mod_check("apla_attn_mod_bwd", p, true);
  if (rc != APLA_OK) return rc;
  const Plan pl = plan_of(*p, true);
  ModArgs a = mod_args(*p, pl);
  const long units = (long)p->S * p->Hkv;
  const int fill = p->fill & ((a.cu_q ? APLA_FILL_DQ : 0) | (a.cu_k || a.len_k ? APLA_FILL_DK | APLA_FILL_DV : 0));
  if (fill) launch_fill(a, fill, stream);
  if (a.doc_k) {
    launch_ranges(a, false, stream);
    if (p->doc_q == p->doc_k && p->cu_q == p->cu_k && p->max_q == p->max_k && !p->len_k) a.rng_q = a.rng_k;      // self-attention: the same tiles
    else launch_ranges(a, true, stream);
  }
  a.nblk = (p->max_q + 127) / 128;
  {
    const dim3 grid((unsigned)unit_grid(units, a.np, (long)a.G * a.nblk * a.sq));
    APLA_MOD_LAUNCH_DOCS(attn_mod_dq_kernel, grid, );
    if (a.sq > 1)
      hipLaunchKernelGGL(attn_mod_sum_kernel, dim3((unsigned)((p->max_q + 31) / 32), (unsigned)p->Hq, (unsigned)p->S), dim3(256), 0, stream, a, (const float*)a.part_q, a.sq, 1, p->Hq,
                         (SumOut{a.dq, a.lddq, a.scale}), (SumOut{}));
  }
  a.nblk = (p->max_k + 127) / 128;
  {
    const dim3 grid((unsigned)unit_grid(units, a.np, (long)a.nblk * a.sk));
#if defined(APLA_FP16)
    if (p->max_k > LIFT_FROM) APLA_MOD_LAUNCH_DOCS(attn_mod_dkdv_kernel, grid, , true);
    else
#endif
      APLA_MOD_LAUNCH_DOCS(attn_mod_dkdv_kernel, grid, );
    if (a.sk > 1)
      hipLaunchKernelGGL(attn_mod_sum_kernel, dim3((unsigned)((p->max_k + 31) / 32), 2u * (unsigned)p->Hkv, (unsigned)p->S), dim3(256), 0, stream, a, (const float*)a.part_k, a.sk, 0, p->Hkv,
                         (SumOut{a.dk, a.lddk, a.scale}), (SumOut{a.dv, a.lddv, 1.f}));
  }
  APLA_CHECK_LAUNCH("apla_attn_mod_bwd");
  return APLA_OK;
}
