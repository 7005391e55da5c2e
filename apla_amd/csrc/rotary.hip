// Rotary positions and the per-head norm of queries and keys (head_dim 64): forward and backward, memory bound.
//
// A head row is 64 x 16 bit = 128 bytes: eight lanes with 16 bytes each, so every load and store instruction of a wave moves eight whole
// lines.  A wave holds either query or key heads (one set of norm parameters, one set of their sums): hb heads of 8 / hb tokens at a
// time (hb the largest of 8, 4, 2, 1 that divides the head count: no lane idles, neighbouring groups are neighbours in memory).  It walks the
// heads of its tokens, so that cosines and sines are loaded once per token and lane and not once per head, DEPTH head blocks requested
// ahead of their use.
//
// Rotation of the pair (a, b) by theta: a' = a cos - b sin, b' = b cos + a sin.  "interleaved": the pair is (2i, 2i+1), both in one
// lane.  "half": (i, i + rot/2), exchanged as fp32 through the wave's own 2 KB of LDS (rot may be any even number: neither a lane nor a
// 16-byte boundary; no barrier, a wave's LDS operations run in order).  The inverse rotation is the same with -sin: the backward pass.
// cos / sin come from a fp32 table built in 64 bits (angles of far positions lose 2^-24 * position in fp32 arithmetic).
//
// Norm backward, g = R^T dy, u = g w, x^ = (x - mean) rstd:  dx = rstd (u - mean(u) - x^ mean(u x^))  (RMS: without mean(u));
// dw = sum g x^, db = sum g over tokens and heads.  The statistics are recomputed from x (it has to be read for x^ anyway).
// A head whose 64 values of dy are all zero gives dx = 0 and adds nothing, whatever x holds and wherever its row stands (rows behind a mask): one look at
// the raw bits and a ballot.
// All arithmetic is fp32; the only rounding is that of the stored result.
//
// Measured (a large copy reaches 4.95 TB/s): rotation forward and backward of 269 MB 56 us, 4.8 TB/s; norm and rotation of 25 216 tokens of 24 heads forward
// (155 MB) 34 us, backward (dy and x read, dx written: 232 MB) 45 us = 5.2 TB/s, the copy's rate, with the vector unit 72 % busy, its sums 5 us;
// few tokens: the launch.
#include "common.h"

namespace {

constexpr int DEPTH = 4;

struct RotArgs {
  const bf16* x; long ldx;       // rotated / normalised rows [T, (heads[0] + heads[1]) * 64]
  const bf16* dy; long lddy;     // backward: incoming gradient of the result
  bf16* y; long ldy;             // result, or dx
  int T, hbl[2], nb[2], splits;  // of queries and keys: log2 of heads per block, blocks; workgroups that share a token's blocks
  const float* table; int P, rot, interleaved, vec;
  const int32_t* pos; int seq_len;
  float sign, eps;
  const float *w[2], *b[2];
  float* partial;                // [2][workgroups][128]: sums for the weight, then the bias
};

__device__ __forceinline__ float group8_sum(float v) {
  v += __shfl_xor(v, 1, 64);
  v += __shfl_xor(v, 2, 64);
  v += __shfl_xor(v, 4, 64);
  return v;
}
__device__ __forceinline__ void unpack8(const bf16x8& r, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (float)r[e];
}

__device__ __forceinline__ bool any_value(const bf16x8& r) {      // other than zero
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 w = __builtin_bit_cast(u32x4, r);
  return ((w[0] | w[1] | w[2] | w[3]) & 0x7fff7fffu) != 0;
}

// v: this lane's 8 elements of a head row (e0 = 8 * lane-in-group); cs / sn: cosine and signed sine of each element (1 / 0 past rot)
__device__ __forceinline__ void rotate8(float (&v)[8], const float (&cs)[8], const float (&sn)[8], int interleaved, int r, int e0, float* xch) {
  float pr[8];
  if (interleaved) {
#pragma unroll
    for (int e = 0; e < 8; ++e) pr[e] = v[e ^ 1];
  } else {
    *(f32x4*)(xch + e0) = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4*)(xch + e0 + 4) = f32x4{v[4], v[5], v[6], v[7]};
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
    if ((r & 3) == 0) {          // four-element groups never straddle a boundary
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = e0 + 4 * h, p = e < r ? e + r : e < 2 * r ? e - r : e;
        const f32x4 t = *(const f32x4*)(xch + p);
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[4 * h + i] = t[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = e0 + i, p = e < r ? e + r : e < 2 * r ? e - r : e;
        pr[i] = xch[p];
      }
    }
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e0 + e < 2 * r ? v[e] * cs[e] + pr[e] * sn[e] : v[e];
}

// NORM: 0 none, 1 LayerNorm, 2 RMS.  blockIdx.y: queries or keys, and which of their blocks.
template <int NORM, bool BWD, bool PAR>
__global__ __launch_bounds__(256) void rotary_kernel(RotArgs a) {
  __shared__ __attribute__((aligned(16))) float xch_all[4][8][68];
  __shared__ float red[PAR ? 4 : 1][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int grp = blockIdx.y / a.splits, sp = blockIdx.y % a.splits;
  const int hbl = a.hbl[grp], nb = a.nb[grp];
  const int g = lane >> 3, e0 = (lane & 7) * 8;
  const int hb = 1 << hbl, sub = g & (hb - 1), tsub = g >> hbl, tpw = 8 >> hbl;
  const int col = (grp ? a.nb[0] << (a.hbl[0] + 6) : 0) + sub * 64 + e0, step = hb * 64;
  float* xch = xch_all[wave][g];
  const int r = a.rot >> 1;
  const int each = (nb + a.splits - 1) / a.splits, b0 = sp * each, b1 = min(nb, b0 + each);
  float w[8], bi[8], aw[8], ab[8];
  if constexpr (NORM != 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = a.w[grp] ? a.w[grp][e0 + e] : 1.f;
      bi[e] = !BWD && a.b[grp] ? a.b[grp][e0 + e] : 0.f;
      aw[e] = ab[e] = 0.f;
    }
  }
  for (long tb = ((long)blockIdx.x * 4 + wave) * tpw; tb < a.T; tb += (long)gridDim.x * 4 * tpw) {
    const bool tv = tb + tsub < a.T;
    const long t = tv ? tb + tsub : a.T - 1;
    float cs[8], sn[8];
    bool outside = false;      // of the wave's tokens any
    if (r > 0) {
      long p = a.pos ? (long)a.pos[t] : a.seq_len ? t % a.seq_len : t;
      const bool pv = p >= 0 && p < a.P;      // a position outside the table gives NaN, not a read outside it
      const float* row = a.table + (pv ? p : 0) * a.rot;
      if (!BWD && NORM == 0) outside = a.sign < 0.f && __ballot(!pv) != 0;
      if (a.vec) {    // the lane's eight angles are four (interleaved) or eight (half) neighbours in the table
        const bool in = e0 < 2 * r;
        const float* c = row + (!in ? 0 : a.interleaved ? e0 >> 1 : e0 < r ? e0 : e0 - r);
        const f32x4 c0 = *(const f32x4*)c, s0 = *(const f32x4*)(c + r);
        if (a.interleaved) {
#pragma unroll
          for (int e = 0; e < 8; ++e) { cs[e] = c0[e >> 1]; sn[e] = (e & 1) ? s0[e >> 1] : -s0[e >> 1]; }
        } else {
          const f32x4 c1 = *(const f32x4*)(c + 4), s1 = *(const f32x4*)(c + r + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) { cs[e] = c0[e]; cs[4 + e] = c1[e]; sn[e] = e0 < r ? -s0[e] : s0[e]; sn[4 + e] = e0 < r ? -s1[e] : s1[e]; }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int el = e0 + e, idx = el >= 2 * r ? 0 : a.interleaved ? el >> 1 : el < r ? el : el - r;
          cs[e] = row[idx];
          sn[e] = (a.interleaved ? !(el & 1) : el < r) ? -row[r + idx] : row[r + idx];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) { cs[e] = pv ? cs[e] : __builtin_nanf(""); sn[e] *= a.sign; }
    }
    const bf16* xr = a.x + t * a.ldx + col;
    const bf16* dr = BWD ? a.dy + t * a.lddy + col : nullptr;
    bf16* yr = a.y + t * a.ldy + col;
    for (int bb = b0; bb < b1; bb += DEPTH) {
      bf16x8 nx[DEPTH], nd[DEPTH];
#pragma unroll
      for (int i = 0; i < DEPTH; ++i)
        if (bb + i < b1) {
          if constexpr (!BWD || NORM != 0) nx[i] = *(const bf16x8*)(xr + (bb + i) * step);
          if constexpr (BWD) nd[i] = *(const bf16x8*)(dr + (bb + i) * step);
        }
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) {
        if (bb + i >= b1) break;
        float v[8], d[8];
        bool none = false;       // no gradient arrives at this head: it passes none on, whatever x holds (masked places may hold infinities and NaN)
        unpack8(nx[i], v);
        if constexpr (BWD) {
          unpack8(nd[i], d);
          const unsigned long long some = __ballot(any_value(nd[i]));
          none = ((some >> (lane & 56)) & 255) == 0;
        }
        float rs = 1.f;
        if constexpr (NORM != 0) {
          if constexpr (NORM == 1) {
            float m = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) m += v[e];
            m = group8_sum(m) * (1.f / 64.f);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] -= m;
          }
          float s = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) s += v[e] * v[e];
          rs = rsqrtf(group8_sum(s) * (1.f / 64.f) + a.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= rs;       // x^
        }
        if constexpr (!BWD) {
          if constexpr (NORM != 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] * w[e] + bi[e];
          }
          if (r > 0) rotate8(v, cs, sn, a.interleaved, r, e0, xch);
          if (NORM == 0 && outside) {      // a gradient turned back at positions outside the table
            const unsigned long long some = __ballot(any_value(nx[i]));
            if (((some >> (lane & 56)) & 255) == 0) {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = 0.f;
            }
          }
        } else {
          if (r > 0) rotate8(d, cs, sn, a.interleaved, r, e0, xch);
          if constexpr (PAR) {
            if (tv && !none) {
#pragma unroll
              for (int e = 0; e < 8; ++e) { aw[e] += d[e] * v[e]; ab[e] += d[e]; }
            }
          }
          float m1 = 0.f, m2 = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            d[e] *= w[e];
            m1 += d[e];
            m2 += d[e] * v[e];
          }
          m1 = NORM == 1 ? group8_sum(m1) * (1.f / 64.f) : 0.f;
          m2 = group8_sum(m2) * (1.f / 64.f);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = none ? 0.f : rs * (d[e] - m1 - v[e] * m2);
        }
        if (tv) {
          bf16x8 out;
#pragma unroll
          for (int e = 0; e < 8; ++e) out[e] = (bf16)v[e];
          *(bf16x8*)(yr + (bb + i) * step) = out;
        }
      }
    }
  }
  if constexpr (PAR) {     // lanes of the same columns (8 groups), then the four waves, in a fixed order
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float u = aw[e], v = ab[e];
#pragma unroll
      for (int o = 8; o < 64; o <<= 1) { u += __shfl_xor(u, o, 64); v += __shfl_xor(v, o, 64); }
      if (g == 0) { red[wave][e0 + e] = u; red[wave][64 + e0 + e] = v; }
    }
    __syncthreads();
    const int i = threadIdx.x;
    if (i < 128) a.partial[((long)blockIdx.y * gridDim.x + blockIdx.x) * 128 + i] = red[0][i] + red[1][i] + red[2][i] + red[3][i];
  }
}

// out [4][64] (query weight, key weight, query bias, key bias) = column sums of partial [2][G][128]: 16 columns per workgroup, 16 row walkers each,
// eight rows requested at a time, summed in a fixed order
__global__ __launch_bounds__(256) void rotary_param_sum_kernel(const float* __restrict__ partial, int G, int groups, float* __restrict__ out) {
  __shared__ float red[16][17];
  const int c = threadIdx.x & 15, w = threadIdx.x >> 4, grp = blockIdx.x >> 3, col = (blockIdx.x & 7) * 16 + c;
  const float* p = partial + (long)grp * G * 128 + col;
  float s = 0.f;
  for (int i = w; grp < groups && i < G; i += 128) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = i + 16 * k < G ? p[(long)(i + 16 * k) * 128] : 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += v[k];
  }
  red[w][c] = s;
  __syncthreads();
  if (w == 0) {
    for (int i = 1; i < 16; ++i) s += red[i][c];
    out[(col >> 6) * 128 + grp * 64 + (col & 63)] = s;
  }
}

// Workgroups of a launch: as many as are resident at once (four per CU, three of the backward with parameter sums, by their registers), each walking
// the tokens; measured at 25 216 tokens of 24 heads, forward: 31 us against 43 with a workgroup per 8 tokens, backward: 46 us against 57 with 1024.
constexpr int ROT_WGS = 1024, PARAM_WGS = 768;

// A wave takes all head blocks of its tokens where that still leaves 4096 waves (16 per CU), else the blocks are spread over blockIdx.y.
dim3 rot_plan(RotArgs& a, int T, int h1, int h2, bool par) {
  const int h[2] = {h1, h2};
  long waves = 0, most = 1;
  for (int g = 0; g < 2; ++g) {
    int hbl = 3;
    while (hbl && (h[g] & ((1 << hbl) - 1))) --hbl;
    a.hbl[g] = hbl;
    a.nb[g] = h[g] >> hbl;
    if (h[g]) {
      const long w = ((long)T + (8 >> hbl) - 1) / (8 >> hbl);
      waves = w > waves ? w : waves;
    }
    most = a.nb[g] > most ? a.nb[g] : most;
  }
  const int r = a.rot >> 1;
  a.vec = r > 0 && r % (a.interleaved ? 4 : 8) == 0 && apla_aligned16(a.table);
  const int groups = h2 ? 2 : 1;
  const long cap = (par ? PARAM_WGS : ROT_WGS) / groups;      // (the workspace of the sums has PARAM_WGS rows)
  long sp = (4096 + waves * groups - 1) / (waves * groups);
  sp = sp < most ? sp : most;
  a.splits = (int)(sp < cap ? sp : cap);
  a.T = T;
  long gx = (waves + 3) / 4;
  if (gx * a.splits > cap) gx = cap / a.splits;
  return dim3((unsigned)gx, (unsigned)(groups * a.splits));
}

int rot_check(const char* who, int T, int h1, int h2, const float* table, int P, int rot, int layout, const int32_t* pos, int seq_len) {
  APLA_REQUIRE(T > 0 && h1 >= 0 && h2 >= 0 && h1 + h2 > 0 && h1 + h2 <= 1024, "%s: need T > 0 and 1..1024 heads (T=%d heads=%d+%d)", who, T, h1, h2);
  APLA_REQUIRE(rot >= 0 && rot <= 64 && rot % 2 == 0 && (rot == 0 || (table && P > 0)), "%s: rot must be even, 0..64, with a table (rot=%d P=%d)", who, rot, P);
  APLA_REQUIRE(layout == APLA_ROT_HALF || layout == APLA_ROT_INTERLEAVED, "%s: unknown layout %d", who, layout);
  APLA_REQUIRE(seq_len >= 0 && (rot == 0 || pos || (seq_len ? seq_len : T) <= P), "%s: positions 0..%d without `pos` do not fit a table of %d rows", who,
               (seq_len ? seq_len : T) - 1, P);
  return APLA_OK;
}
int rows_check(const char* who, const char* name, const void* p, long ld, int heads) {
  APLA_REQUIRE(p && apla_aligned16(p) && ld >= heads * 64L && ld % 8 == 0, "%s: %s must be 16-byte aligned with a row stride >= %d that is a multiple of 8 (got %ld)",
               who, name, heads * 64, ld);
  return APLA_OK;
}

}  // namespace

extern "C" int apla_rotary(const void* x, long ldx, void* y, long ldy, int T, int heads, const float* table, int P, int rot, int layout,
                           const int32_t* pos, int seq_len, int inverse, hipStream_t stream) {
  int rc = rot_check("apla_rotary", T, heads, 0, table, P, rot, layout, pos, seq_len);
  if (rc == APLA_OK) rc = rows_check("apla_rotary", "x", x, ldx, heads);
  if (rc == APLA_OK) rc = rows_check("apla_rotary", "y", y, ldy, heads);
  if (rc != APLA_OK) return rc;
  RotArgs a = {};
  a.table = table; a.P = P; a.rot = rot; a.interleaved = layout == APLA_ROT_INTERLEAVED; a.pos = pos; a.seq_len = seq_len;
  const dim3 grid = rot_plan(a, T, heads, 0, false);
  a.x = (const bf16*)x; a.ldx = ldx; a.y = (bf16*)y; a.ldy = ldy;
  a.sign = inverse ? -1.f : 1.f;
  hipLaunchKernelGGL((rotary_kernel<0, false, false>), grid, dim3(256), 0, stream, a);
  APLA_CHECK_LAUNCH("apla_rotary");
  return APLA_OK;
}

extern "C" long apla_qk_norm_rotary_workspace_bytes(void) { return (long)PARAM_WGS * 128 * 4; }

extern "C" int apla_qk_norm_rotary_fwd(const void* x, long ldx, void* y, long ldy, int T, int Hq, int Hkv, int norm, float eps, const float* qw,
                                       const float* kw, const float* qb, const float* kb, const float* table, int P, int rot, int layout,
                                       const int32_t* pos, int seq_len, hipStream_t stream) {
  int rc = rot_check("apla_qk_norm_rotary_fwd", T, Hq, Hkv, table, P, rot, layout, pos, seq_len);
  if (rc == APLA_OK) rc = rows_check("apla_qk_norm_rotary_fwd", "x", x, ldx, Hq + Hkv);
  if (rc == APLA_OK) rc = rows_check("apla_qk_norm_rotary_fwd", "y", y, ldy, Hq + Hkv);
  if (rc != APLA_OK) return rc;
  APLA_REQUIRE((norm == APLA_NORM_LAYER || norm == APLA_NORM_RMS) && eps >= 0.f, "apla_qk_norm_rotary_fwd: unknown norm %d or eps < 0", norm);
  RotArgs a = {};
  a.table = table; a.P = P; a.rot = rot; a.interleaved = layout == APLA_ROT_INTERLEAVED; a.pos = pos; a.seq_len = seq_len;
  const dim3 grid = rot_plan(a, T, Hq, Hkv, false);
  a.x = (const bf16*)x; a.ldx = ldx; a.y = (bf16*)y; a.ldy = ldy;
  a.sign = 1.f; a.eps = eps; a.w[0] = qw; a.w[1] = kw; a.b[0] = qb; a.b[1] = kb;
  if (norm == APLA_NORM_LAYER) hipLaunchKernelGGL((rotary_kernel<1, false, false>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((rotary_kernel<2, false, false>), grid, dim3(256), 0, stream, a);
  APLA_CHECK_LAUNCH("apla_qk_norm_rotary_fwd");
  return APLA_OK;
}

extern "C" int apla_qk_norm_rotary_bwd(const void* dy, long lddy, const void* x, long ldx, void* dx, long lddx, int T, int Hq, int Hkv, int norm,
                                       float eps, const float* qw, const float* kw, const float* table, int P, int rot, int layout,
                                       const int32_t* pos, int seq_len, float* dparams, void* workspace, long workspace_bytes, hipStream_t stream) {
  int rc = rot_check("apla_qk_norm_rotary_bwd", T, Hq, Hkv, table, P, rot, layout, pos, seq_len);
  if (rc == APLA_OK) rc = rows_check("apla_qk_norm_rotary_bwd", "dy", dy, lddy, Hq + Hkv);
  if (rc == APLA_OK) rc = rows_check("apla_qk_norm_rotary_bwd", "x", x, ldx, Hq + Hkv);
  if (rc == APLA_OK) rc = rows_check("apla_qk_norm_rotary_bwd", "dx", dx, lddx, Hq + Hkv);
  if (rc != APLA_OK) return rc;
  APLA_REQUIRE((norm == APLA_NORM_LAYER || norm == APLA_NORM_RMS) && eps >= 0.f, "apla_qk_norm_rotary_bwd: unknown norm %d or eps < 0", norm);
  APLA_REQUIRE(!dparams || (workspace && workspace_bytes >= apla_qk_norm_rotary_workspace_bytes()), "apla_qk_norm_rotary_bwd: parameter gradients need %ld bytes of workspace (got %ld)",
               apla_qk_norm_rotary_workspace_bytes(), workspace_bytes);
  RotArgs a = {};
  a.table = table; a.P = P; a.rot = rot; a.interleaved = layout == APLA_ROT_INTERLEAVED; a.pos = pos; a.seq_len = seq_len;
  const dim3 grid = rot_plan(a, T, Hq, Hkv, dparams != nullptr);
  a.dy = (const bf16*)dy; a.lddy = lddy; a.x = (const bf16*)x; a.ldx = ldx; a.y = (bf16*)dx; a.ldy = lddx;
  a.sign = -1.f; a.eps = eps; a.w[0] = qw; a.w[1] = kw; a.partial = (float*)workspace;
  if (norm == APLA_NORM_LAYER) {
    if (dparams) hipLaunchKernelGGL((rotary_kernel<1, true, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((rotary_kernel<1, true, false>), grid, dim3(256), 0, stream, a);
  } else {
    if (dparams) hipLaunchKernelGGL((rotary_kernel<2, true, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((rotary_kernel<2, true, false>), grid, dim3(256), 0, stream, a);
  }
  APLA_CHECK_LAUNCH("apla_qk_norm_rotary_bwd");
  if (dparams) {
    hipLaunchKernelGGL(rotary_param_sum_kernel, dim3(16), dim3(256), 0, stream, (const float*)workspace, (int)(grid.x * a.splits), Hkv ? 2 : 1, dparams);
    APLA_CHECK_LAUNCH("apla_qk_norm_rotary_bwd");
  }
  return APLA_OK;
}
