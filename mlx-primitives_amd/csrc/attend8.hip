// Attention over the 8-bit paged KV cache on gfx950 (mpx_cache8.h has the
// formula): decode, a few queries behind a prefix, prompts.
//
// The rows of one K/V head are its group's query heads for every query: row
// rho = query * G + head of the group, in blocks of 16 NR rows. A workgroup
// takes one block and one partition of the tokens, of which each of its four waves
// takes a quarter, one run, in tiles of 32; they meet in LDS at the end. Or its waves
// take four heads and all of the partition each. Partitions meet in
// attend8_merge_kernel.
//
// Codes go from memory to registers in the layout that the matrix
// instructions take them in, no LDS and no exchange between lanes:
//   S^T (16 tokens x 16 rows) = K Q^T. Lane i + 16 q reads token row i, bytes
//   [16 (q + 4 j), 16 (q + 4 j) + 16): any order of the summed dims is one, so
//   Q is read in the same. Token row i of half f is token 8 (i / 4) + 4 f + i % 4
//   of the tile, so that the values of S^T that lane (i, q) gets (C rows 4 q + r
//   of both halves) are row i's tokens 8 q .. 8 q + 7: the slice of P^T that it
//   holds in the second product.
//   O^T (16 dims x 16 rows) = V^T P^T. Lane (i, q) reads of tokens 8 q .. 8 q + 7
//   the D / 16 bytes of dims D / 16 i .. and has, byte n of the eight, the operand
//   of dims {D / 16 i + n}: a transposition of bytes within the lane. Lane (i, q)
//   ends with dims D / 4 q .. of row i.
// The products are fp16 for both 16-bit types of queries (float32 ones have their
// own, 16 x 16 x 4). e4m3 codes are decoded to it exactly. int8 codes are not
// decoded at all: with the sign bit turned, a code k is the byte k + 128, and with
// a zero byte above it the fp16 number (k + 128) 2^-24, a subnormal, which the matrix
// instructions take exactly; 128 times the sum of the other operand is taken off
// again, for S before the sum starts, for O at its end. K's scales multiply S
// (float32); V's multiply P, in the exponent. A row has two running maxima: of a score,
// x, for the sum of weights, and of x + log2 of V's scale for P and O, so that P, which is
// rounded once to fp16 (relative error 2^-11), starts at 2^14 for the largest contribution
// and keeps its bits down to 2^-28 of that, however far apart the scales of V are. bf16
// outputs do not show that rounding; for fp16 ones what it leaves is a second operand.
//
// Decode is memory bound where it fills the chip: 64 sequences of 512 to 8192 tokens,
// 32 heads of D 128, int8: 422 us and 7.6 for the merge, 2.29 GB at 5.4 TB/s (a large copy
// runs at 4.91); 560 us before the look-ups, codes and products of consecutive tiles
// overlapped, and 504 with waves that share a head's tokens. Small calls are chains of
// latencies (lengths, page ids, scales, codes, products, sums, merge): four sequences
// of 700 to 2100 tokens, 32 heads over 8: 8.0 and 3.2 us.
#include <algorithm>
#include <cmath>

#include "mpx_code8.h"
#include "mpx_rows.h"

namespace mpx {

struct Attend8Params {
  const void* q;
  const unsigned char *kpool, *vpool;
  const float *kscale, *vscale;
  const int32_t *bt, *cl, *qstart;
  const float* slopes;
  void* o;
  int64_t qs[3], os[3];  // (batch, head, seq) element strides
  float* ws_o;           // (B H Sq, max_parts, DK)
  float* ws_ml;          // (B H Sq, max_parts, 2), m in log2 units
  int B, Sq, H, H_kv, G, D, num_blocks, bs, max_blocks, causal;
  int o_rows16;    // o's base and strides are multiples of 16 bytes
  int wave_heads;  // the waves of the register form take heads, not tokens
  int part, max_parts;   // tokens of a partition, and how many there is room for
  int reach, step;       // tokens that fit them; partitions of longer sequences grow, in
                         // multiples of this power of two
  int blocks, span;      // row blocks and their rows
  u32 magic, shift;      // n / bs = n * magic / 2^(32 + shift) for n < 2^31
  float c;               // scale * log2(e)
};

constexpr int kTile8 = 32;

// Where a sequence's queries start: positions past any cache, or before all, are
// alike, and what follows stays within 32 bits.
__device__ __forceinline__ int start8(const Attend8Params& p, int b) {
  return p.qstart ? max(-(1 << 30), min(p.qstart[b], 1 << 30)) : 0;
}
// Tokens that rows up to `rho` (the last of a block) can see.
__device__ __forceinline__ int seen8(const Attend8Params& p, int ctx, int b, int rho) {
  if (!p.causal) return ctx;
  const int sq = min(rho, p.Sq * p.G - 1) / p.G;
  return max(0, min(ctx, start8(p, b) + sq + 1));
}
__device__ __forceinline__ int context8(const Attend8Params& p, int b) {
  return max(0, min(p.cl[b], p.max_blocks * p.bs));
}
// Tokens of a partition of a sequence: the plan's where all of its tokens fit that many
// partitions, else its tokens over the partitions. (The host knows the table's width, which
// may be many times what is in it.)
__device__ __forceinline__ int part8(const Attend8Params& p, int ctx, int b) {
  const int seen = seen8(p, ctx, b, p.Sq * p.G - 1);
  if (seen <= p.reach) return p.part;
  const u32 n = (u32)p.max_parts, each = ((u32)seen + n - 1) / n;
  return (int)((each + (u32)p.step - 1) & ~((u32)p.step - 1));
}
// Page of the n-th token of a table.
__device__ __forceinline__ u32 page_of8(const Attend8Params& p, u32 n) {
  return p.bs == 1 ? n : __umulhi(n, p.magic) >> p.shift;
}

template <int QT>
struct Operand8 {
  typedef u32x4 T;
};
template <>
struct Operand8<MPX_F32> {
  typedef f32x4 T;
};

// N values (4, 8 or 16) rounded to T, in as few stores as o's rows allow.
template <int N, typename T>
__device__ __forceinline__ void store_row8(T* out, const float* x, int rows16) {
  if (!rows16) {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = from_f<T>(x[i]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *(f32x4*)(out + i) = (f32x4){x[i], x[i + 1], x[i + 2], x[i + 3]};
  } else {
    constexpr bool BF = __is_same(T, __bf16);
    if constexpr (N == 4) {
      *(u32x2*)out = (u32x2){pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3])};
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 8)
        *(u32x4*)(out + i) = (u32x4){pack2<BF>(x[i], x[i + 1]), pack2<BF>(x[i + 2], x[i + 3]),
                                     pack2<BF>(x[i + 4], x[i + 5]), pack2<BF>(x[i + 6], x[i + 7])};
    }
  }
}

__device__ __forceinline__ u32 bytes4(u32 hi, u32 lo, u32 sel) {
  return __builtin_amdgcn_perm(hi, lo, sel);
}

// WHOLE8: page sizes that are multiples of 8, where tokens 8 q .. 8 q + 7 share a
// page and its scales (partitions start at multiples of 128).
template <int QT, bool I8, int DK, int NR, bool WHOLE8>
__global__ __launch_bounds__(256) void attend8_kernel(Attend8Params p) {
  constexpr int KJ = DK / 64;  // 16-byte chunks of a token row a lane reads
  constexpr int VB = DK / 16;  // V bytes of a token a lane reads
  constexpr int VW = VB / 4;
  constexpr int NK = WHOLE8 ? 1 : 2, NV = WHOLE8 ? 1 : 8;  // pages of a lane's K rows and V rows
  constexpr bool F32 = QT == MPX_F32, RAW = I8 && !F32;    // RAW: codes as fp16's subnormal bits
  typedef typename Elem<QT>::T T;
  __shared__ float s_ml[4][NR][16][3];
  __shared__ __align__(16) float s_o[4][NR][4][64][VB];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i16 = lane & 15, q4 = lane >> 4;
  // The waves take four heads of the same tokens, or one head and a share each.
  const bool heads = p.wave_heads != 0;
  const int hs = heads ? p.H_kv >> 2 : p.H_kv;
  const int blk = p.blocks == 1 ? 0 : (int)(blockIdx.x / (u32)hs), hx = blockIdx.x - blk * hs;
  const int hk = heads ? 4 * hx + wave : hx, part = blockIdx.y, b = blockIdx.z;
  const int R = p.Sq * p.G, rho0 = blk * 16 * NR;
  const int ctx = context8(p, b);
  const int tmax = seen8(p, ctx, b, rho0 + 16 * NR - 1);
  const int tokens = part8(p, ctx, b);
  const int p0 = part * tokens, p1 = min(p0 + tokens, tmax);
  const bool alone = p.max_parts == 1 || tmax <= tokens;  // no other partition: o right away
  if (p0 >= p1 && (!alone || part > 0)) return;  // (the merge knows)
  const int pg0 = page_of8(p, p0), base = pg0 * p.bs;
  const int32_t* const table = p.bt + (int64_t)b * p.max_blocks + pg0;

  // The waves share the partition's tokens evenly, each a run [w0, w1). Its pages
  // are looked up a window at a time: lane l has the first row, and the scales, of
  // unit l of the window, a unit being eight tokens (WHOLE8) or one; tokens past
  // the run are clamped into it. Lanes then fetch what they need from each other.
  constexpr int kUnit = WHOLE8 ? 8 : 1, kWindow = 64 * kUnit;
  const int share = heads ? p1 - p0 : ((p1 - p0 + 3) / 4 + kTile8 - 1) / kTile8 * kTile8;
  const int w0 = heads ? p0 : p0 + wave * share, w1 = min(w0 + share, p1);
  const int edge = (w1 - 1) & ~(kUnit - 1);
  const float* const ks_head = p.kscale + hk;
  const float* const vs_head = p.vscale + hk;
  struct Window {
    u32 row;  // ~0: no page
    float ks, vs;
  };
  struct Found {
    int id;
    u32 slot;
  };
  auto find = [&](int t0) __attribute__((always_inline)) {
    const u32 n = (u32)(min(t0 + kUnit * lane, edge) - base);
    const u32 i = page_of8(p, n);
    return Found{table[i], n - i * (u32)p.bs};
  };
  auto open = [&](const Found& f) __attribute__((always_inline)) {
    const bool ok = (u32)f.id < (u32)p.num_blocks;
    const uint64_t at = (uint64_t)(ok ? (u32)f.id : 0u) * (u32)p.H_kv;
    const float ks = ks_head[at], vs = vs_head[at];
    return Window{ok ? (u32)f.id * (u32)p.bs + f.slot : ~0u, ok ? ks : 0.f, ok ? vs : 0.f};
  };
  Found found[2];
  if (w0 < w1) {
    found[0] = find(w0);
    found[1] = find(w0 + kWindow);
  }

  // Rows: their position, limit and slope, and Q in the operand layout. (A
  // negative scale turns Q round: what is left is positive.) bf16 rows become
  // fp16 times a power of two that brings their largest value to 2^13: exact but
  // for values under 2^-27 of it, whose rounding is that of float32 sums.
  const bool turn = p.c < 0.f;
  int lim[NR], pos[NR];
  float slope[NR], c[NR];  // c: what S of the row is multiplied by, but for K's scales
  u32x4 qb[NR][F32 ? 1 : 2 * KJ];
  float qf[NR][F32 ? 16 * KJ : 1];
  f32x4 start[NR];         // where the sums of S start: 0, or for RAW -128 sum q
  int least = w1;          // what all rows see
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int rho = rho0 + 16 * n + i16;
    const bool have = rho < R;
    const int sq = have ? rho / p.G : 0, h = hk * p.G + (have ? rho - sq * p.G : 0);
    pos[n] = p.qstart || p.Sq > 1 ? start8(p, b) + sq : ctx;
    lim[n] = have && p.causal ? min(w1, pos[n] + 1) : w1;
    least = min(least, lim[n]);
    slope[n] = p.slopes ? p.slopes[h] * kLog2e : 0.f;
    const T* row = (const T*)p.q + b * p.qs[0] + h * p.qs[1] + sq * p.qs[2];
    V8<T> x[2 * KJ];
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 2 * KJ; ++j) {
      const int d = 16 * (q4 + 4 * (j >> 1)) + 8 * (j & 1);
      if (have && d < p.D) {
        x[j] = load8(row + d);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[j].v[e] = from_f<T>(0.f);
      }
      if constexpr (QT == MPX_BF16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(to_f(x[j].v[e])));
      }
    }
    float up = turn ? -1.f : 1.f;
    c[n] = fabsf(p.c);
    if constexpr (QT == MPX_BF16) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = pair_max32(top);
      const int e = min(max((int)(__float_as_uint(top) >> 23), 14), 253);  // exponent, 127 over
      up *= __uint_as_float((u32)(267 - e) << 23);                         // 2^(13 - (e - 127))
      c[n] *= __uint_as_float((u32)(e - 13) << 23);
    }
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 2 * KJ; ++j) {
      if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) qf[n][8 * j + e] = x[j].v[e] * up;
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const u32 y = pack2<false>(to_f(x[j].v[2 * w]) * up, to_f(x[j].v[2 * w + 1]) * up);
          qb[n][j][w] = y;
          // (subnormals included, which a dot product may drop)
          if constexpr (RAW) sum += h2f<false>((uint16_t)y) + h2f<false>((uint16_t)(y >> 16));
        }
      }
    }
    start[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if constexpr (RAW) {
      sum += __shfl_xor(sum, 16, 64);
      sum = pair_sum32(sum) * -0x1p-17f;
      start[n] = (f32x4){sum, sum, sum, sum};
      c[n] *= 0x1p24f;
    }
  }
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1) least = min(least, __shfl_xor(least, off, 64));
  least = __builtin_amdgcn_readfirstlane(least);

  f32x4 o[NR][VB];
  // Running maxima, whole numbers, of x and of x + log2 of V's scale; sums of 2^(x - m).
  float m[NR], my[NR], l[NR];
  f32x4 pw[NR];  // RAW: what the 128 of every code adds to O, alike for all dims
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    m[n] = my[n] = -INFINITY;
    l[n] = 0.f;
    pw[n] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < VB; ++v) o[n][v] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  // P is 2^kStart at its running maximum, which moves where a row's grows by more than
  // kSlack, so that O is seldom rescaled; that of the sum has float32's range (kFar).
  constexpr float kStart = F32 ? 0.f : 14.f, kSlack = F32 ? 8.f : 1.5f, kFar = 64.f;
  const u32 row_bytes = (u32)p.H_kv * (u32)p.D;
  // This lane's bytes of a row: K chunks 16 (q + 4 j), V bytes VB i. (Lanes past the
  // head dim read others of the row, which Q's zeros and the stores leave out.)
  const int k_at = 16 * q4 < p.D ? 16 * q4 : 0, v_at = VB * i16 < p.D ? VB * i16 : 0;
  const unsigned char* const k_lane = p.kpool + (u32)(hk * p.D + k_at);
  const unsigned char* const v_lane = p.vpool + (u32)(hk * p.D + v_at);
  u32 k_more[KJ];
#pragma unroll
  for (int j = 0; j < KJ; ++j) k_more[j] = k_at + 64 * j < p.D ? 64 * j : 0;
  const bool all_dims = p.D == DK;

  struct Raw {
    u32x4 k[2][KJ];
    u32 v[8][VW];
    float ks[NV], vs[NV];
    u32 ok;  // V's pages, by bits
  };
  // The codes of the tile that starts at token `in` of the window.
  auto load = [&](const Window& w, int in, Raw& r) __attribute__((always_inline)) {
    auto of = [&](int unit, auto x) __attribute__((always_inline)) {
      return __builtin_bit_cast(
          decltype(x), __builtin_amdgcn_ds_bpermute(4 * unit, __builtin_bit_cast(int, x)));
    };
    const int unit = in / kUnit;
    u32 kr = 0;
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      if (WHOLE8 && f) {
        kr += 4;
      } else {
        kr = of(unit + (WHOLE8 ? i16 >> 2 : 8 * (i16 >> 2) + 4 * f + (i16 & 3)), w.row);
        kr = (kr == ~0u ? 0u : kr) + (WHOLE8 ? i16 & 3 : 0);
      }
      const unsigned char* src = k_lane + (uint64_t)kr * row_bytes;
#pragma unroll
      for (int j = 0; j < KJ; ++j) r.k[f][j] = *(const u32x4*)(src + k_more[j]);
    }
    r.ok = 0;
    const unsigned char* src = nullptr;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j == 0 || !WHOLE8) {
        const int at = unit + (WHOLE8 ? q4 : 8 * q4 + j);
        const u32 vr = of(at, w.row);
        r.ks[WHOLE8 ? 0 : j] = of(at, w.ks);
        r.vs[WHOLE8 ? 0 : j] = of(at, w.vs);
        r.ok |= vr == ~0u ? 0u : (WHOLE8 ? 0xffu : 1u << j);
        src = v_lane + (uint64_t)(vr == ~0u ? 0u : vr) * row_bytes;
      } else {
        src += row_bytes;
      }
      if constexpr (VW == 4) {
        const u32x4 x = *(const u32x4*)src;
#pragma unroll
        for (int w2 = 0; w2 < 4; ++w2) r.v[j][w2] = x[w2];
      } else if constexpr (VW == 2) {
        const u32x2 x = *(const u32x2*)src;
        r.v[j][0] = x[0];
        r.v[j][1] = x[1];
      } else {
        r.v[j][0] = *(const u32*)src;
      }
    }
  };

  auto step = [&](int t0, Raw& r) __attribute__((always_inline)) {
    // Tokens behind the partition or without a page: no weight, and e4m3 codes
    // none that may be NaN (0 * NaN is none).
    u32 live = r.ok;
    const int rest = w1 - t0 - 8 * q4;
    if (rest < 8) live &= rest <= 0 ? 0u : (1u << rest) - 1;
    const bool plain = __all(live == 0xffu) && t0 + kTile8 <= least && !p.slopes;
    if (__any(live != 0xffu)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!((live >> j) & 1u)) {
          if constexpr (!I8) {
#pragma unroll
            for (int w = 0; w < VW; ++w) r.v[j][w] = 0u;
          }
          if (j < NV) r.ks[j] = r.vs[j] = 0.f;
        }
      }
    }
    if (!I8 && !all_dims) {
#pragma unroll
      for (int j = 0; j < KJ; ++j)
        if (16 * (q4 + 4 * j) >= p.D) r.k[0][j] = r.k[1][j] = (u32x4){0u, 0u, 0u, 0u};
    }
    f32x4 s[NR][2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
#pragma unroll
      for (int n = 0; n < NR; ++n) s[n][f] = start[n];
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        if constexpr (F32) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float a = decode1<I8>(r.k[f][j][e >> 2], e & 3);
#pragma unroll
            for (int n = 0; n < NR; ++n)
              s[n][f] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, qf[n][16 * j + e], s[n][f], 0, 0, 0);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            u32x4 a;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const u32 x = r.k[f][j][2 * e + w];
              if constexpr (RAW) {
                a[2 * w] = bytes4(0u, x ^ 0x80808080u, 0x0c010c00u);
                a[2 * w + 1] = bytes4(0u, x ^ 0x80808080u, 0x0c030c02u);
              } else {
                a[2 * w] = decode2<false, false>(x, 0);
                a[2 * w + 1] = decode2<false, false>(x, 1);
              }
            }
#pragma unroll
            for (int n = 0; n < NR; ++n)
              s[n][f] = mfma16x16x32<false>(a, qb[n][2 * j + e], s[n][f]);
          }
        }
      }
    }
    // V's scales as 2^(ve + vl), ve whole: exact sums with the maxima. (Scales under 2^-120
    // count as that.)
    float ve[NV], vl[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const float v = fmaxf(r.vs[j], 0x1p-120f);
      ve[j] = (float)__builtin_amdgcn_frexp_expf(v);
      vl[j] = __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(v));
    }
    float pv[NR][8];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float k = WHOLE8 ? r.ks[0] * c[n] : 1.f;  // what pv is multiplied by yet
#pragma unroll
      for (int j = 0; j < 8; ++j)
        pv[n][j] = s[n][j >> 2][j & 3] * (WHOLE8 ? 1.f : r.ks[WHOLE8 ? 0 : j] * c[n]);
      if (!plain) {
        int t = t0 + 8 * q4;
        asm volatile("" : "+v"(t));  // (not ahead of the branch)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float x = pv[n][j] * k;
          if (p.slopes) x += slope[n] * (float)(t + j - pos[n]);
          pv[n][j] = t + j < lim[n] && ((live >> j) & 1u) ? x : -INFINITY;
        }
        k = 1.f;
      }
      float mx = pv[n][0], ym = WHOLE8 ? 0.f : pv[n][0] + (ve[0] + vl[0]);
#pragma unroll
      for (int j = 1; j < 8; ++j) {
        mx = fmaxf(mx, pv[n][j]);
        if constexpr (!WHOLE8) ym = fmaxf(ym, pv[n][j] + (ve[WHOLE8 ? 0 : j] + vl[WHOLE8 ? 0 : j]));
      }
      mx *= k;
      if constexpr (WHOLE8) ym = mx + (ve[0] + vl[0]);
      if (__any(ym > my[n] + kSlack || mx > m[n] + kFar)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        ym = fmaxf(ym, __shfl_xor(ym, 16, 64));
        const float mn = fmaxf(m[n], ceilf(pair_max32(mx)));
        const float yn = fmaxf(my[n], ceilf(pair_max32(ym)));
        const float alpha = my[n] == -INFINITY ? 0.f : fast_exp2(my[n] - yn);
        l[n] *= m[n] == -INFINITY ? 0.f : fast_exp2(m[n] - mn);
        pw[n] *= alpha;
#pragma unroll
        for (int v = 0; v < VB; ++v) o[n][v] *= alpha;
        m[n] = mn;
        my[n] = yn;
      }
      const float ref = my[n] == -INFINITY ? 0.f : my[n] - kStart;
      const float sub = m[n] == -INFINITY ? 0.f : m[n];
      if constexpr (WHOLE8) {
        // The sum of the weights takes V's scale out again. So that P is in float32's range for
        // any weight that counts there, a scale counts as 2^-80 of the largest contribution's
        // at least (nothing to O).
        const float low = my[n] - m[n] - 80.f;  // (NaN before the first token)
        const bool tiny = low > ve[0] + vl[0];
        const float e = tiny ? low : ve[0], f = tiny ? 0.f : vl[0];
        const float off = (e - ref) + f;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          pv[n][j] = fast_exp2(__builtin_fmaf(pv[n][j], k, off));
          sum += pv[n][j];
        }
        l[n] = __builtin_fmaf(sum, fast_exp2((ref - e - sub) - f), l[n]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int at = WHOLE8 ? 0 : j;
          l[n] += fast_exp2(pv[n][j] - sub);
          pv[n][j] = fast_exp2(pv[n][j] + ((ve[at] - ref) + vl[at]));
        }
      }
    }
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int v = 0; v < VB; ++v) {
          const float a = decode1<I8>(r.v[j][v >> 2], v & 3);
#pragma unroll
          for (int n = 0; n < NR; ++n)
            o[n][v] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, pv[n][j], o[n][v], 0, 0, 0);
        }
    } else {
      // (float16 outputs show P's rounding: what it leaves is a second operand)
      constexpr int PP = QT == MPX_F16 ? 2 : 1;
      u32x4 pb[PP][NR];
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const u32 x = pack2<false>(pv[n][2 * w], pv[n][2 * w + 1]);
          pb[0][n][w] = x;
          if constexpr (PP == 2)
            pb[PP - 1][n][w] = pack2<false>(pv[n][2 * w] - h2f<false>((uint16_t)x),
                                            pv[n][2 * w + 1] - h2f<false>((uint16_t)(x >> 16)));
        }
      if constexpr (RAW) {
        const u32x4 a = {0x00800080u, 0x00800080u, 0x00800080u, 0x00800080u};
#pragma unroll
        for (int k = 0; k < PP; ++k)
#pragma unroll
          for (int n = 0; n < NR; ++n) pw[n] = mfma16x16x32<false>(a, pb[k][n], pw[n]);
      }
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        u32 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = RAW ? r.v[j][w] ^ 0x80808080u : r.v[j][w];
        u32 col[4][2];  // e4m3: dword of byte n: tokens 0..3, 4..7
        if constexpr (!RAW) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const u32* y = x + 4 * g;
            const u32 x0 = bytes4(y[1], y[0], 0x05010400u), x1 = bytes4(y[1], y[0], 0x07030602u);
            const u32 y0 = bytes4(y[3], y[2], 0x05010400u), y1 = bytes4(y[3], y[2], 0x07030602u);
            col[0][g] = bytes4(y0, x0, 0x05040100u);
            col[1][g] = bytes4(y0, x0, 0x07060302u);
            col[2][g] = bytes4(y1, x1, 0x05040100u);
            col[3][g] = bytes4(y1, x1, 0x07060302u);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u32x4 a;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            a[k] = RAW ? bytes4(x[2 * k + 1], x[2 * k], 0x0c040c00u + 0x00010001u * e)
                       : decode2<false, false>(col[e][k >> 1], k & 1);
#pragma unroll
          for (int k = 0; k < PP; ++k)
#pragma unroll
            for (int n = 0; n < NR; ++n)
              o[n][4 * w + e] = mfma16x16x32<false>(a, pb[k][n], o[n][4 * w + e]);
        }
      }
    }
  };

  // While a tile is computed, the next one's codes are on their way, and while a
  // window is, the scales of the next one and the page ids of the one after that.
  if (w0 < w1) {
    Raw raw[2];
    Window now = open(found[0]);
    load(now, 0, raw[0]);
    for (int t0 = w0; t0 < w1; t0 += kWindow) {
      const Window then = open(found[1]);
      found[1] = find(t0 + 2 * kWindow);
#pragma unroll 1
      for (int in = 0; in < kWindow && t0 + in < w1; in += 2 * kTile8) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int t = t0 + in + u * kTile8;
          if (t < w1) {
            const bool last = in + (u + 1) * kTile8 == kWindow;
            Window w;
            w.row = last ? then.row : now.row;
            w.ks = last ? then.ks : now.ks;
            w.vs = last ? then.vs : now.vs;
            load(w, last ? 0 : in + (u + 1) * kTile8, raw[u ^ 1]);
            step(t, raw[u]);
          }
        }
      }
      now = then;
    }
  }

  // The waves meet once: each leaves its sums and maxima and takes a quarter of the dims of
  // all four. What leaves the workgroup is O over the sum of weights (no larger than V), and for
  // a partition that sum with the maximum it stands over.
  constexpr int kBack = RAW ? 24 : 0;  // (subnormal codes are 2^-24)
  auto factor = [&](float y, float M) __attribute__((always_inline)) {  // 2^(y - kStart - M)
    return y == -INFINITY ? 0.f : __builtin_amdgcn_ldexpf(1.f, (int)(y - M - kStart) + kBack);
  };
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    l[n] += __shfl_xor(l[n], 16, 64);
    l[n] = pair_sum32(l[n]);
    if (!heads && q4 == 0) {
      s_ml[wave][n][i16][0] = m[n];
      s_ml[wave][n][i16][1] = l[n];
      s_ml[wave][n][i16][2] = my[n];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int v = 0; v < VB; v += 4) {
        f32x4 x;
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = o[n][v + k][e] = o[n][v + k][e] - (RAW ? pw[n][0] : 0.f);
        if (!heads) *(f32x4*)&s_o[wave][n][e][lane][v] = x;
      }
  }
  if (!heads) __syncthreads();
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const int rho = rho0 + 16 * n + i16;
    if (rho >= R) continue;
    const int sq = rho / p.G, h = hk * p.G + rho - sq * p.G;
    const int64_t slot = (((int64_t)b * p.H + h) * p.Sq + sq) * p.max_parts + part;
    T* const row = (T*)p.o + b * p.os[0] + h * p.os[1] + sq * p.os[2];
    // 1 / l for a row's end (no token: 0 * inf = NaN), or a partition's.
    auto over = [&](float L) __attribute__((always_inline)) {
      return !alone && L == 0.f ? 0.f : 1.f / L;
    };
    // VB dims from d on.
    auto put = [&](int d, const float* x) __attribute__((always_inline)) {
      if (alone) {
        if (d >= p.D) return;
        store_row8<VB>(row + d, x, p.o_rows16);
      } else {
#pragma unroll
        for (int v = 0; v < VB; v += 4)
          *(f32x4*)(p.ws_o + slot * DK + d + v) = (f32x4){x[v], x[v + 1], x[v + 2], x[v + 3]};
      }
    };
    auto put_ml = [&](float M, float L) __attribute__((always_inline)) {
      if (!alone && q4 == 0) {
        p.ws_ml[2 * slot] = M;
        p.ws_ml[2 * slot + 1] = L;
      }
    };
    if (heads) {
      const float inv = over(l[n]), f = factor(my[n], m[n]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x[VB];
#pragma unroll
        for (int v = 0; v < VB; ++v) x[v] = o[n][v][e] * inv * f;
        put(4 * VB * q4 + VB * e, x);
      }
      put_ml(m[n], l[n]);
      continue;
    }
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, s_ml[w][n][i16][0]);
    float acc[VB];
#pragma unroll
    for (int v = 0; v < VB; ++v) acc[v] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = s_ml[w][n][i16][0];
      L = fmaf(mw == -INFINITY ? 0.f : fast_exp2(mw - M), s_ml[w][n][i16][1], L);
    }
    const float inv = over(L);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = factor(s_ml[w][n][i16][2], M);
#pragma unroll
      for (int v = 0; v < VB; ++v) acc[v] = fmaf(s_o[w][n][wave][lane][v] * inv, f, acc[v]);
    }
    put(4 * VB * q4 + VB * wave, acc);
    if (wave == 0) put_ml(M, L);
  }
}

// ---------------------------------------------------------------------------
// More rows than that (prompts, longer chat turns; 16-bit queries): 128 rows a
// workgroup, 32 for each of its four waves, which share each tile of tokens in
// LDS as 16-bit values. What the register form above does for every 32 rows, the
// decoding, is done once for 128, and a wave has the larger matrix instructions
// (32 x 32 x 16) to feed:
//   S^T (32 tokens x 32 rows) = K Q^T: lane (i, h) = (l % 32, l / 32) reads token row
//   i with its bits 2 and 3 exchanged, so that the scores it gets, C rows
//   8 (r / 4) + 4 h + r % 4 of row i, are tokens 16 (r / 8) + 8 h + r % 8: the slices of
//   P^T that it holds in O^T (32 dims x 32 rows) = V^T P^T. V^T comes through the
//   transposing LDS read. LDS chunks of 16 bytes are exchanged by the row so that
//   the reads of 16 rows meet different banks.
// Bound by the matrix instructions and the softmax and decoding next to them: four
// prompts of 4096 tokens, 32 heads over 8 of D 128, bf16 over e4m3: 628 us, 876
// TFLOP/s; the library's 8192^3 product runs at 1290 on the same card. A tile takes
// 1.15 us of a CU with two workgroups on it, of which 0.43 are products.
//
// While a tile is computed, the codes of the next one are on their way to
// registers, and the first wave looks up pages and scales of the one after that;
// one barrier a tile.
// Decoded values: bf16 holds value = code * scale exactly where the scale is a
// power of two (any other: rounded once, 2^-8). fp16 holds code * scale / reference *
// 2^7, the reference of K being the largest scale of the tile, that of V the
// largest so far: exact down to 2^-22 of it. The weights are rounded to the type of the
// values that they are multiplied with, as the framework's other 16-bit attention does
// (bf16: outputs 2.1e-3 from 64 bits, one rounding alone is 1.6e-3); their float32 sum is
// of the rounded ones, so that what they have in common cancels.
constexpr int kRows8 = 128;

template <int DK>
constexpr int kTokens8 = DK == 256 ? 32 : 64;  // tokens of a tile (two stages: 64 KB at most)

// Slot of chunk c of row r (K's rows are read one a lane, V's four rows of a
// 16-lane group at a time).
template <int DK>
__device__ __forceinline__ int k_slot8(int r, int c) {
  return DK == 64 ? c ^ (((r >> 1) & 1) << 2 | ((r >> 2) & 3)) : c ^ (r & 15);
}
template <int DK>
__device__ __forceinline__ int v_slot8(int r, int c) {
  return DK == 64 ? c ^ (((r >> 1) & 1) << 2 | ((r >> 2) & 3)) : c ^ (4 * (r & 3)) ^ (r & 1);
}

// Four codes times s as two packed pairs. POW2: s is a power of two, which the
// conversion of e4m3 takes along. int8 codes with the sign bit turned are the bytes
// k + 128: under fp16's exponent of 2^10 they are 1024 + 128 + k, else float32 with
// 128 s taken off in the product (one rounding, that of k s).
template <bool I8, bool BF16, bool POW2>
__device__ __forceinline__ u32x2 value4(u32 x, float s) {
  if constexpr (!I8 && POW2) {
    if constexpr (BF16)
      return (u32x2){__builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, s, false)),
                     __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, s, true))};
    else
      return (u32x2){__builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, s, false)),
                     __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, s, true))};
  }
  if constexpr (I8) {
    const u32 y = x ^ 0x80808080u;
    if constexpr (POW2 && !BF16) {
      const f16x2 off = {(_Float16)-1152.f, (_Float16)-1152.f}, k = {(_Float16)s, (_Float16)s};
      const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, y, 0x04010400u));
      const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, y, 0x04030402u));
      return (u32x2){__builtin_bit_cast(u32, (lo + off) * k), __builtin_bit_cast(u32, (hi + off) * k)};
    }
    const float c = -128.f * s;
    auto value = [&](int i) { return __builtin_fmaf((float)((y >> (8 * i)) & 0xffu), s, c); };
    return (u32x2){pack2<BF16>(value(0), value(1)), pack2<BF16>(value(2), value(3))};
  }
  return (u32x2){pack2<BF16>(decode1<I8>(x, 0) * s, decode1<I8>(x, 1) * s),
                 pack2<BF16>(decode1<I8>(x, 2) * s, decode1<I8>(x, 3) * s)};
}

template <bool BF16, bool I8, int DK>
__global__ __launch_bounds__(256, DK == 256 ? 1 : 2) void attend8_rows_kernel(Attend8Params p) {
  constexpr int BN = kTokens8<DK>, NH = BN / 32;  // halves of 32 tokens
  constexpr int ROWB = 2 * DK, TILEB = BN * ROWB;
  constexpr int CPR = DK / 16;              // chunks of 16 codes of a row
  constexpr int RPT = BN * CPR / 256;       // rows a thread stages
  constexpr int RSTEP = 256 / CPR;
  constexpr float kUp = BF16 ? 1.f : 128.f;
  // P is 2^kStart at the running maximum and at most 2^kSlack over that: fp16 weights
  // keep their bits down to 2^-28 of the largest, as in the register form.
  constexpr float kStart = BF16 ? 0.f : 14.f, kSlack = BF16 ? 8.f : 1.5f;
  typedef typename Elem<BF16 ? MPX_BF16 : MPX_F16>::T T;
  __shared__ __align__(16) unsigned char tile[2][2][TILEB];
  struct Info {
    u32 row[BN];        // row of the pools (page * bs + slot); ~0: none
    float ks[BN], vs[BN];  // factors of the codes
    uint64_t valid;
    float kback, vref;  // what S is multiplied by; V's reference
    int pow2;           // all factors are powers of two (or 0)
  };
  __shared__ Info info[4];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i32 = lane & 31, h2 = lane >> 5;
  // Later rows see more tokens: theirs start first, of all sequences and heads. Where
  // all workgroups are resident at once, two a CU, the second of a CU are the short
  // ones, the shortest beside the longest (two prompts of 2048 tokens, 16 heads over
  // one: 62 us; 84 with one sequence after the other).
  u32 at = (blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
  const u32 wgs = gridDim.x * gridDim.y * gridDim.z, heads = (u32)p.H_kv * (u32)p.B;
  if (DK <= 128 && wgs <= 512 && at >= 256) at = wgs - 1 - (at - 256);
  const int z = at / heads, head = at - z * heads;
  const int b = head / p.H_kv, hk = head - b * p.H_kv;
  const int blk = p.blocks - 1 - z % p.blocks, part = z / p.blocks;
  const int R = p.Sq * p.G, rho0 = blk * kRows8;
  const int ctx = context8(p, b);
  const int tmax = seen8(p, ctx, b, rho0 + kRows8 - 1);
  const int tokens = part8(p, ctx, b);
  const int p0 = part * tokens, p1 = min(p0 + tokens, tmax);
  const bool alone = p.max_parts == 1 || tmax <= tokens;  // no other partition: o right away
  if (p0 >= p1 && (!alone || part > 0)) return;  // (the merge knows)

  const int rho = rho0 + 32 * wave + i32;
  const bool have = rho < R;
  const int sq = have ? rho / p.G : 0, h = hk * p.G + (have ? rho - sq * p.G : 0);
  const int pos = p.qstart || p.Sq > 1 ? start8(p, b) + sq : ctx;
  const int lim = min(p1, !have ? 0 : p.causal ? min(ctx, pos + 1) : ctx);
  const float slope = p.slopes ? p.slopes[h] * kLog2e : 0.f;
  // (a negative scale turns Q round, so that the largest score is that of the
  // largest product)
  const float c_abs = fabsf(p.c);
  const u32 turn = p.c < 0.f ? 0x80008000u : 0u;
  u32x4 qb[DK / 16];
  {
    const T* row = (const T*)p.q + b * p.qs[0] + h * p.qs[1] + sq * p.qs[2];
#pragma unroll
    for (int s = 0; s < DK / 16; ++s) {
      const int d = 16 * s + 8 * h2;
      qb[s] = have && d < p.D ? *(const u32x4*)(row + d) : (u32x4){0u, 0u, 0u, 0u};
      qb[s] ^= (u32x4){turn, turn, turn, turn};
    }
  }
  // What all rows of the wave see, and what any does.
  int least = lim, most = lim;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    least = min(least, __shfl_xor(least, off, 64));
    most = max(most, __shfl_xor(most, off, 64));
  }
  least = __builtin_amdgcn_readfirstlane(least);
  most = __builtin_amdgcn_readfirstlane(most);

  const u32 row_bytes = (u32)p.H_kv * (u32)p.D;
  const int n_tiles = p0 < p1 ? (p1 - p0 + BN - 1) / BN : 0;

  // The first wave's look-ups: lane = token of the tile.
  const int pg0 = page_of8(p, p0), base = pg0 * p.bs;
  const int32_t* const table = p.bt + (int64_t)b * p.max_blocks + pg0;
  auto page_of = [&](int t) __attribute__((always_inline)) {  // from the partition's first on
    return page_of8(p, (u32)(t - base));
  };
  auto page_id = [&](int it) __attribute__((always_inline)) {
    const int t = p0 + it * BN + lane;
    if (lane >= BN || t >= p1) return -1;
    return table[page_of(t)];
  };
  float vref = 0.f;
  auto scales = [&](int id, float& ks, float& vs) __attribute__((always_inline)) {
    const bool ok = id >= 0 && id < p.num_blocks;
    ks = ok ? p.kscale[(int64_t)id * p.H_kv + hk] : 0.f;
    vs = ok ? p.vscale[(int64_t)id * p.H_kv + hk] : 0.f;
  };
  auto write_info = [&](int it, int id, float ks, float vs) __attribute__((always_inline)) {
    const bool ok = id >= 0 && id < p.num_blocks;
    Info& f = info[it & 3];
    const int t = p0 + it * BN + lane;
    const uint64_t valid = __ballot(ok);
    float kback = c_abs;
    if constexpr (!BF16) {
      float km = ks, vm = vs;
#pragma unroll
      for (int off = 32; off >= 1; off >>= 1) {
        km = fmaxf(km, __shfl_xor(km, off, 64));
        vm = fmaxf(vm, __shfl_xor(vm, off, 64));
      }
      km = fmaxf(km, 0x1p-100f);
      vref = fmaxf(vref, fmaxf(vm, 0x1p-100f));
      kback = c_abs * km * (1.f / kUp);
      ks = ks * (kUp / km);
      vs = vs * (kUp / vref);
    }
    if (lane < BN) {
      f.row[lane] = ok ? (u32)id * (u32)p.bs + ((u32)(t - base) - page_of(t) * (u32)p.bs) : ~0u;
      f.ks[lane] = ks;
      f.vs[lane] = vs;
    }
    const bool pow2 = __all(((__float_as_uint(ks) | __float_as_uint(vs)) & 0x7fffffu) == 0);
    if (lane == 0) {
      f.pow2 = pow2;
      f.valid = valid;
      f.kback = kback;
      f.vref = BF16 ? 1.f : vref;
    }
  };

  // Codes of this thread's chunk of rows tid / CPR + j RSTEP.
  const int chunk = tid % CPR, row0 = tid / CPR;
  const bool chunk_on = 16 * chunk < p.D;
  u32x4 rk[RPT], rv[RPT];
  const u32 lane_at = (u32)(hk * p.D + 16 * chunk);
  const unsigned char* const k_lane = p.kpool + lane_at;
  const unsigned char* const v_lane = p.vpool + lane_at;
  constexpr uint64_t kAll = BN == 64 ? ~0ull : (1ull << BN) - 1;
  auto fetch = [&](int it) __attribute__((always_inline)) {
    const Info& f = info[it & 3];
    u32 row[RPT];
#pragma unroll
    for (int j = 0; j < RPT; ++j) row[j] = f.row[row0 + j * RSTEP];
    if (f.valid == kAll && p.D == DK) {
#pragma unroll
      for (int j = 0; j < RPT; ++j) {
        rk[j] = *(const u32x4*)(k_lane + (uint64_t)row[j] * row_bytes);
        rv[j] = *(const u32x4*)(v_lane + (uint64_t)row[j] * row_bytes);
      }
    } else {
#pragma unroll
      for (int j = 0; j < RPT; ++j) {
        const bool on = row[j] != ~0u && chunk_on;
        rk[j] = on ? *(const u32x4*)(k_lane + (uint64_t)row[j] * row_bytes) : (u32x4){0u, 0u, 0u, 0u};
        rv[j] = on ? *(const u32x4*)(v_lane + (uint64_t)row[j] * row_bytes) : (u32x4){0u, 0u, 0u, 0u};
      }
    }
  };
  auto place_as = [&](int it, auto pow2) __attribute__((always_inline)) {
    constexpr bool P2 = decltype(pow2)::value != 0;
    const Info& f = info[it & 3];
    unsigned char *kt = tile[it & 1][0], *vt = tile[it & 1][1];
#pragma unroll
    for (int j = 0; j < RPT; ++j) {
      const int r = row0 + j * RSTEP;
      const float ks = f.ks[r], vs = f.vs[r];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const u32x2 a = value4<I8, BF16, P2>(rk[j][2 * e], ks);
        const u32x2 c = value4<I8, BF16, P2>(rk[j][2 * e + 1], ks);
        *(u32x4*)(kt + r * ROWB + 16 * k_slot8<DK>(r, 2 * chunk + e)) = (u32x4){a[0], a[1], c[0], c[1]};
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const u32x2 a = value4<I8, BF16, P2>(rv[j][2 * e], vs);
        const u32x2 c = value4<I8, BF16, P2>(rv[j][2 * e + 1], vs);
        *(u32x4*)(vt + r * ROWB + 16 * v_slot8<DK>(r, 2 * chunk + e)) = (u32x4){a[0], a[1], c[0], c[1]};
      }
    }
  };
  auto place = [&](int it) __attribute__((always_inline)) {
    if ((I8 && BF16) || __builtin_amdgcn_readfirstlane(info[it & 3].pow2))
      place_as(it, Const<1>{});
    else
      place_as(it, Const<0>{});
  };
  auto meet = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    stage_barrier();
  };

  f32x16 o[DK / 32];
#pragma unroll
  for (int d = 0; d < DK / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  float m = -INFINITY, l = 0.f, ref = BF16 ? 1.f : 0.f;

  int id_next = -1;  // page ids of tile it + 2 (first wave)
  if (n_tiles > 0) {
    if (wave == 0) {  // (both tiles' look-ups at once)
      const int id0 = page_id(0), id1 = page_id(1);
      id_next = page_id(2);
      float ks[2], vs[2];
      scales(id0, ks[0], vs[0]);
      scales(id1, ks[1], vs[1]);
      write_info(0, id0, ks[0], vs[0]);
      write_info(1, id1, ks[1], vs[1]);
    }
    meet();
    fetch(0);
    place(0);
    meet();
  }
  for (int it = 0; it < n_tiles; ++it) {
    float ks_next = 0.f, vs_next = 0.f;
    int id_later = -1;
    if (wave == 0) {
      scales(id_next, ks_next, vs_next);
      id_later = page_id(it + 3);
    }
    if (it + 1 < n_tiles) fetch(it + 1);
    const int t0 = p0 + it * BN;
    if (t0 < most) {
      const Info& f = info[it & 3];
      const unsigned char *kt = tile[it & 1][0], *vt = tile[it & 1][1];
      f32x16 s[NH];
      const int kr = (i32 & 0x13) | ((i32 & 4) << 1) | ((i32 & 8) >> 1);
#pragma unroll
      for (int n = 0; n < NH; ++n) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[n][e] = 0.f;
#pragma unroll
        for (int c = 0; c < DK / 16; ++c) {
          const int r = 32 * n + kr;
          const u32x4 a = *(const u32x4*)(kt + r * ROWB + 16 * k_slot8<DK>(r, 2 * c + h2));
          s[n] = mfma32x32x16<BF16>(a, qb[c], s[n]);
        }
      }
      float c = BF16 ? c_abs : f.kback;
      if constexpr (!BF16) {
        const float vr = f.vref;
        if (vr != ref) {
          const float k = ref / vr;
#pragma unroll
          for (int d = 0; d < DK / 32; ++d) o[d] *= k;
          ref = vr;
        }
      }
      const uint64_t valid = f.valid;
      // Masks (and ALiBi) only where needed: the scores are then in log2 units
      // already. (The empty asm keeps their arithmetic from being done ahead of
      // the branch, for every tile.)
      if (t0 + BN > least || valid != kAll || p.slopes) {
        int shift = 8 * h2;
        asm volatile("" : "+v"(shift));
        const uint64_t mine = valid >> shift;
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int at = 32 * n + 16 * (e >> 3) + (e & 7);  // and 8 h2
            const int t = t0 + at + shift;
            float x = s[n][e] * c;
            if (p.slopes) x += slope * (float)(t - pos);
            s[n][e] = t < lim && ((mine >> at) & 1u) ? x : -INFINITY;
          }
        c = 1.f;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[n][e]);
      mx = pair_max32(mx) * c;
      // The running maximum moves where a row's grows by more than kSlack (or from
      // nothing), so that O is seldom rescaled.
      if (__any(mx > m + kSlack)) {
        const float mn = fmaxf(m, mx);
        const float k = m == -INFINITY ? 0.f : fast_exp2(m - mn);
        l *= k;
#pragma unroll
        for (int d = 0; d < DK / 32; ++d) o[d] *= k;
        m = mn;
      }
      const float sub = m == -INFINITY ? 0.f : m - kStart;
      u32x4 pb[BN / 16];
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const u32 w = pack2<BF16>(fast_exp2(__builtin_fmaf(s[n][e], c, -sub)),
                                    fast_exp2(__builtin_fmaf(s[n][e + 1], c, -sub)));
          pb[2 * n + (e >> 3)][(e & 7) >> 1] = w;
          l = dot2_sum<BF16>(w, l);
        }
      // (16 tokens after 16: the products of the first can start while the weights of
      // the others are still to come)
#pragma unroll
      for (int k = 0; k < BN / 16; ++k) {
        const int s16 = lane & 15, g = lane >> 4;
#pragma unroll
        for (int d = 0; d < DK / 32; ++d) {
          const int cc = 4 * d + 2 * (g & 1) + ((s16 & 3) >> 1);
          const int r = 16 * k + 8 * (g >> 1) + (s16 >> 2);
          const u32x2 lo = lds_read_tr16(vt + r * ROWB + 16 * v_slot8<DK>(r, cc) + 8 * (s16 & 1));
          const u32x2 hi =
              lds_read_tr16(vt + (r + 4) * ROWB + 16 * v_slot8<DK>(r + 4, cc) + 8 * (s16 & 1));
          o[d] = mfma32x32x16<BF16>((u32x4){lo[0], lo[1], hi[0], hi[1]}, pb[k], o[d]);
        }
      }
    }
    if (it + 1 < n_tiles) place(it + 1);
    if (wave == 0 && it + 2 < n_tiles) write_info(it + 2, id_next, ks_next, vs_next);
    id_next = id_later;
    meet();
  }

  l = pair_sum32(l);
  if (alone && p.o_rows16) {
    // Rows leave through the wave's part of the idle tiles, 16 bytes a lane and whole
    // rows an instruction, instead of 8-byte pieces of 32 rows (its own LDS only:
    // nothing to wait for but its own writes).
    const float inv = l == 0.f ? NAN : ref * (1.f / kUp) / l;  // (no token: 0 / 0 = NaN)
    unsigned char* const own = &tile[0][0][0] + wave * 32 * ROWB;
    static_assert(4 * 32 * ROWB <= sizeof(tile), "a wave's rows fit its part of the tiles");
    constexpr int CH = DK / 8;  // 16-byte chunks of a row
#pragma unroll
    for (int d = 0; d < DK / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int at = 32 * d + 2 * e + 4 * h2;
        const u32x2 w = {pack2<BF16>(o[d][e] * inv, o[d][e + 1] * inv),
                         pack2<BF16>(o[d][e + 2] * inv, o[d][e + 3] * inv)};
        *(u32x2*)(own + i32 * ROWB + 16 * ((at >> 3) ^ (i32 & (CH - 1))) + 2 * (at & 7)) = w;
      }
    const int64_t row = b * p.os[0] + h * p.os[1] + sq * p.os[2];
    const u32 row_lo = (u32)row, row_hi = (u32)((uint64_t)row >> 32);
    constexpr int RPI = 64 / CH;  // rows an instruction stores
#pragma unroll
    for (int k = 0; k < 32 / RPI; ++k) {
      const int r = k * RPI + lane / CH, cc = lane % CH;
      const u32x4 x = *(const u32x4*)(own + r * ROWB + 16 * (cc ^ (r & (CH - 1))));
      const uint64_t to = (uint64_t)(u32)__builtin_amdgcn_ds_bpermute(4 * r, (int)row_hi) << 32 |
                          (u32)__builtin_amdgcn_ds_bpermute(4 * r, (int)row_lo);
      if (rho0 + 32 * wave + r < R && 8 * cc < p.D) *(u32x4*)((T*)p.o + (int64_t)to + 8 * cc) = x;
    }
    return;
  }
  const int64_t part_slot = (((int64_t)b * p.H + h) * p.Sq + sq) * p.max_parts + part;
  if (!alone && have && h2 == 0) {
    p.ws_ml[2 * part_slot] = m;
    p.ws_ml[2 * part_slot + 1] = l;
  }
  if constexpr (DK <= 128) {
    if (!alone) {  // the same way for a partition's
      const float back = l == 0.f ? 0.f : ref * (1.f / kUp) / l;
      constexpr int SB = 4 * DK;  // bytes of a row of sums
      unsigned char* const own = &tile[0][0][0] + wave * 32 * SB;
      static_assert(4 * 32 * SB <= sizeof(tile), "a wave's rows fit its part of the tiles");
      constexpr int CH = DK / 4;
#pragma unroll
      for (int d = 0; d < DK / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int at = 32 * d + 2 * e + 4 * h2;
          *(f32x4*)(own + i32 * SB + 16 * ((at >> 2) ^ (i32 & (CH - 1)))) =
              (f32x4){o[d][e] * back, o[d][e + 1] * back, o[d][e + 2] * back, o[d][e + 3] * back};
        }
      const u32 lo = (u32)part_slot, hi = (u32)((uint64_t)part_slot >> 32);
      constexpr int RPI = 64 / CH;
#pragma unroll
      for (int k = 0; k < 32 / RPI; ++k) {
        const int r = k * RPI + lane / CH, cc = lane % CH;
        const f32x4 x = *(const f32x4*)(own + r * SB + 16 * (cc ^ (r & (CH - 1))));
        const uint64_t to = (uint64_t)(u32)__builtin_amdgcn_ds_bpermute(4 * r, (int)hi) << 32 |
                            (u32)__builtin_amdgcn_ds_bpermute(4 * r, (int)lo);
        if (rho0 + 32 * wave + r < R) *(f32x4*)(p.ws_o + (int64_t)to * DK + 4 * cc) = x;
      }
      return;
    }
  }
  if (!have) return;
  // This lane's dims of its row: 32 d + 8 (e / 4) + 4 h2 + e % 4.
  if (alone) {
    // (no token: 0 / 0 = NaN)
    const float inv = l == 0.f ? NAN : ref * (1.f / kUp) / l;
    T* out = (T*)p.o + b * p.os[0] + h * p.os[1] + sq * p.os[2];
#pragma unroll
    for (int d = 0; d < DK / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int at = 32 * d + 2 * e + 4 * h2;
        const float y[4] = {o[d][e] * inv, o[d][e + 1] * inv, o[d][e + 2] * inv, o[d][e + 3] * inv};
        if (at < p.D) store_row8<4>(out + at, y, p.o_rows16);
      }
  } else {
    const float back = l == 0.f ? 0.f : ref * (1.f / kUp) / l;
    float* out = p.ws_o + part_slot * DK + 4 * h2;
#pragma unroll
    for (int d = 0; d < DK / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *(f32x4*)(out + 32 * d + 2 * e) = (f32x4){o[d][e] * back, o[d][e + 1] * back,
                                                  o[d][e + 2] * back, o[d][e + 3] * back};
  }
}

// Joins the partitions of a row, which are o / l each: weights l 2^(m - M) over the largest
// maximum. A chain of latencies: 3.2 us for 128 rows of six partitions, 7.7 for 4160 of
// ten (22 MB). WAVES (1 or 4) waves a row, which take eight partitions at a time in turn:
// one round trip to memory joins 8 or 32.
template <int QT, int WAVES>
__global__ __launch_bounds__(256) void attend8_merge_kernel(Attend8Params p, int DK) {
  typedef typename Elem<QT>::T T;
  __shared__ __align__(16) float s_acc[WAVES == 1 ? 1 : 3][64][4];
  __shared__ float s_m[4], s_l[4];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t rows = (int64_t)p.B * p.H * p.Sq;
  const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * 4 + wave : (int64_t)blockIdx.x;
  if (row >= rows) return;
  int sq, h, b;
  if (rows < (1ll << 32)) {  // (a division of 64 bits takes some hundred instructions)
    const u32 bh = (u32)row / (u32)p.Sq;
    sq = (int)((u32)row - bh * (u32)p.Sq);
    b = (int)(bh / (u32)p.H);
    h = (int)(bh - (u32)b * (u32)p.H);
  } else {
    const int64_t bh = row / p.Sq;
    sq = (int)(row - bh * p.Sq);
    b = (int)(bh / p.H);
    h = (int)(bh - (int64_t)b * p.H);
  }
  const int rho = sq * p.G + h % p.G;
  const float* ml = p.ws_ml + 2 * row * p.max_parts;
  const float* wo = p.ws_o + row * p.max_parts * DK + 4 * lane;
  float M = -INFINITY, L = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const bool on = 4 * lane < DK;
  // Eight partitions at a time, asked for before the context (and with it how
  // many were written) is known; what was not written is left out below.
  const int first = WAVES == 1 ? 0 : 8 * wave;
  int n = p.max_parts;
  bool alone = false;  // one partition or no token: o is there
  auto written = [&]() __attribute__((always_inline)) {
    const int ctx = context8(p, b);
    const int tmax = seen8(p, ctx, b, rho / p.span * p.span + p.span - 1);
    const int tokens = part8(p, ctx, b);
    alone = tmax <= tokens;
    n = (tmax + tokens - 1) / tokens;
  };
  if (WAVES == 1 && rows > 16384) {  // (the loads themselves count there)
    written();
    if (alone) return;
  }
  for (int i0 = first; i0 < n; i0 += 8 * WAVES) {
    const int have = min(8, p.max_parts - i0);
    float2 mli = make_float2(-INFINITY, 0.f);
    if (lane < have) mli = *(const float2*)(ml + 2 * (i0 + lane));
    f32x4 ov[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      ov[u] = u < have && on ? *(const f32x4*)(wo + (int64_t)(i0 + u) * DK)
                             : (f32x4){0.f, 0.f, 0.f, 0.f};
    if (i0 == first) {
      written();
      if (alone) break;
    }
    const int c = n - i0;
    const float mi = lane < min(c, 8) ? mli.x : -INFINITY, li = mli.y;
    float mn = mi;
#pragma unroll
    for (int off = 4; off >= 1; off >>= 1) mn = fmaxf(mn, __shfl_xor(mn, off, 64));
    mn = fmaxf(M, __shfl(mn, 0, 64));
    const float keep = M == -INFINITY ? 0.f : fast_exp2(M - mn);
    acc *= keep;
    L *= keep;
    M = mn;
    const float w = mi == -INFINITY ? 0.f : fast_exp2(mi - M);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (u >= c) break;
      const float wu = __shfl(w * li, u, 64);
      L += wu;
      acc += wu * ov[u];
    }
  }
  if constexpr (WAVES == 1) {
    if (alone) return;
  } else {
    if (lane == 0) {
      s_m[wave] = M;
      s_l[wave] = L;
    }
    if (wave > 0) *(f32x4*)s_acc[wave - 1][lane] = acc;
    __syncthreads();
    if (wave > 0 || alone) return;
    const float most = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    const float keep = M == -INFINITY ? 0.f : fast_exp2(M - most);
    L *= keep;
    acc *= keep;
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      const float f = s_m[w] == -INFINITY ? 0.f : fast_exp2(s_m[w] - most);
      L = fmaf(f, s_l[w], L);
      acc += f * *(const f32x4*)s_acc[w - 1][lane];
    }
  }
  if (4 * lane >= p.D) return;
  T* out = (T*)p.o + b * p.os[0] + h * p.os[1] + sq * p.os[2] + 4 * lane;
  const float y[4] = {acc[0] / L, acc[1] / L, acc[2] / L, acc[3] / L};  // no token: 0 / 0 = NaN
  store_row8<4>(out, y, p.o_rows16);
}

namespace {

// magic = ceil(2^(32 + shift) / bs) with the largest shift whose magic fits 32 bits: over by
// less than bs <= 2^(shift + 1) in 2^(32 + shift), which n < 2^31 does not make a whole one of.
// (A power of two divides exactly.)
void page_magic8(int bs, u32& magic, u32& shift) {
  shift = 0;
  while ((2ll << shift) < bs) ++shift;
  magic = (u32)(((1ull << (32 + shift)) + bs - 1) / bs);
}

int kernel_dim8(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

struct Plan8 {
  int span, blocks, part, max_parts, step, wave_heads;
};

constexpr int64_t kMostSums8 = 256ll << 20;  // bytes of partitions' sums of a call

// Partitions of the rows form, from a model of its time in microseconds (fitted to
// 100 measured pairs of shapes and partitions at head dim 128, which it meets within
// 20%): a tile of 64 tokens takes a workgroup 1.65 alone on its CU and 2.45 with
// another (512 workgroups are resident), 1.15 of a CU's time where the chip is full,
// with half of the last partition behind (one a CU and twice the times at D 256); a start
// 4.5; the merge 4.5 more and each partition's sums a write and a read at 5 TB/s. Sequences
// share no partition, so a batch of prompts takes one each, 65 queries behind 4100 tokens
// (two sequences) ten of 448: 37.7 us, against 42.4 with 16 of 256 and 43.5 with seven of 640.
int64_t rows_parts8(int64_t groups, int64_t rows, int64_t tokens, int DK) {
  const double tile = DK / 128.0;
  const int64_t resident = DK <= 128 ? 512 : 256;
  if (groups >= 2 * resident) return 1;  // (empty partitions would cost more than a tail)
  double best = 0.0;
  int64_t parts = 0;
  for (int64_t n = 1; n <= 64; ++n) {
    const int64_t tiles = (tokens + 64 * n - 1) / (64 * n);
    if (n > 1 && tiles < 2) break;
    const int64_t wgs = groups * n;
    double t = tiles * tile * (wgs <= 256 || DK > 128 ? 1.65 : 2.45);
    if (wgs > resident)
      t = std::max(t, groups * ((tokens + 63) / 64) * tile * 1.15 / 256.0 + 0.5 * t);
    if (n > 1) t += 4.5 + (double)rows * n * DK * 8.0 / 5e6;
    if (parts == 0 || t < best) {
      best = t;
      parts = n;
    }
  }
  return parts;
}

// Rows of a block: 16 or 32 in the register form (16 for float32, whose operands
// take the registers, and for head dims above 128), 128 above; and the partitions of the
// tokens. Tokens are those that a row may see as far as the host knows: the table's width, or
// for causal rows at positions of their own (from 0) the queries' number. The table may be far
// wider than what is in it, so a plan is for both: as many partitions as the width asks for,
// within kMostSums8, and as short as `near` tokens ask for; longer sequences spread over all of
// them (part8). Two turns of 65 queries behind 4100 tokens: 38 us in tables of 4144 tokens, 39 in
// tables of 32768 and of 131072 (138 and 169 with the partitions that 32768 and 131072 tokens
// get); decode of 16 sequences of 301 to 4100: 23.6, 26.6, 26.6 (34 and 98).
Plan8 plan8(int B, int Sq, int H, int H_kv, int D, int block_size, int max_blocks, int dtype,
            bool causal, bool positions) {
  Plan8 s;
  const int64_t R = (int64_t)Sq * (H / H_kv);
  s.span = dtype == MPX_F32 || R <= 16 ? 16 : R <= 32 && D <= 128 ? 32 : kRows8;
  s.blocks = (int)((R + s.span - 1) / s.span);
  int64_t width = std::max<int64_t>(1, (int64_t)max_blocks * block_size);
  if (causal && !positions && Sq > 1) width = std::min<int64_t>(width, Sq);
  const int64_t groups = (int64_t)B * H_kv * s.blocks;
  const int64_t room =
      std::max<int64_t>(1, kMostSums8 / ((int64_t)B * H * Sq * (kernel_dim8(D) + 2) * 4));
  // parts(tokens): how many partitions that many tokens ask for.
  auto plan = [&](auto parts, int64_t near, int64_t step) {
    const int64_t n = std::min(parts(width), room);
    auto each = [&](int64_t tokens, int64_t k) {
      return ((tokens + k - 1) / k + step - 1) / step * step;
    };
    int64_t part = each(width, n);
    if (n > 1 && width > near + near / 4) part = std::min(part, each(near, parts(near)));
    s.part = (int)part;
    s.max_parts = (int)std::min(n, (width + part - 1) / part);
    s.step = (int)step;
  };
  s.wave_heads = 0;
  if (s.span == kRows8) {
    const int64_t rows = (int64_t)B * H * Sq;
    plan([&](int64_t tokens) { return rows_parts8(groups, rows, tokens, kernel_dim8(D)); }, 4096,
         64);
    return s;
  }
  // The waves of the register form take four heads of the same tokens, whose rows
  // are neighbours in memory, where partitions of 512 tokens fill the chip that
  // way (8 workgroups for each of 256 CUs); else a share of one head's tokens each.
  // Only for few rows: the sums of a partition's rows go through memory. 64 decode
  // rows over 512 to 8192 tokens, 32 heads: 420 us, 433 with partitions of 1024 and
  // 428 of 256; with shares of one head 467 to 510.
  // (A table may be wider than what is in it: 16384 of its tokens count. Eight sequences of 4096
  // tokens, 32 heads over 8, in tables of 131072: 21 us, 33 with waves that take heads.)
  const int64_t p512 = (std::min<int64_t>(width, 16384) + 511) / 512;
  if (R <= 32 && H_kv % 4 == 0 && groups / 4 * p512 >= 2048) {
    s.wave_heads = 1;
    plan([&](int64_t tokens) { return std::min<int64_t>((tokens + 511) / 512, 64); }, 2048, 512);
    return s;
  }
  // As many partitions as give each CU a workgroup, none above 1024 tokens where rows are
  // few (contexts differ: the long ones have to spread; up to 64 partitions) or under 256
  // (128 of float32, whose products take longer); one where there are no more than 512 tokens
  // for 16-bit queries.
  // 32 heads over 8 of D 128, bf16, us: one sequence of 512 tokens 8.3 (two
  // partitions 9.5), 8192 tokens 10.2 (of 1024: 13.5), 32768 19.6 (of 512: 21.5, of
  // 4096: 31.7); four of 8192 19.0 (of 512: 20.3); 40 of 586 to 8192 102 (of 2048:
  // 117, of 4096 123).
  const bool wide = dtype != MPX_F32;
  const int64_t least = wide ? 256 : 128;
  plan([&](int64_t tokens) {
    if (wide && tokens <= 512) return (int64_t)1;
    int64_t n = std::min(std::max<int64_t>(1, 256 / groups), (tokens + least - 1) / least);
    // (16 sequences of 301 to 4100 in tables of 131072: 26 us with room for 32, 33 for 64)
    const int64_t most = std::min<int64_t>(64, std::max<int64_t>(32, 4096 / groups));
    if (R <= 32) n = std::max(n, std::min((tokens + 1023) / 1024, most));
    return n;
  }, 2048, 128);
  return s;
}

// Sizes that the grid has room for: 2^32 threads in x, 65535 workgroups in z.
bool grid_fits8(int B, int Sq, int H, int H_kv, int dtype) {
  const int64_t R = (int64_t)Sq * (H / H_kv);
  const int64_t blocks = (R + 15) / 16;  // (those of the least rows)
  return B <= 65535 && (dtype == MPX_F32 || R <= 32 ? blocks : (R + kRows8 - 1) / kRows8) * H_kv <
                           (1 << 24);
}

size_t ws_bytes8(int B, int Sq, int H, int D, const Plan8& s) {
  if (s.max_parts == 1) return 0;
  return (size_t)B * H * Sq * s.max_parts * (kernel_dim8(D) + 2) * sizeof(float);
}

template <int QT, bool I8, int DK, int NR>
void launch_attend_pages(const Attend8Params& p, dim3 grid, hipStream_t st) {
  if (p.bs % 8 == 0)
    hipLaunchKernelGGL((attend8_kernel<QT, I8, DK, NR, true>), grid, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((attend8_kernel<QT, I8, DK, NR, false>), grid, dim3(256), 0, st, p);
}
template <int QT, bool I8, int DK>
void launch_attend_nr(const Attend8Params& p, dim3 grid, hipStream_t st) {
  if constexpr (QT != MPX_F32) {
    if (p.span == kRows8) {
      hipLaunchKernelGGL((attend8_rows_kernel<QT == MPX_BF16, I8, DK>), grid, dim3(256), 0, st, p);
      return;
    }
    if constexpr (DK <= 128) {
      if (p.span == 32) {
        launch_attend_pages<QT, I8, DK, 2>(p, grid, st);
        return;
      }
    }
  }
  launch_attend_pages<QT, I8, DK, 1>(p, grid, st);
}
template <int QT, bool I8>
hipError_t launch_attend(const Attend8Params& p, hipStream_t st) {
  const dim3 grid((p.wave_heads ? p.H_kv / 4 : p.H_kv) * p.blocks, p.max_parts, p.B);
  const int dk = kernel_dim8(p.D);
  if (dk == 64) launch_attend_nr<QT, I8, 64>(p, grid, st);
  else if (dk == 128) launch_attend_nr<QT, I8, 128>(p, grid, st);
  else launch_attend_nr<QT, I8, 256>(p, grid, st);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.max_parts == 1) return e;
  const int64_t rows = (int64_t)p.B * p.H * p.Sq;
  // (four waves a row where the rows alone leave the chip idle: 17 partitions of 32 rows 10.2 us
  // instead of 12.4 in all; for 4160 rows of ten 40.7 instead of 37.7)
  if (p.max_parts > 8 && rows <= 1024)
    hipLaunchKernelGGL((attend8_merge_kernel<QT, 4>), dim3((unsigned)rows), dim3(256), 0, st, p,
                       dk);
  else
    hipLaunchKernelGGL((attend8_merge_kernel<QT, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0,
                       st, p, dk);
  return hipGetLastError();
}
template <int QT>
hipError_t launch_attend_code(const Attend8Params& p, int code, hipStream_t st) {
  return code == MPX8_INT8 ? launch_attend<QT, true>(p, st) : launch_attend<QT, false>(p, st);
}

}  // namespace
}  // namespace mpx

using namespace mpx;

extern "C" size_t mpx_paged_attend8_call_workspace_bytes(int B, int Sq, int H, int H_kv, int D,
                                                         int block_size, int max_blocks, int dtype,
                                                         int causal, int positions) {
  if (B <= 0 || Sq <= 0 || H <= 0 || H_kv <= 0 || H % H_kv != 0 || D <= 0 || block_size <= 0 ||
      max_blocks < 0 || !grid_fits8(B, Sq, H, H_kv, dtype))
    return 0;
  return ws_bytes8(B, Sq, H, D, plan8(B, Sq, H, H_kv, D, block_size, max_blocks, dtype,
                                      causal != 0, positions != 0));
}

extern "C" size_t mpx_paged_attend8_workspace_bytes(int B, int Sq, int H, int H_kv, int D,
                                                    int block_size, int max_blocks, int dtype) {
  if (B <= 0 || Sq <= 0 || H <= 0 || H_kv <= 0 || H % H_kv != 0 || D <= 0 || block_size <= 0 ||
      max_blocks < 0 || !grid_fits8(B, Sq, H, H_kv, dtype))
    return 0;
  // (as much as any causal and query_start ask for)
  return std::max(ws_bytes8(B, Sq, H, D, plan8(B, Sq, H, H_kv, D, block_size, max_blocks, dtype,
                                               false, false)),
                  mpx_paged_attend8_call_workspace_bytes(B, Sq, H, H_kv, D, block_size, max_blocks,
                                                         dtype, 1, 0));
}

extern "C" int mpx_paged_attend8(const void* q, const void* k_pool, const void* v_pool,
                                 const float* k_scales, const float* v_scales,
                                 const int32_t* block_tables, const int32_t* context_lens,
                                 const int32_t* query_start, const float* alibi_slopes, void* o,
                                 const int64_t* q_strides, const int64_t* o_strides, int B, int Sq,
                                 int H, int H_kv, int D, int num_blocks, int block_size,
                                 int max_blocks, float scale, int causal, int dtype, int code,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  const char* fn = "mpx_paged_attend8";
  MPX_CHECK_ARG(dtype == MPX_F32 || dtype == MPX_F16 || dtype == MPX_BF16,
                "%s: unknown dtype code %d", fn, dtype);
  MPX_CHECK_ARG(code == MPX8_E4M3 || code == MPX8_INT8, "%s: unknown code format %d", fn, code);
  MPX_CHECK_ARG(B >= 0 && Sq >= 0 && H >= 0 && num_blocks >= 0 && max_blocks >= 0,
                "%s: negative size", fn);
  MPX_CHECK_ARG(H_kv > 0 ? H % H_kv == 0 : H == 0,
                "%s: %d query heads are not a multiple of %d K/V heads", fn, H, H_kv);
  MPX_CHECK_ARG(block_size > 0 && block_size <= MPX8_MAX_BLOCK_SIZE,
                "%s: block_size must be in 1..%d", fn, MPX8_MAX_BLOCK_SIZE);
  if (D <= 0 || D > 256 || D % 16 != 0) {
    set_error("%s: head_dim %d not supported (a multiple of 16 up to 256)", fn, D);
    return MPX_EUNSUPPORTED;
  }
  MPX_CHECK_ARG(std::isfinite(scale), "%s: scale must be finite", fn);
  if ((int64_t)B * Sq * H == 0) return MPX_OK;
  MPX_CHECK_ARG(q && o && context_lens && q_strides && o_strides, "%s: null pointer argument", fn);
  MPX_CHECK_ARG(max_blocks == 0 || num_blocks == 0 ||
                    (k_pool && v_pool && k_scales && v_scales && block_tables),
                "%s: null pool, scale or table pointer", fn);
  const int vec = dtype == MPX_F32 ? 4 : 8;
  MPX_CHECK_ARG(((uintptr_t)q & 15u) == 0 && ((uintptr_t)k_pool & 15u) == 0 &&
                    ((uintptr_t)v_pool & 15u) == 0 && q_strides[0] % vec == 0 &&
                    q_strides[1] % vec == 0 && q_strides[2] % vec == 0,
                "%s: q (and its strides) and the pools must be 16-byte aligned", fn);
  MPX_CHECK_ARG((int64_t)max_blocks * block_size < (1LL << 30), "%s: block table too large", fn);
  MPX_CHECK_ARG((int64_t)H_kv * D < (1 << 24), "%s: head count too large", fn);
  MPX_CHECK_ARG((int64_t)Sq * H < (1LL << 30), "%s: too many queries in one call", fn);
  MPX_CHECK_ARG((int64_t)num_blocks * block_size < (1LL << 32) - 1, "%s: too many pages", fn);
  MPX_CHECK_ARG(grid_fits8(B, Sq, H, H_kv, dtype), "%s: grid too large", fn);
  Attend8Params p;
  const Plan8 s = plan8(B, Sq, H, H_kv, D, block_size, num_blocks ? max_blocks : 0, dtype,
                        causal != 0, query_start != nullptr);
  const size_t need = ws_bytes8(B, Sq, H, D, s);
  MPX_CHECK_ARG(need == 0 || (workspace && ((uintptr_t)workspace & 15u) == 0 &&
                              workspace_bytes >= need),
                "%s: 16-byte aligned workspace of %zu bytes required, %zu given", fn, need,
                workspace_bytes);
  p.q = q; p.kpool = (const unsigned char*)k_pool; p.vpool = (const unsigned char*)v_pool;
  p.kscale = k_scales; p.vscale = v_scales; p.bt = block_tables; p.cl = context_lens;
  p.qstart = query_start; p.slopes = alibi_slopes; p.o = o;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = q_strides[i];
    p.os[i] = o_strides[i];
  }
  p.o_rows16 = ((uintptr_t)o & 15u) == 0 && o_strides[0] % vec == 0 && o_strides[1] % vec == 0 &&
               o_strides[2] % vec == 0;
  p.B = B; p.Sq = Sq; p.H = H; p.H_kv = H_kv; p.G = H / H_kv; p.D = D;
  p.num_blocks = num_blocks; p.bs = block_size; p.max_blocks = num_blocks ? max_blocks : 0;
  // one query without a position of its own sees its whole context
  p.causal = causal && (query_start || Sq > 1);
  p.part = s.part; p.max_parts = s.max_parts; p.reach = s.part * s.max_parts; p.step = s.step;
  p.blocks = s.blocks; p.span = s.span; p.wave_heads = s.wave_heads;
  page_magic8(block_size, p.magic, p.shift);
  p.c = scale * kLog2e;
  p.ws_o = (float*)workspace;
  p.ws_ml = (float*)workspace + (size_t)B * H * Sq * s.max_parts * kernel_dim8(D);
  hipStream_t st = (hipStream_t)stream;
  hipError_t e;
  if (dtype == MPX_F32) e = launch_attend_code<MPX_F32>(p, code, st);
  else if (dtype == MPX_F16) e = launch_attend_code<MPX_F16>(p, code, st);
  else e = launch_attend_code<MPX_BF16>(p, code, st);
  MPX_CHECK_HIP(e);
  return MPX_OK;
}
