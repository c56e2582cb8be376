// RMS norm of queries and keys for each head with the rotary rotation in the
// same pass, and its gradient, for gfx950.
//
// With x a head row of D values, w the weight, c and s the row's half tables:
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w,
//   y1 = n1 c - n2 s,  y2 = n1 s + n2 c                      (halves 1 and 2)
// and for a gradient dy, turned back (the rotation is orthogonal):
//   g1 = dy1 c + dy2 s,  g2 = dy2 c - dy1 s,
//   dw = sum over rows of g x r,   dx = r (g w - x r^2 mean(g w x)).
// Everything in float32, each result rounded once.
//
// Memory bound (8 to 24 operations an element of 2 or 4 bytes). A row is held
// by LPR lanes, 8 pairs each (dims [8c, 8c + 8) of both halves, so that a
// rotation stays in its lane): the sums of a row are LPR-lane shuffles and
// nothing goes through LDS. A wave takes 64 / LPR heads of one token at a time,
// whose rows are neighbours in memory, and keeps the token's table rows in
// registers for all of them.
//
// Measured (a large copy runs at 4.91 TB/s on the same card): 4 x 4096 tokens of 32 + 8
// heads of D 128 in bf16, forward 61 us (5.5 TB/s), backward 109 us (4.6 TB/s) and 4.9 us for
// the sum of dw's parts: 173 us in all, 840 MB at 4.86 TB/s. One token of 24 sequences: 4.0 us,
// a launch and one chain of loads.
#include "mpx_rows.h"

#include <algorithm>
#include <cmath>

#include "mpx_norm.h"

namespace mpx {

struct NormParams {
  const void *q, *k, *wq, *wk, *cos, *sin;
  void *oq, *ok;              // y; for the gradient dq, dk
  const void *gq, *gk;        // gradient: dy of q and k
  float* ws;                  // gradient: (workgroups, 2, D) partial sums of dw
  int64_t qs[3], ks[3];       // (batch, seq, head) element strides
  int64_t gqs[3], gks[3];
  const int32_t* pos;
  int32_t* err;
  int B, S, H, H_kv, D, offset, n_pos, wdt;
  int tokens, parts, per;     // waves a token, head iterations of each
  float eps;
};

// Eight elements of a type that is only known at run time, as float32.
__device__ __forceinline__ void load8f(const void* p, int64_t at, int dt, float* out) {
  if (dt == MPX_F32) {
    R8<float> v;
    v.load((const float*)p + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = v.get(e);
  } else if (dt == MPX_F16) {
    R8<_Float16> v;
    v.load((const _Float16*)p + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = v.get(e);
  } else {
    R8<__bf16> v;
    v.load((const __bf16*)p + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = v.get(e);
  }
}

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int off = LPR / 2; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// One lane's 16 values of a row: the chunk of the first half and of the second.
template <typename T>
struct Halves {
  R8<T> a, b;
};
template <typename T>
__device__ __forceinline__ Halves<T> load_halves(const T* row, int d, int half, bool on) {
  Halves<T> r;
  r.a.clear();
  r.b.clear();
  if (on) {
    r.a.load(row + d);
    r.b.load(row + half + d);
  }
  return r;
}

// What a wave works on: part `part` of token `tok`, heads in iterations of RPW
// rows, those of q first.
template <typename C>
struct Token {
  int64_t at;       // token's index, b * S + s
  int b, s;
  bool in;          // its position has a table row
  R8<C> cos, sin;
  __device__ __forceinline__ void place(const NormParams& p, int tok) {
    at = tok;
    b = tok / p.S;
    s = tok - b * p.S;
  }
  __device__ __forceinline__ void read(const NormParams& p, int d, bool on) {
    const int64_t pos = (int64_t)(p.pos ? p.pos[b] : p.offset) + s;
    in = pos >= 0 && pos < p.n_pos;
    cos.clear();
    sin.clear();
    if (in && on) {
      const int64_t base = pos * (p.D / 2) + d;
      cos.load((const C*)p.cos + base);
      sin.load((const C*)p.sin + base);
    }
  }
};

// The error word, by a workgroup of its own: whether a row's position has no
// table row (a word that is only ever set would have to be cleared by a launch
// before).
__device__ void norm_error(const NormParams& p) {
  int bad = 0;
  for (int b = threadIdx.x; b < p.B; b += 256)
    bad |= p.pos[b] < 0 || (int64_t)p.pos[b] + p.S > p.n_pos;
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) p.err[0] = bad ? 1 : 0;
}

template <int XT, int CT, int LPR>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(NormParams p) {
  typedef typename Elem<XT>::T T;
  typedef typename Elem<CT>::T C;
  constexpr int RPW = 64 / LPR;
  const u32 wg = blockIdx.y * gridDim.x + blockIdx.x;
  if (p.pos && wg == gridDim.x * gridDim.y - 1) {
    norm_error(p);
    return;
  }
  const int lane = threadIdx.x & 63;
  const u32 item = wg * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const u32 token = item / (u32)p.parts;
  if (token >= (u32)p.tokens) return;
  const int tok = (int)token, part = (int)(item - token * (u32)p.parts);
  const int grp = lane / LPR, d = (lane % LPR) * 8, half = p.D / 2;
  const bool on = d < half;
  const int nq = (p.H + RPW - 1) / RPW, n_it = nq + (p.H_kv + RPW - 1) / RPW;
  const int first = part * p.per, last = min(first + p.per, n_it);

  auto row_of = [&](int it, const T*& x, T*& y, const Token<C>& t) __attribute__((always_inline)) {
    const bool isq = it < nq;
    const int h = (isq ? it : it - nq) * RPW + grp, n = isq ? p.H : p.H_kv;
    const int64_t* st = isq ? p.qs : p.ks;
    x = (const T*)(isq ? p.q : p.k) + t.b * st[0] + t.s * st[1] + h * st[2];
    y = (T*)(isq ? p.oq : p.ok) + (t.at * n + h) * p.D;
    return on && h < n;
  };
  Token<C> t;
  t.place(p, tok);
  const T* x;
  T* to;
  bool live = row_of(first, x, to, t);
  Halves<T> next = load_halves(x, d, half, live);
  t.read(p, d, on);
  float w[16];
  int have = -1;
  for (int it = first; it < last; ++it) {
    const Halves<T> cur = next;
    T* const out = to;
    const bool mine = live;
    if (it + 1 < last) {
      live = row_of(it + 1, x, to, t);
      next = load_halves(x, d, half, live);
    }
    if ((it < nq) != have) {
      have = it < nq;
      const void* wp = have ? p.wq : p.wk;
      if (on) {
        load8f(wp, d, p.wdt, w);
        load8f(wp, half + d, p.wdt, w + 8);
      }
    }
    float sq = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = cur.a.get(e), b = cur.b.get(e);
      sq = fmaf(a, a, sq);
      sq = fmaf(b, b, sq);
    }
    const float r = 1.0f / sqrtf(row_sum<LPR>(sq) / (float)p.D + p.eps);
    if (!mine) continue;
    float y1[8], y2[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      rope_pair(cur.a.get(e) * r * w[e], cur.b.get(e) * r * w[8 + e], t.cos.get(e), t.sin.get(e),
                y1[e], y2[e]);
      y1[e] = t.in ? y1[e] : 0.f;
      y2[e] = t.in ? y2[e] : 0.f;
    }
    Halves<T> y;
    y.a.set(y1);
    y.b.set(y2);
    y.a.store(out + d);
    y.b.store(out + half + d);
  }
}

// The gradient: the same walk over the rows, by as many workgroups as fill the
// chip, each of which keeps its sums of dw in registers until its end and
// leaves them in its slot of the workspace.
template <int XT, int CT, int LPR>
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_kernel(NormParams p) {
  typedef typename Elem<XT>::T T;
  typedef typename Elem<CT>::T C;
  constexpr int RPW = 64 / LPR;
  __shared__ float sums[4][2][256];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = lane / LPR, d = (lane % LPR) * 8, half = p.D / 2;
  const bool on = d < half;
  const int nq = (p.H + RPW - 1) / RPW, n_it = nq + (p.H_kv + RPW - 1) / RPW;
  const int64_t items = (int64_t)p.tokens * p.parts;
  float wv[2][16], dw[2][16];
#pragma unroll
  for (int e = 0; e < 16; ++e) wv[0][e] = wv[1][e] = dw[0][e] = dw[1][e] = 0.f;
  if (on) {
    load8f(p.wq, d, p.wdt, wv[0]);
    load8f(p.wq, half + d, p.wdt, wv[0] + 8);
    load8f(p.wk, d, p.wdt, wv[1]);
    load8f(p.wk, half + d, p.wdt, wv[1] + 8);
  }
  for (int64_t item = (int64_t)blockIdx.x * 4 + wave; item < items; item += (int64_t)gridDim.x * 4) {
    const int tok = (int)(item / p.parts), part = (int)(item - (int64_t)tok * p.parts);
    Token<C> t;
    t.place(p, tok);
    t.read(p, d, on);
    const int first = part * p.per, last = min(first + p.per, n_it);
    auto rows = [&](auto which, int lo, int hi) __attribute__((always_inline)) {
      constexpr int K = decltype(which)::value;  // 0: q, 1: k
      const int n = K ? p.H_kv : p.H;
      const int64_t* xs = K ? p.ks : p.qs;
      const int64_t* gs = K ? p.gks : p.gqs;
      const T* xb = (const T*)(K ? p.k : p.q) + t.b * xs[0] + t.s * xs[1];
      const T* gb = (const T*)(K ? p.gk : p.gq) + t.b * gs[0] + t.s * gs[1];
      T* ob = (T*)(K ? p.ok : p.oq) + t.at * n * p.D;
      if (lo >= hi) return;
      // (the next rows are on their way while one is worked on)
      auto row = [&](int it, Halves<T>& x, Halves<T>& g) __attribute__((always_inline)) {
        const int h = it * RPW + grp;
        const bool read = on && h < n && t.in;
        x = load_halves(xb + h * xs[2], d, half, read);
        g = load_halves(gb + h * gs[2], d, half, read);
      };
      Halves<T> nx, ng;
      row(lo, nx, ng);
      for (int it = lo; it < hi; ++it) {
        const int h = it * RPW + grp;
        const bool live = on && h < n;
        const Halves<T> x = nx, g = ng;
        if (it + 1 < hi) row(it + 1, nx, ng);
        float gr[16], sq = 0.f, gwx = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = x.a.get(e), b = x.b.get(e);
          rope_pair(g.a.get(e), g.b.get(e), t.cos.get(e), -t.sin.get(e), gr[e], gr[8 + e]);
          sq = fmaf(a, a, sq);
          sq = fmaf(b, b, sq);
          gwx = fmaf(gr[e] * wv[K][e], a, gwx);
          gwx = fmaf(gr[8 + e] * wv[K][8 + e], b, gwx);
        }
        // (nothing from lanes without a row, whose 1 / sqrt(eps) is infinite for eps = 0)
        const float rms = sqrtf(row_sum<LPR>(sq) / (float)p.D + p.eps);
        const float r = h < n && t.in ? 1.0f / rms : 0.f;
        const float m = row_sum<LPR>(gwx) / (float)p.D * r * r;
        float y1[8], y2[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = x.a.get(e), b = x.b.get(e);
          dw[K][e] = fmaf(gr[e] * r, a, dw[K][e]);
          dw[K][8 + e] = fmaf(gr[8 + e] * r, b, dw[K][8 + e]);
          y1[e] = r * fmaf(-a, m, gr[e] * wv[K][e]);
          y2[e] = r * fmaf(-b, m, gr[8 + e] * wv[K][8 + e]);
          y1[e] = t.in ? y1[e] : 0.f;  // (also where a weight is not finite)
          y2[e] = t.in ? y2[e] : 0.f;
        }
        if (live) {
          Halves<T> y;
          y.a.set(y1);
          y.b.set(y2);
          y.a.store(ob + (int64_t)h * p.D + d);
          y.b.store(ob + (int64_t)h * p.D + half + d);
        }
      }
    };
    rows(Const<0>{}, first, min(last, nq));
    rows(Const<1>{}, max(first, nq) - nq, last - nq);
  }
  // Row groups of the wave, then the waves, in a fixed order.
#pragma unroll
  for (int K = 0; K < 2; ++K)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float x = dw[K][e];
#pragma unroll
      for (int off = 32; off >= LPR; off >>= 1) x += __shfl_xor(x, off, 64);
      if (grp == 0 && on) sums[wave][K][(e >> 3) * half + d + (e & 7)] = x;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.D; i += 256) {
    const int K = i >= p.D, j = i - K * p.D;
    p.ws[(int64_t)blockIdx.x * 2 * p.D + i] =
        ((sums[0][K][j] + sums[1][K][j]) + sums[2][K][j]) + sums[3][K][j];
  }
}

// dw[j] = sum over the workgroups' slots: 16 columns a workgroup, 16 threads
// each, whose sums are added in order.
template <typename W>
__device__ __forceinline__ void store_dw(void* q, void* k, int D, int i, float v) {
  W* out = (W*)(i < D ? q : k);
  out[i < D ? i : i - D] = from_f<W>(v);
}
__global__ __launch_bounds__(256) void qk_norm_dw_kernel(const float* ws, void* dwq, void* dwk,
                                                         int D, int n, int wdt) {
  __shared__ float part[16][17];
  const int col = threadIdx.x & 15, row = threadIdx.x >> 4;
  const int i = blockIdx.x * 16 + col;  // (2 D is a multiple of 16)
  float s = 0.f;
#pragma unroll 8
  for (int j = row; j < n; j += 16) s += ws[(int64_t)j * 2 * D + i];
  part[row][col] = s;
  __syncthreads();
  if (row != 0) return;
#pragma unroll
  for (int j = 1; j < 16; ++j) s += part[j][col];
  if (wdt == MPX_F32)
    store_dw<float>(dwq, dwk, D, i, s);
  else if (wdt == MPX_F16)
    store_dw<_Float16>(dwq, dwk, D, i, s);
  else
    store_dw<__bf16>(dwq, dwk, D, i, s);
}

namespace {

int lanes_per_row(int D) {
  int n = 1;
  while (n * 16 < D) n *= 2;
  return n;
}

// Workgroups of the gradient: two for each of 256 CUs, fewer where the tokens
// do not fill them (each leaves 2 D floats that the last launch has to sum).
int bwd_groups(int64_t waves) { return (int)std::min<int64_t>((waves + 3) / 4, 512); }

// Parts that a token's heads are cut into: one (its tables are read once) where
// the tokens alone give 4096 waves, else up to one for each head iteration.
void cut(NormParams& p) {
  const int rpw = 64 / lanes_per_row(p.D);
  const int n_it = (p.H + rpw - 1) / rpw + (p.H_kv + rpw - 1) / rpw;
  const int want = (int)std::max<int64_t>(1, std::min<int64_t>(n_it, 4096 / std::max(1, p.tokens)));
  p.per = (n_it + want - 1) / want;
  p.parts = (n_it + p.per - 1) / p.per;
}

template <int XT, int CT, int LPR>
hipError_t launch_one(const NormParams& p, bool bwd, hipStream_t st) {
  const int64_t waves = (int64_t)p.tokens * p.parts;
  if (bwd)
    hipLaunchKernelGGL((qk_norm_rope_bwd_kernel<XT, CT, LPR>), dim3(bwd_groups(waves)), dim3(256),
                       0, st, p);
  else {
    // (a grid has room for 2^32 threads in x)
    const int64_t wgs = (waves + 3) / 4 + (p.pos != nullptr), wide = std::min<int64_t>(wgs, 1 << 20);
    hipLaunchKernelGGL((qk_norm_rope_kernel<XT, CT, LPR>),
                       dim3((unsigned)wide, (unsigned)((wgs + wide - 1) / wide)), dim3(256), 0, st, p);
  }
  return hipGetLastError();
}
template <int XT, int CT>
hipError_t launch_lpr(const NormParams& p, bool bwd, hipStream_t st) {
  switch (lanes_per_row(p.D)) {
    case 1: return launch_one<XT, CT, 1>(p, bwd, st);
    case 2: return launch_one<XT, CT, 2>(p, bwd, st);
    case 4: return launch_one<XT, CT, 4>(p, bwd, st);
    case 8: return launch_one<XT, CT, 8>(p, bwd, st);
    default: return launch_one<XT, CT, 16>(p, bwd, st);
  }
}
template <int XT>
hipError_t launch_ct(const NormParams& p, int cdt, bool bwd, hipStream_t st) {
  if (cdt == MPX_F32) return launch_lpr<XT, MPX_F32>(p, bwd, st);
  if (cdt == MPX_F16) return launch_lpr<XT, MPX_F16>(p, bwd, st);
  return launch_lpr<XT, MPX_BF16>(p, bwd, st);
}
hipError_t launch_norm(const NormParams& p, int dt, int cdt, bool bwd, hipStream_t st) {
  if (dt == MPX_F32) return launch_ct<MPX_F32>(p, cdt, bwd, st);
  if (dt == MPX_F16) return launch_ct<MPX_F16>(p, cdt, bwd, st);
  return launch_ct<MPX_BF16>(p, cdt, bwd, st);
}

bool known(int dt) { return dt == MPX_F32 || dt == MPX_F16 || dt == MPX_BF16; }
bool aligned(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// Checks and parameters that both directions share.
int norm_params(NormParams& p, const char* fn, const void* q, const void* k, const void* wq,
                const void* wk, const void* cos, const void* sin, const int64_t* qs,
                const int64_t* ks, int B, int S, int H, int H_kv, int D, int offset,
                const int32_t* pos, int n_pos, float eps, int dt, int wdt, int cdt) {
  MPX_CHECK_ARG(known(dt) && known(wdt) && known(cdt), "%s: unknown dtype code %d, %d or %d", fn,
                dt, wdt, cdt);
  MPX_CHECK_ARG(B >= 0 && S >= 0 && H >= 0 && H_kv >= 0 && n_pos >= 0, "%s: negative size", fn);
  if (D <= 0 || D % 16 != 0 || D > 256) {
    set_error("%s: head_dim %d not supported (a multiple of 16 up to 256)", fn, D);
    return MPX_EUNSUPPORTED;
  }
  MPX_CHECK_ARG(std::isfinite(eps) && eps >= 0.f, "%s: eps must be finite and not negative", fn);
  MPX_CHECK_ARG((int64_t)B * S * ((int64_t)H + H_kv) < (1LL << 31), "%s: too many rows", fn);
  p.tokens = B * S;
  if ((int64_t)p.tokens * ((int64_t)H + H_kv) == 0) return MPX_OK;
  MPX_CHECK_ARG((H == 0 || q) && (H_kv == 0 || k) && wq && wk && cos && sin && qs && ks,
                "%s: null pointer argument", fn);
  MPX_CHECK_ARG(aligned(q) && aligned(k) && aligned(wq) && aligned(wk) && aligned(cos) &&
                    aligned(sin),
                "%s: tensors must be 16-byte aligned", fn);
  MPX_CHECK_ARG(pos || (offset >= 0 && (int64_t)offset + S <= n_pos),
                "%s: positions %d..%lld exceed the tables' %d rows", fn, offset,
                (long long)offset + S - 1, n_pos);
  const int es = dt == MPX_F32 ? 4 : 2;
  for (int i = 0; i < 3; ++i)
    MPX_CHECK_ARG(qs[i] >= 0 && (qs[i] * es) % 16 == 0 && ks[i] >= 0 && (ks[i] * es) % 16 == 0,
                  "%s: strides must be non-negative multiples of 16 bytes", fn);
  p.q = q; p.k = k; p.wq = wq; p.wk = wk; p.cos = cos; p.sin = sin;
  for (int i = 0; i < 3; ++i) {
    p.qs[i] = qs[i];
    p.ks[i] = ks[i];
  }
  p.pos = pos; p.B = B; p.S = S; p.H = H; p.H_kv = H_kv; p.D = D; p.offset = offset;
  p.n_pos = n_pos; p.eps = eps; p.wdt = wdt;
  cut(p);
  return MPX_OK;
}

}  // namespace
}  // namespace mpx

using namespace mpx;

extern "C" int mpx_qk_norm_rope(const void* q, const void* k, const void* q_weight,
                                const void* k_weight, const void* cos_cache, const void* sin_cache,
                                void* q_out, void* k_out, const int64_t* q_strides,
                                const int64_t* k_strides, int B, int S, int H, int H_kv, int D,
                                int offset, const int32_t* positions, int n_pos, float eps,
                                int dtype, int weight_dtype, int cache_dtype, int32_t* errors,
                                void* stream) {
  clear_error();
  NormParams p = {};
  const int rc = norm_params(p, "mpx_qk_norm_rope", q, k, q_weight, k_weight, cos_cache, sin_cache,
                             q_strides, k_strides, B, S, H, H_kv, D, offset, positions, n_pos, eps,
                             dtype, weight_dtype, cache_dtype);
  if (rc != MPX_OK) return rc;
  if (p.parts == 0) return MPX_OK;  // no row
  MPX_CHECK_ARG((H == 0 || q_out) && (H_kv == 0 || k_out) && (!positions || errors),
                "mpx_qk_norm_rope: null pointer argument");
  MPX_CHECK_ARG(aligned(q_out) && aligned(k_out),
                "mpx_qk_norm_rope: tensors must be 16-byte aligned");
  p.oq = q_out;
  p.ok = k_out;
  p.err = errors;
  MPX_CHECK_HIP(launch_norm(p, dtype, cache_dtype, false, (hipStream_t)stream));
  return MPX_OK;
}

extern "C" size_t mpx_qk_norm_rope_bwd_workspace_bytes(int B, int S, int H, int H_kv, int D) {
  if (B <= 0 || S <= 0 || H < 0 || H_kv < 0 || D <= 0 || D > 256 || D % 16 != 0 ||
      (int64_t)B * S * ((int64_t)H + H_kv) >= (1LL << 31))
    return 0;
  NormParams p = {};
  p.tokens = B * S; p.H = H; p.H_kv = H_kv; p.D = D;
  if (H + H_kv == 0) return 0;
  cut(p);
  return (size_t)bwd_groups((int64_t)p.tokens * p.parts) * 2 * D * sizeof(float);
}

extern "C" int mpx_qk_norm_rope_bwd(
    const void* q, const void* k, const void* q_weight, const void* k_weight, const void* cos_cache,
    const void* sin_cache, const void* dq_out, const void* dk_out, void* dq, void* dk,
    void* dq_weight, void* dk_weight, const int64_t* q_strides, const int64_t* k_strides,
    const int64_t* dq_out_strides, const int64_t* dk_out_strides, int B, int S, int H, int H_kv,
    int D, int offset, const int32_t* positions, int n_pos, float eps, int dtype, int weight_dtype,
    int cache_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  NormParams p = {};
  const int rc = norm_params(p, "mpx_qk_norm_rope_bwd", q, k, q_weight, k_weight, cos_cache,
                             sin_cache, q_strides, k_strides, B, S, H, H_kv, D, offset, positions,
                             n_pos, eps, dtype, weight_dtype, cache_dtype);
  if (rc != MPX_OK) return rc;
  hipStream_t st = (hipStream_t)stream;
  MPX_CHECK_ARG(dq_weight && dk_weight, "mpx_qk_norm_rope_bwd: null pointer argument");
  int groups = 0;
  if (p.parts != 0) {
    MPX_CHECK_ARG((H == 0 || (dq_out && dq)) && (H_kv == 0 || (dk_out && dk)) && dq_out_strides &&
                      dk_out_strides,
                  "mpx_qk_norm_rope_bwd: null pointer argument");
    MPX_CHECK_ARG(aligned(dq_out) && aligned(dk_out) && aligned(dq) && aligned(dk),
                  "mpx_qk_norm_rope_bwd: tensors must be 16-byte aligned");
    const int es = dtype == MPX_F32 ? 4 : 2;
    for (int i = 0; i < 3; ++i) {
      MPX_CHECK_ARG(dq_out_strides[i] >= 0 && (dq_out_strides[i] * es) % 16 == 0 &&
                        dk_out_strides[i] >= 0 && (dk_out_strides[i] * es) % 16 == 0,
                    "mpx_qk_norm_rope_bwd: strides must be non-negative multiples of 16 bytes");
      p.gqs[i] = dq_out_strides[i];
      p.gks[i] = dk_out_strides[i];
    }
    const size_t need = mpx_qk_norm_rope_bwd_workspace_bytes(B, S, H, H_kv, D);
    MPX_CHECK_ARG(workspace && aligned(workspace) && workspace_bytes >= need,
                  "mpx_qk_norm_rope_bwd: 16-byte aligned workspace of %zu bytes required, %zu given",
                  need, workspace_bytes);
    p.gq = dq_out; p.gk = dk_out; p.oq = dq; p.ok = dk; p.ws = (float*)workspace;
    groups = bwd_groups((int64_t)p.tokens * p.parts);
    MPX_CHECK_HIP(launch_norm(p, dtype, cache_dtype, true, st));
  }
  hipLaunchKernelGGL(qk_norm_dw_kernel, dim3(2 * D / 16), dim3(256), 0, st,
                     (const float*)workspace, dq_weight, dk_weight, D, groups, weight_dtype);
  MPX_CHECK_HIP(hipGetLastError());
  return MPX_OK;
}
