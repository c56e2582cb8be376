// The 8-bit paged KV cache on gfx950: append with quantisation (and K's
// rotation) on the way, and read-back. The formats and the rules of the scales
// are in mpx_cache8.h, the codes in mpx_code8.h.
#include <algorithm>

#include "mpx_code8.h"
#include "mpx_rows.h"

namespace mpx {

struct Append8Params {
  const void *k, *v, *cos, *sin;
  unsigned char *kpool, *vpool;
  float *kscale, *vscale;
  const int32_t *bt, *start, *ntok;
  int32_t* err;
  int64_t ks[3], vs[3];  // source (batch, token, head) strides in elements
  int B, T, H, D, num_blocks, bs, max_blocks, n_pos, pages, groups;
  int keep;  // slots that the call does not write keep their values, behind it too
};

// A sequence's tokens that have a place: positions [lo, hi).
struct Span8 {
  int64_t start, end, lo, hi;
  __device__ __forceinline__ Span8(const Append8Params& p, int b) {
    start = p.start[b];
    end = start + (p.ntok ? max(0, min(p.ntok[b], p.T)) : p.T);
    lo = max((int64_t)0, start);
    hi = min(end, (int64_t)p.max_blocks * p.bs);
    if (p.cos) hi = min(hi, (int64_t)p.n_pos);
  }
  __device__ __forceinline__ int64_t first_page(const Append8Params& p) const {
    return (u32)lo / (u32)p.bs;  // (lo < 2^31)
  }
};

// The error words, by a workgroup of its own (words that are only ever set
// would have to be cleared by a launch before).
__device__ void append8_errors(const Append8Params& p) {
  int neg = 0, past = 0, bad = 0, rope = 0;
  const int64_t cap = (int64_t)p.max_blocks * p.bs;
  const u32 n = (u32)p.B * (u32)p.pages;  // (under 2^31)
  for (u32 i0 = 0; i0 < n; i0 += 1024) {
    int page[4];
    bool look[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {  // (four look-ups on their way at once)
      const u32 i = i0 + 256 * u + threadIdx.x;
      const int b = i < n ? (int)(i / (u32)p.pages) : 0;
      const Span8 s(p, b);
      const bool any = i < n && s.end > s.start;
      neg |= any && s.start < 0;
      past |= any && s.end > cap;
      rope |= any && p.cos && min(s.end, cap) > max(s.lo, (int64_t)p.n_pos);
      const int64_t at = s.first_page(p) + (i - (u32)b * (u32)p.pages);
      look[u] = any && s.lo < s.hi && at * p.bs < s.hi;
      page[u] = look[u] ? p.bt[(int64_t)b * p.max_blocks + at] : 0;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) bad |= look[u] && (page[u] < 0 || page[u] >= p.num_blocks);
  }
  neg = __syncthreads_or(neg);
  past = __syncthreads_or(past);
  bad = __syncthreads_or(bad);
  rope = __syncthreads_or(rope);
  if (threadIdx.x != 0) return;
  p.err[0] = neg ? 1 : 0;
  p.err[1] = past ? 1 : 0;
  p.err[2] = bad ? 1 : 0;
  if (p.cos) p.err[3] = rope ? 1 : 0;
}

// A value to float32 by rounding to odd: what it loses stays in its last bit, so that
// rounding it to a code is rounding the value (a float32 rounded to nearest may land on
// the border between two codes, and the code be the wrong one of them).
__device__ __forceinline__ float odd_f32(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const u32 lo = (u32)b, kept = (lo & 0xe0000000u) | ((lo & 0x1fffffffu) ? 0x20000000u : 0u);
  return (float)__builtin_bit_cast(double, (b >> 32 << 32) | kept);
}

// One wave for each (sequence, page, head) and each of K and V: the scale of
// such a unit depends on all of its tokens. A token's row is held by LPR lanes,
// 64 / LPR tokens at a time. Two passes over the unit's new tokens: their largest
// value, which gives the scale, then the codes; rows that fit stay in registers
// in between (read again: 93 us instead of 81 for the append below). Where the scale
// grew, the page's earlier codes are brought to it. Memory bound: 4 x 4096 tokens of
// 32 heads of D 128, bf16 to int8, K rotated, 86 us (403 MB read and written;
// 82 with the rotation in float32, whose codes are now and then the neighbours of
// the right ones). One token of 64 sequences 5.0 us, a launch and one chain of loads.
template <int XT, int CT, bool I8, int LPR, bool ROPE>
__global__ __launch_bounds__(256) void kv_append8_kernel(Append8Params p) {
  typedef typename Elem<XT>::T T;
  typedef typename Elem<CT>::T C;
  constexpr int TPW = 64 / LPR;  // tokens at a time
  const u32 index = blockIdx.y * gridDim.x + blockIdx.x;
  if (index == 0) {
    append8_errors(p);
    return;
  }
  const int lane = threadIdx.x & 63;
  // workgroup 1 + (sequence * pages + page) * units' groups + group
  const u32 wg = index - 1, seq_page = wg / (u32)p.groups;
  if (seq_page >= (u32)p.B * (u32)p.pages) return;
  const int b = p.pages == 1 ? (int)seq_page : (int)(seq_page / (u32)p.pages);
  const int at_page = (int)(seq_page - (u32)b * (u32)p.pages);
  const int unit = (int)(wg - seq_page * (u32)p.groups) * 4 +
                   __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = unit >> 1;
  const bool isk = !(unit & 1);
  if (h >= p.H) return;
  const Span8 seq(p, b);
  const int64_t page_at = seq.first_page(p) + at_page;
  const int64_t base = page_at * p.bs;
  const int s0 = (int)max((int64_t)0, seq.lo - base), s1 = (int)min((int64_t)p.bs, seq.hi - base);
  if (s0 >= s1) return;
  const int page = p.bt[(int64_t)b * p.max_blocks + page_at];
  // This lane's 16 values of a row: 8 pairs of K that is rotated, else 16 in a row.
  const int half = p.D / 2, c = lane % LPR;
  const bool on = 8 * c < half, turn = ROPE && isk;
  const int d0 = turn ? 8 * c : 16 * c, d1 = turn ? half + 8 * c : 16 * c + 8;
  const int64_t* st = isk ? p.ks : p.vs;
  const T* src = (const T*)(isk ? p.k : p.v) + b * st[0] + (base - seq.start) * st[1] + h * st[2];
  const int first = s0 + lane / LPR;
  struct Row {
    R8<T> a, b;
  };
  auto read = [&](int s, Row& r) __attribute__((always_inline)) {
    r.a.clear();
    r.b.clear();
    if (on && s < s1) {
      r.a.load(src + s * st[1] + d0);
      r.b.load(src + s * st[1] + d1);
    }
  };
  auto values = [&](int s, const Row& r, float* x) __attribute__((always_inline)) {
    if (turn && on && s < s1) {
      const int64_t at = (base + s) * half + d0;
      R8<C> cs, sn;
      cs.load((const C*)p.cos + at);
      sn.load((const C*)p.sin + at);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // (products of float32 numbers are exact in float64)
        const double a = r.a.get(e), b = r.b.get(e), c = cs.get(e), n = sn.get(e);
        x[e] = odd_f32(__builtin_fma(a, c, -(b * n)));
        x[8 + e] = odd_f32(__builtin_fma(a, n, b * c));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = r.a.get(e);
        x[8 + e] = r.b.get(e);
      }
    }
  };
  // Rows that fit stay in registers between the passes (they are asked for before
  // the page is known), others are read again.
  constexpr int HOLD = 4;
  const int n_new = s1 - s0;
  float held[HOLD][16];
  {
    Row rows[HOLD];
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
      if (i * TPW < n_new) read(first + i * TPW, rows[i]);
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
      if (i * TPW < n_new) values(first + i * TPW, rows[i], held[i]);
  }
  if (page < 0 || page >= p.num_blocks) return;
  unsigned char* dst = (isk ? p.kpool : p.vpool) + ((int64_t)page * p.bs * p.H + h) * p.D;
  const int64_t row = (int64_t)p.H * p.D;
  float* scale_at = (isk ? p.kscale : p.vscale) + (int64_t)page * p.H + h;
  const float was = *scale_at;

  // f(slot, values) for every new row.
  auto each = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
      if (i * TPW < n_new) f(first + i * TPW, held[i]);
    for (int s = first + HOLD * TPW; s - first + s0 < s1; s += TPW) {
      Row r;
      float x[16];
      read(s, r);
      values(s, r, x);
      f(s, x);
    }
  };
  // The largest value by its bits, infinities and NaN on top; where there are
  // such, or values past what the largest scale holds, once more without them.
  u32 top = 0;
  each([&](int, const float* x) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
  });
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = max(top, (u32)__shfl_xor((int)top, off, 64));
  const bool in_range = top < 0x78000000u;  // 2^113
  float amax = __uint_as_float(top);
  if (!in_range) {
    amax = 0.f;
    each([&](int, const float* x) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float a = fabsf(x[e]);
        amax = fmaxf(amax, a < INFINITY ? a : 0.f);
      }
    });
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off, 64));
  }
  const int e = need_exp8<I8>(amax);
  const float need = pow2f(e);
  const bool anew = s0 == 0 && (!p.keep || s1 == p.bs);
  const float now = anew ? need : fmaxf(was, need);
  // (a scale kept from before need not be a power of two)
  const float inv = now == need ? pow2f(-e) : 1.0f / now;
  auto place = [&](unsigned char* at, u32x2 x, u32x2 y) __attribute__((always_inline)) {
    if (turn) {
      *(u32x2*)(at + d0) = x;
      *(u32x2*)(at + d1) = y;
    } else {
      *(u32x4*)(at + d0) = (u32x4){x[0], x[1], y[0], y[1]};
    }
  };
  each([&](int s, const float* x) __attribute__((always_inline)) {
    if (!on || s >= s1) return;
    u32 w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      w[q] = in_range ? encode4_in_range<I8>(x + 4 * q, inv)
                      : encode4<I8>(x[4 * q] * inv, x[4 * q + 1] * inv, x[4 * q + 2] * inv,
                                    x[4 * q + 3] * inv);
    place(dst + s * row, (u32x2){w[0], w[1]}, (u32x2){w[2], w[3]});
  });
  const int rest = p.keep ? p.bs : s0;  // slots whose codes are brought to a larger scale
  if (!anew && now != was) {
    const float f = was * inv;
    for (int s = lane / LPR; s < rest; s += TPW) {
      if (!on || (s >= s0 && s < s1)) continue;
      unsigned char* at = dst + s * row;
      u32x2 x = *(const u32x2*)(at + d0), y = *(const u32x2*)(at + d1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[i] = encode4<I8>(decode1<I8>(x[i], 0) * f, decode1<I8>(x[i], 1) * f,
                           decode1<I8>(x[i], 2) * f, decode1<I8>(x[i], 3) * f);
        y[i] = encode4<I8>(decode1<I8>(y[i], 0) * f, decode1<I8>(y[i], 1) * f,
                           decode1<I8>(y[i], 2) * f, decode1<I8>(y[i], 3) * f);
      }
      place(at, x, y);
    }
  }
  if (lane == 0) *scale_at = now;
}

struct Load8Params {
  const unsigned char *kpool, *vpool;
  const float *kscale, *vscale;
  const int32_t *bt, *start, *ntok;
  void *k, *v;
  int B, T, H, D, num_blocks, bs, max_blocks;
};

// One thread for 16 codes of a token row: a 16-byte load, two or four 16-byte
// stores. Memory bound: 4 x 4096 tokens of 32 heads of D 128 to bf16 69 us (403 MB,
// 5.8 TB/s).
template <int XT, bool I8>
__global__ __launch_bounds__(256) void kv_load8_kernel(Load8Params p) {
  typedef typename Elem<XT>::T T;
  const int cpr = p.H * p.D / 16;  // chunks of a token
  const int64_t n = (int64_t)p.B * p.T * cpr;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    int c, b, t;
    if (n < (1ll << 32)) {  // (a division of 64 bits takes some hundred instructions)
      const u32 tok = (u32)i / (u32)cpr;
      c = (int)((u32)i - tok * (u32)cpr);
      b = (int)(tok / (u32)p.T);
      t = (int)(tok - (u32)b * (u32)p.T);
    } else {
      const int64_t tok = i / cpr;
      c = (int)(i - tok * cpr);
      b = (int)(tok / p.T);
      t = (int)(tok - (int64_t)b * p.T);
    }
    const int64_t pos = (int64_t)p.start[b] + t;
    u32x4 kc = {0u, 0u, 0u, 0u}, vc = kc;
    float ks = 0.f, vs = 0.f;
    if (t < p.ntok[b] && pos >= 0 && pos < (int64_t)p.max_blocks * p.bs) {
      const int64_t at = (u32)pos / (u32)p.bs;  // (pos < 2^30)
      const int page = p.bt[(int64_t)b * p.max_blocks + at];
      if (page >= 0 && page < p.num_blocks) {
        const int64_t off = (((int64_t)page * p.bs + (pos - at * p.bs)) * cpr + c) * 16;
        kc = *(const u32x4*)(p.kpool + off);
        vc = *(const u32x4*)(p.vpool + off);
        const int64_t sc = (int64_t)page * p.H + c * 16 / p.D;
        ks = p.kscale[sc];
        vs = p.vscale[sc];
      }
    }
    auto put = [&](void* out, u32x4 x, float s) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = decode1<I8>(x[2 * q + (e >> 2)], e & 3) * s;
        R8<T> y;
        y.set(v);
        y.store((T*)out + i * 16 + q * 8);
      }
    };
    put(p.k, kc, ks);
    put(p.v, vc, vs);
  }
}

namespace {

int lanes_per_row8(int D) {
  int n = 1;
  while (n * 16 < D) n *= 2;
  return n;
}

template <int XT, int CT, bool I8, bool ROPE>
void launch_append_lpr(const Append8Params& p, dim3 grid, hipStream_t st) {
  switch (lanes_per_row8(p.D)) {
    case 1: hipLaunchKernelGGL((kv_append8_kernel<XT, CT, I8, 1, ROPE>), grid, dim3(256), 0, st, p); break;
    case 2: hipLaunchKernelGGL((kv_append8_kernel<XT, CT, I8, 2, ROPE>), grid, dim3(256), 0, st, p); break;
    case 4: hipLaunchKernelGGL((kv_append8_kernel<XT, CT, I8, 4, ROPE>), grid, dim3(256), 0, st, p); break;
    case 8: hipLaunchKernelGGL((kv_append8_kernel<XT, CT, I8, 8, ROPE>), grid, dim3(256), 0, st, p); break;
    default: hipLaunchKernelGGL((kv_append8_kernel<XT, CT, I8, 16, ROPE>), grid, dim3(256), 0, st, p);
  }
}
template <int XT, bool I8>
void launch_append8(const Append8Params& p, int cdt, dim3 grid, hipStream_t st) {
  if (!p.cos)
    launch_append_lpr<XT, MPX_F32, I8, false>(p, grid, st);
  else if (cdt == MPX_F32)
    launch_append_lpr<XT, MPX_F32, I8, true>(p, grid, st);
  else if (cdt == MPX_F16)
    launch_append_lpr<XT, MPX_F16, I8, true>(p, grid, st);
  else
    launch_append_lpr<XT, MPX_BF16, I8, true>(p, grid, st);
}

bool known8(int dt) { return dt == MPX_F32 || dt == MPX_F16 || dt == MPX_BF16; }
bool aligned8(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// Checks that both directions share.
int check_cache8(const char* fn, int B, int T, int H, int D, int num_blocks, int block_size,
                 int max_blocks, int dtype, int code) {
  MPX_CHECK_ARG(known8(dtype), "%s: unknown dtype code %d", fn, dtype);
  MPX_CHECK_ARG(code == MPX8_E4M3 || code == MPX8_INT8, "%s: unknown code format %d", fn, code);
  MPX_CHECK_ARG(B >= 0 && T >= 0 && H >= 0 && num_blocks >= 0 && max_blocks >= 0,
                "%s: negative size", fn);
  MPX_CHECK_ARG(block_size > 0 && block_size <= MPX8_MAX_BLOCK_SIZE,
                "%s: block_size must be in 1..%d", fn, MPX8_MAX_BLOCK_SIZE);
  if (D <= 0 || D % 16 != 0 || D > 256) {
    set_error("%s: head_dim %d not supported (a multiple of 16 up to 256)", fn, D);
    return MPX_EUNSUPPORTED;
  }
  MPX_CHECK_ARG((int64_t)H * D < (1 << 24), "%s: head count too large", fn);
  MPX_CHECK_ARG((int64_t)max_blocks * block_size < (1LL << 30), "%s: block table too large", fn);
  return MPX_OK;
}

}  // namespace
}  // namespace mpx

using namespace mpx;

namespace {

int append8(const char* fn, int keep, const void* k, const void* v, void* k_pool, void* v_pool,
            float* k_scales, float* v_scales, const int32_t* block_tables,
            const int32_t* start_pos, const int32_t* n_tokens, const int64_t* k_strides,
            const int64_t* v_strides, int B, int T, int H, int D, int num_blocks, int block_size,
            int max_blocks, int dtype, int code, const void* cos_cache, const void* sin_cache,
            int n_pos, int cache_dtype, int32_t* errors, void* stream) {
  clear_error();
  const int rc = check_cache8(fn, B, T, H, D, num_blocks, block_size, max_blocks, dtype, code);
  if (rc != MPX_OK) return rc;
  const bool rope = cos_cache || sin_cache;
  MPX_CHECK_ARG(!rope || (cos_cache && sin_cache && n_pos >= 0 && known8(cache_dtype)),
                "%s: cos and sin tables go together", fn);
  if ((int64_t)B * T * H == 0) return MPX_OK;
  MPX_CHECK_ARG(k && v && (block_tables || max_blocks == 0) && start_pos && k_strides &&
                    v_strides && errors &&
                    ((k_pool && v_pool && k_scales && v_scales) || num_blocks == 0),
                "%s: null pointer argument", fn);
  MPX_CHECK_ARG(aligned8(k) && aligned8(v) && aligned8(k_pool) && aligned8(v_pool) &&
                    aligned8(cos_cache) && aligned8(sin_cache),
                "%s: tensors must be 16-byte aligned", fn);
  const int vec = dtype == MPX_F32 ? 4 : 8;
  Append8Params p;
  for (int i = 0; i < 3; ++i) {
    MPX_CHECK_ARG(k_strides[i] >= 0 && k_strides[i] % vec == 0 && v_strides[i] >= 0 &&
                      v_strides[i] % vec == 0,
                  "%s: strides must be non-negative multiples of %d elements", fn, vec);
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
  }
  p.k = k; p.v = v; p.cos = cos_cache; p.sin = sin_cache;
  p.kpool = (unsigned char*)k_pool; p.vpool = (unsigned char*)v_pool;
  p.kscale = k_scales; p.vscale = v_scales;
  p.bt = block_tables; p.start = start_pos; p.ntok = n_tokens; p.err = errors;
  p.B = B; p.T = T; p.H = H; p.D = D; p.num_blocks = num_blocks; p.bs = block_size;
  p.max_blocks = max_blocks; p.n_pos = n_pos; p.keep = keep;
  // T tokens touch at most this many pages, wherever they start
  p.pages = (int)(((int64_t)T + block_size - 2) / block_size + 1);
  p.groups = (2 * H + 3) / 4;
  const int64_t a_seq = (int64_t)p.pages * p.groups;
  MPX_CHECK_ARG(B < 65535 && a_seq < (1ll << 31) && 1 + a_seq * B < (1ll << 31),
                "%s: too many tokens in one call", fn);
  const int64_t wgs = 1 + a_seq * B, wide = std::min<int64_t>(wgs, 1 << 20);
  const dim3 grid((unsigned)wide, (unsigned)((wgs + wide - 1) / wide));
  hipStream_t st = (hipStream_t)stream;
  if (code == MPX8_INT8) {
    if (dtype == MPX_F32) launch_append8<MPX_F32, true>(p, cache_dtype, grid, st);
    else if (dtype == MPX_F16) launch_append8<MPX_F16, true>(p, cache_dtype, grid, st);
    else launch_append8<MPX_BF16, true>(p, cache_dtype, grid, st);
  } else {
    if (dtype == MPX_F32) launch_append8<MPX_F32, false>(p, cache_dtype, grid, st);
    else if (dtype == MPX_F16) launch_append8<MPX_F16, false>(p, cache_dtype, grid, st);
    else launch_append8<MPX_BF16, false>(p, cache_dtype, grid, st);
  }
  MPX_CHECK_HIP(hipGetLastError());
  return MPX_OK;
}

}  // namespace

extern "C" int mpx_kv_append8(const void* k, const void* v, void* k_pool, void* v_pool,
                              float* k_scales, float* v_scales, const int32_t* block_tables,
                              const int32_t* start_pos, const int32_t* n_tokens,
                              const int64_t* k_strides, const int64_t* v_strides, int B, int T,
                              int H, int D, int num_blocks, int block_size, int max_blocks,
                              int dtype, int code, const void* cos_cache, const void* sin_cache,
                              int n_pos, int cache_dtype, int32_t* errors, void* stream) {
  return append8("mpx_kv_append8", 0, k, v, k_pool, v_pool, k_scales, v_scales, block_tables,
                 start_pos, n_tokens, k_strides, v_strides, B, T, H, D, num_blocks, block_size,
                 max_blocks, dtype, code, cos_cache, sin_cache, n_pos, cache_dtype, errors, stream);
}

extern "C" int mpx_kv_write8(const void* k, const void* v, void* k_pool, void* v_pool,
                             float* k_scales, float* v_scales, const int32_t* block_tables,
                             const int32_t* start_pos, const int32_t* n_tokens,
                             const int64_t* k_strides, const int64_t* v_strides, int B, int T,
                             int H, int D, int num_blocks, int block_size, int max_blocks,
                             int dtype, int code, const void* cos_cache, const void* sin_cache,
                             int n_pos, int cache_dtype, int32_t* errors, void* stream) {
  return append8("mpx_kv_write8", 1, k, v, k_pool, v_pool, k_scales, v_scales, block_tables,
                 start_pos, n_tokens, k_strides, v_strides, B, T, H, D, num_blocks, block_size,
                 max_blocks, dtype, code, cos_cache, sin_cache, n_pos, cache_dtype, errors, stream);
}

extern "C" int mpx_kv_load8(const void* k_pool, const void* v_pool, const float* k_scales,
                            const float* v_scales, const int32_t* block_tables,
                            const int32_t* start_pos, const int32_t* n_tokens, void* k_out,
                            void* v_out, int B, int T, int H, int D, int num_blocks,
                            int block_size, int max_blocks, int dtype, int code, void* stream) {
  clear_error();
  const char* fn = "mpx_kv_load8";
  const int rc = check_cache8(fn, B, T, H, D, num_blocks, block_size, max_blocks, dtype, code);
  if (rc != MPX_OK) return rc;
  if ((int64_t)B * T * H == 0) return MPX_OK;
  MPX_CHECK_ARG(start_pos && n_tokens && k_out && v_out && (block_tables || max_blocks == 0) &&
                    ((k_pool && v_pool && k_scales && v_scales) || num_blocks == 0),
                "%s: null pointer argument", fn);
  MPX_CHECK_ARG(aligned8(k_pool) && aligned8(v_pool) && aligned8(k_out) && aligned8(v_out),
                "%s: tensors must be 16-byte aligned", fn);
  Load8Params p;
  p.kpool = (const unsigned char*)k_pool; p.vpool = (const unsigned char*)v_pool;
  p.kscale = k_scales; p.vscale = v_scales; p.bt = block_tables; p.start = start_pos;
  p.ntok = n_tokens; p.k = k_out; p.v = v_out;
  p.B = B; p.T = T; p.H = H; p.D = D; p.num_blocks = num_blocks; p.bs = block_size;
  p.max_blocks = max_blocks;
  const int64_t n = (int64_t)B * T * (H * D / 16);
  const dim3 grid((unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20));
  hipStream_t st = (hipStream_t)stream;
#define MPX_LOAD8(XT)                                                                     \
  do {                                                                                    \
    if (code == MPX8_INT8)                                                                \
      hipLaunchKernelGGL((kv_load8_kernel<XT, true>), grid, dim3(256), 0, st, p);         \
    else                                                                                  \
      hipLaunchKernelGGL((kv_load8_kernel<XT, false>), grid, dim3(256), 0, st, p);        \
  } while (0)
  if (dtype == MPX_F32) MPX_LOAD8(MPX_F32);
  else if (dtype == MPX_F16) MPX_LOAD8(MPX_F16);
  else MPX_LOAD8(MPX_BF16);
#undef MPX_LOAD8
  MPX_CHECK_HIP(hipGetLastError());
  return MPX_OK;
}
