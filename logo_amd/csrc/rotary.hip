// Rotary embedding by positions, and the append of keys and values to a paged
// cache with that rotation on the way, for gfx950.
//
// A pair (a, b) of a head's first R elements -- (i, i + R / 2), or (2 i, 2 i + 1)
// interleaved -- of a token at position p turns by t = p f_i:
//   a' = m (a cos t - b sin t),   b' = m (b cos t + a sin t)
// and elements R .. D - 1 pass through.  The transpose (the backward pass) turns
// by -t.  Sums and products in fp32, one rounding at the end.
//
// Angles.  f_i comes as turns per position in 64-bit fixed point, F_i = f_i /
// (2 pi) 2^64 mod 2^64, so p F_i mod 2^64 is the angle's fraction of a turn,
// exact to p 2^-65 turns however far p is (in fp32, p f_i itself is off by whole
// degrees from p = 10^6 on).  Its distance to the nearest quarter turn, an integer
// below 2^29 in units of 2^-32 turns, converts to fp32 with a relative error of
// 2^-24, and sine and cosine of at most pi / 4 are their Taylor polynomials up to
// x^11 and x^10, whose next terms are below 2^-24 of the result.
//
// Bound by memory: each row is read and written once.  A workgroup takes a few
// tokens of one tensor; cos and sin of its tokens are worked out once into LDS
// and serve all heads.  A thread keeps its place in the row and walks the rows, two
// in flight at a time; the first two are on their way before the tokens' positions
// are known.  Loads and stores are streaming (nothing is read again).
//
// Measured: 4 x 8192 tokens of 16 + 4 heads of 128 in bf16, 336 MB a pass in 60 us (5.6
// TB/s; a large copy with streaming loads and stores 5.9), the training step's two
// passes 121 us; 32K keys and values of 4 heads and 16 query heads of 128 in fp16
// appended and rotated, 306 MB in 57 us; a decode step of 8 or 32 sequences 5 to 6 us, a
// launch's own time.  Workgroups of 1024 items: of 256, which pay for their tokens'
// angles, the training step takes 128 us and the append 90, of 4096 128 and 62.  Two
// items in flight: one takes 126 and 57 us, four 119 and 69.
#include <math.h>

#include <algorithm>

#include "capi.hpp"
#include "common.hpp"
#include "paged.hpp"

namespace logo {

constexpr int kRotThreads = 256;
constexpr int kRotMaxTok = 16;     // tokens per workgroup
constexpr int kRotItems = 1024;    // items (row chunks) a workgroup aims for
constexpr int kRotFlight = 2;      // items of a thread in flight
constexpr int kRotMaxDim = 256;    // a row has at most as many items as a workgroup threads

struct RotRows {
  const void* x;
  void* y;
  int64_t x_batch, x_token, x_head;  // strides in elements
  int64_t y_batch, y_token, y_head;  // (paged rows: page, slot, head)
  int heads;
  int tok, hc;                       // tokens and heads per workgroup
  bool rotate, paged;
};

struct RotArgs {
  RotRows r[4];
  const void* positions;  // int32 or int64 [n] (rotary), else null
  bool pos64;
  uint32_t n, per_batch;  // tokens (below 2^31); tokens per batch entry
  const uint64_t* turns;  // [rot / 2]
  float amp;
  int rot, d, units, pair_units;  // units: items per row, of which pair_units rotate
  int rows;                       // rows that the threads of a workgroup cover at once
  bool inter, inverse;
  // append
  const int32_t* table;
  int64_t table_row;
  int table_width, page_shift, nseq;
  int64_t pages;
  const int32_t* cu;
  const int32_t* lens;
};

// Cosine and sine of a fraction of a turn in units of 2^-64.
__device__ __forceinline__ float2 turn_cos_sin(uint64_t frac) {
  const uint32_t hi = (uint32_t)(frac >> 32);
  const uint32_t quarter = (hi + 0x20000000u) >> 30;            // nearest quarter turn
  const int32_t rest = (int32_t)(hi - (quarter << 30));         // in [-2^29, 2^29)
  const float x = (float)rest * (float)(6.283185307179586 / 4294967296.0);
  const float x2 = x * x;
  float s = fmaf(x2, -1.f / 39916800.f, 1.f / 362880.f);
  s = fmaf(x2, s, -1.f / 5040.f);
  s = fmaf(x2, s, 1.f / 120.f);
  s = fmaf(x2, s, -1.f / 6.f);
  s = fmaf(x * x2, s, x);
  float c = fmaf(x2, -1.f / 3628800.f, 1.f / 40320.f);
  c = fmaf(x2, c, -1.f / 720.f);
  c = fmaf(x2, c, 1.f / 24.f);
  c = fmaf(x2, c, -0.5f);
  c = fmaf(x2, c, 1.f);
  const float cs = (quarter & 1) ? s : c, sn = (quarter & 1) ? c : s;
  // quarter turns: (c, s), (-s, c), (-c, -s), (s, -c)
  const bool negc = ((quarter + 1) & 2) != 0, negs = (quarter & 2) != 0;
  return float2{negc ? -cs : cs, negs ? -sn : sn};
}

// What a workgroup knows of each of its tokens.
struct RotTok {
  int64_t pos;    // position
  int64_t y_off;  // batch and token part of the destination row's offset; paged: of the page and slot
  int state;      // 0: written; 1: zero row (no position); 2: nothing to write
};

template <typename T, int VEC, bool APPEND, bool INTER>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(const RotArgs a) {
  typedef T vec __attribute__((ext_vector_type(VEC)));
  const RotRows& r = a.r[blockIdx.z];
  const uint32_t n0 = blockIdx.x * (uint32_t)r.tok;
  const int h0 = blockIdx.y * r.hc;
  if (n0 >= a.n || h0 >= r.heads) return;
  const int ntok = min(r.tok, (int)(a.n - n0)), tid = threadIdx.x;
  extern __shared__ __attribute__((aligned(16))) char rot_smem[];
  RotTok* const info = reinterpret_cast<RotTok*>(rot_smem);                      // [kRotMaxTok]
  float2* const cs = reinterpret_cast<float2*>(rot_smem + kRotMaxTok * sizeof(RotTok));  // [ntok][rot / 2]
  // the thread's place: item u of every a.rows-th (token, head) row from rg on
  const int nh = min(r.hc, r.heads - h0), half = a.rot >> 1;
  const int rg = tid / a.units, u = tid - rg * a.units;
  const int dt = a.rows / nh, dh = a.rows - dt * nh;
  const bool pair = u < a.pair_units;
  const int e0 = !pair ? a.rot + VEC * (u - a.pair_units) : INTER ? 2 * VEC * u : VEC * u;
  const int e1 = !pair ? e0 : INTER ? e0 + VEC : half + VEC * u;
  const T* const x = static_cast<const T*>(r.x) + (int64_t)h0 * r.x_head;
  T* const y = static_cast<T*>(r.y) + (int64_t)h0 * r.y_head;
  const int items = rg < a.rows ? (ntok * nh - rg + a.rows - 1) / a.rows : 0;
  vec v0[kRotFlight], v1[kRotFlight];
  int it = rg / nh, ih = rg - it * nh;  // the next row to load
  int ot = it, oh = ih;                 // and to store
  auto next = [&](int& t, int& h) {
    t += dt;
    h += dh;
    if (h >= nh) h -= nh, ++t;
  };
  auto load = [&](int q) {
    const uint32_t n = n0 + it;
    int64_t off = n * r.x_token;
    if (!APPEND && a.per_batch < a.n) {
      const uint32_t b = n / a.per_batch;
      off = b * r.x_batch + (n - b * a.per_batch) * r.x_token;
    }
    const T* const xr = x + off + (int64_t)ih * r.x_head;
    v0[q] = ld_nt(reinterpret_cast<const vec*>(xr + e0));
    if (pair) v1[q] = ld_nt(reinterpret_cast<const vec*>(xr + e1));
    next(it, ih);
  };
#pragma unroll
  for (int q = 0; q < kRotFlight; ++q)
    if (q < items) load(q);

  // the frequency whose angles the thread works out (rot / 2 <= 256 = the threads), and of which tokens
  const int steps = half > 0 ? kRotThreads / half : 1, my_t = half > 0 ? tid / half : 0, my_i = tid - my_t * half;
  const uint64_t my_turns = r.rotate && my_t < steps && my_i < half ? a.turns[my_i] : 0;
  if constexpr (APPEND) {
    // the first wave, a lane a token
    if (tid < 64) {
      int cnt = 0;  // sequences that end at or before the lane's token
      for (int c = 0; c < a.nseq; c += 64) {
        const int32_t e = c + tid < a.nseq ? a.cu[c + tid + 1] : 0x7fffffff;
        for (int t = 0; t < ntok; ++t) {
          const int k = __builtin_popcountll(__ballot(e <= (int)n0 + t));
          cnt += tid == t ? k : 0;
        }
      }
      const int n = (int)n0 + tid;
      RotTok k{0, n * r.y_token, 1};
      if (tid < ntok && cnt < a.nseq) {
        const int lo = a.cu[cnt], hi = a.cu[cnt + 1];
        k.pos = (int64_t)a.lens[cnt] - hi + n;
        if (n >= lo && k.pos >= 0) k.state = 0;
      }
      if (r.paged) {
        const int64_t col = k.pos >> a.page_shift;
        int page = -1;
        if (k.state == 0 && col < a.table_width) page = a.table[cnt * a.table_row + col];
        const bool held = page >= 0 && page < a.pages;
        k.y_off = held ? page * r.y_batch + (k.pos & ((1 << a.page_shift) - 1)) * r.y_token : 0;
        if (!held) k.state = 2;
      }
      if (tid < ntok) info[tid] = k;
    }
  } else {
    if (tid < ntok) {
      const uint32_t n = n0 + tid, b = n / a.per_batch, t = n - b * a.per_batch;
      const int64_t p = a.pos64 ? static_cast<const int64_t*>(a.positions)[n] : static_cast<const int32_t*>(a.positions)[n];
      info[tid] = RotTok{p, b * r.y_batch + t * r.y_token, 0};
    }
  }
  __syncthreads();
  if (r.rotate) {
    if (my_t < steps)
      for (int t = my_t; t < ntok; t += steps) {
        float2 v = turn_cos_sin((uint64_t)info[t].pos * my_turns);
        v.x *= a.amp;
        v.y *= a.inverse ? -a.amp : a.amp;
        cs[t * half + my_i] = v;
      }
    __syncthreads();
  }
  for (int k0 = 0; k0 < items; k0 += kRotFlight) {
#pragma unroll
    for (int q = 0; q < kRotFlight; ++q) {
      if (k0 + q >= items) break;
      const int t = ot;
      const RotTok k = info[t];
      T* const yr = y + k.y_off + (int64_t)oh * r.y_head;
      next(ot, oh);
      vec a0 = v0[q], a1 = v1[q];
      if (k0 + q + kRotFlight < items) load(q);
      if (pair && r.rotate) {
        const float2* const c = cs + t * half + VEC * u;
        T in[2 * VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) in[e] = a0[e], in[VEC + e] = a1[e];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          constexpr int S = INTER ? 2 : 1, B = INTER ? 1 : VEC;
          const float p = (float)in[S * e], q2 = (float)in[S * e + B];
          in[S * e] = (T)(p * c[e].x - q2 * c[e].y);
          in[S * e + B] = (T)(q2 * c[e].x + p * c[e].y);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) a0[e] = in[e], a1[e] = in[VEC + e];
      }
      if (k.state == 1) a0 = vec{}, a1 = vec{};
      if (k.state != 2) {
        *reinterpret_cast<vec*>(yr + e0) = a0;
        if (pair) *reinterpret_cast<vec*>(yr + e1) = a1;
      }
    }
  }
}

// The widest vector of at most 16 bytes whose multiples all rows' offsets are.
static int rot_vec(const RotArgs& a, int nr, int size) {
  int64_t bits = a.rot / 2 | (a.d - a.rot);
  for (int i = 0; i < nr; ++i) {
    const RotRows& r = a.r[i];
    bits |= r.x_batch | r.x_token | r.x_head | r.y_batch | r.y_token | r.y_head;
    bits |= (int64_t)(((uintptr_t)r.x | (uintptr_t)r.y) / size);
  }
  int v = 16 / size;
  while (v > 1 && bits % v) v >>= 1;
  return v;
}

template <typename T, int VEC, bool APPEND>
static int rot_launch(RotArgs a, int nr, bool inplace, hipStream_t st) {
  a.pair_units = a.rot / 2 / VEC;
  a.units = a.pair_units + (inplace ? 0 : (a.d - a.rot) / VEC);
  a.rows = std::max(1, kRotThreads / a.units);
  int64_t gx = 1;
  int gy = 1, tok = 1;
  for (int i = 0; i < nr; ++i) {
    RotRows& r = a.r[i];
    r.hc = std::min(r.heads, std::max(a.rows, kRotItems / a.units));
    r.tok = std::max(1, std::min(kRotMaxTok, kRotItems / (r.hc * a.units)));
    gx = std::max(gx, ((int64_t)a.n + r.tok - 1) / r.tok);
    gy = std::max(gy, (r.heads + r.hc - 1) / r.hc);
    tok = std::max(tok, r.tok);
  }
  LOGO_REQUIRE(gx < ((int64_t)1 << 31) && gy <= 65535, "too many tokens or heads");
  const size_t smem = kRotMaxTok * sizeof(RotTok) + (size_t)tok * (a.rot / 2) * sizeof(float2);
  auto kern = a.inter ? rotary_kernel<T, VEC, APPEND, true> : rotary_kernel<T, VEC, APPEND, false>;
  hipLaunchKernelGGL(kern, dim3((unsigned)gx, gy, nr), dim3(kRotThreads), smem, st, a);
  LOGO_LAUNCH_CHECK("rotary_kernel");
  return LOGO_OK;
}

template <typename T, bool APPEND>
static int rot_dispatch(const RotArgs& a, int nr, bool inplace, hipStream_t st) {
  const int v = rot_vec(a, nr, sizeof(T));
  if constexpr (sizeof(T) == 2)
    if (v == 8) return rot_launch<T, 8, APPEND>(a, nr, inplace, st);
  if (v == 4) return rot_launch<T, 4, APPEND>(a, nr, inplace, st);
  if (v == 2) return rot_launch<T, 2, APPEND>(a, nr, inplace, st);
  return rot_launch<T, 1, APPEND>(a, nr, inplace, st);
}

static int rot_check(int d, int rot, const void* turns, float amp) {
  LOGO_REQUIRE(d >= 1 && d <= kRotMaxDim, "head dim %d unsupported (at most %d)", d, kRotMaxDim);
  LOGO_REQUIRE(rot >= 0 && rot <= d && rot % 2 == 0, "rot (%d) must be even and at most the head dim (%d)", rot, d);
  LOGO_REQUIRE(rot == 0 || turns != nullptr, "null turns");
  LOGO_REQUIRE(isfinite(amp), "amplitude must be finite");
  return LOGO_OK;
}

}  // namespace logo

using namespace logo;

extern "C" int logo_rotary(const logo_rows* rows, int n_rows, const void* positions, int position_bits,
                           int64_t n_tokens, int64_t tokens_per_batch, int d, const uint64_t* turns, int rot,
                           int interleaved, float amplitude, int inverse, int dtype, void* stream) {
  LOGO_REQUIRE(dtype == LOGO_DTYPE_BF16 || dtype == LOGO_DTYPE_F16 || dtype == LOGO_DTYPE_F32, "dtype %d unsupported",
               dtype);
  const int rc = rot_check(d, rot, turns, amplitude);
  if (rc != LOGO_OK) return rc;
  LOGO_REQUIRE(rows != nullptr && n_rows >= 1 && n_rows <= 4, "one to four tensors");
  LOGO_REQUIRE(position_bits == 32 || position_bits == 64, "positions must be int32 or int64");
  LOGO_REQUIRE(n_tokens >= 0 && n_tokens < ((int64_t)1 << 31) && tokens_per_batch >= 1, "bad token counts");
  if (n_tokens == 0) return LOGO_OK;
  LOGO_REQUIRE(positions != nullptr, "null positions");
  RotArgs a{};
  bool inplace = true;
  for (int i = 0; i < n_rows; ++i) {
    const logo_rows& s = rows[i];
    LOGO_REQUIRE(s.x && s.y && s.heads >= 1, "tensor %d: null pointer or no heads", i);
    a.r[i] = RotRows{s.x, s.y, s.x_batch, s.x_token, s.x_head, s.y_batch, s.y_token, s.y_head, s.heads, 1, 1, true,
                     false};
    // in place, what passes through stays where it is
    inplace = inplace && s.x == s.y && s.x_batch == s.y_batch && s.x_token == s.y_token && s.x_head == s.y_head;
  }
  if (inplace && rot == 0) return LOGO_OK;
  a.positions = positions;
  a.pos64 = position_bits == 64;
  a.n = (uint32_t)n_tokens;
  a.per_batch = (uint32_t)std::min(tokens_per_batch, n_tokens);
  a.turns = turns;
  a.amp = amplitude;
  a.rot = rot;
  a.d = d;
  a.inter = interleaved != 0;
  a.inverse = inverse != 0;
  hipStream_t st = as_stream(stream);
  if (dtype == LOGO_DTYPE_BF16) return rot_dispatch<bf16, false>(a, n_rows, inplace, st);
  if (dtype == LOGO_DTYPE_F16) return rot_dispatch<f16, false>(a, n_rows, inplace, st);
  return rot_dispatch<float, false>(a, n_rows, inplace, st);
}

extern "C" int logo_paged_append(const logo_paged_cache* cache, const void* k, int64_t k_token, int64_t k_head,
                                 const void* v, int64_t v_token, int64_t v_head, const void* q, int64_t q_token,
                                 int64_t q_head, void* q_out, int hq, int64_t n_tokens, int d, const uint64_t* turns,
                                 int rot, int interleaved, float amplitude, int dtype, void* stream) {
  LOGO_REQUIRE(dtype == LOGO_DTYPE_BF16 || dtype == LOGO_DTYPE_F16, "only 16-bit tensors are supported");
  int rc = rot_check(d, rot, turns, amplitude);
  if (rc != LOGO_OK) return rc;
  rc = paged_check(cache, d);
  if (rc != LOGO_OK) return rc;
  LOGO_REQUIRE(n_tokens >= 0 && n_tokens < ((int64_t)1 << 31), "n_tokens must be in [0, 2^31)");
  LOGO_REQUIRE((q == nullptr) == (q_out == nullptr) && (q == nullptr || hq >= 1), "q needs an output and heads");
  if (n_tokens == 0 || cache->nseq == 0) return LOGO_OK;
  LOGO_REQUIRE(k && v, "null pointer argument");
  const logo_paged_cache& c = *cache;
  RotArgs a{};
  a.r[0] = RotRows{k, c.k, 0, k_token, k_head, c.k_page, c.k_slot, c.k_head, c.heads, 1, 1, rot > 0, true};
  a.r[1] = RotRows{v, c.v, 0, v_token, v_head, c.v_page, c.v_slot, c.v_head, c.heads, 1, 1, false, true};
  a.r[2] = RotRows{q, q_out, 0, q_token, q_head, 0, (int64_t)hq * d, d, hq, 1, 1, rot > 0, false};
  a.n = a.per_batch = (uint32_t)n_tokens;
  a.turns = turns;
  a.amp = amplitude;
  a.rot = rot;
  a.d = d;
  a.inter = interleaved != 0;
  a.table = c.table;
  a.table_row = c.table_row;
  a.table_width = c.table_width;
  a.page_shift = __builtin_ctz((unsigned)c.page_size);
  a.nseq = c.nseq;
  a.pages = c.pages;
  a.cu = c.cu;
  a.lens = c.lens;
  const int nr = q != nullptr ? 3 : 2;
  hipStream_t st = as_stream(stream);
  if (dtype == LOGO_DTYPE_BF16) return rot_dispatch<bf16, true>(a, nr, false, st);
  return rot_dispatch<f16, true>(a, nr, false, st);
}
