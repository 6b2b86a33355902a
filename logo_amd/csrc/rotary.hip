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
// and serve all heads.
#include <math.h>

#include <algorithm>

#include "capi.hpp"
#include "common.hpp"
#include "paged.hpp"

namespace logo {

constexpr int kRotThreads = 256;
constexpr int kRotMaxTok = 16;     // tokens per workgroup
constexpr int kRotItems = 1024;    // items (row chunks) a workgroup aims for
constexpr int kRotMaxDim = 512;

struct RotRows {
  const void* x;
  void* y;
  int64_t x_batch, x_token, x_head;  // strides in elements
  int64_t y_batch, y_token, y_head;  // (paged rows: page, slot, head)
  int heads;
  int tok, hc;                       // tokens and heads per workgroup
  uint32_t hc_magic;                 // ceil(2^32 / hc)
  bool rotate, paged;
};

struct RotArgs {
  RotRows r[4];
  const void* positions;  // int32 or int64 [n] (rotary), else null
  bool pos64;
  int64_t n, per_batch;   // tokens; tokens per batch entry
  const uint64_t* turns;  // [rot / 2]
  float amp;
  int rot, d, units, pair_units;  // units: items per row, of which pair_units rotate
  uint32_t units_magic;
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
  int64_t x_off;  // batch and token part of the source row's offset
  int64_t y_off;  // of the destination row's; paged: of the page and slot
  int state;      // 0: written; 1: zero row (no position); 2: nothing to write
};

template <typename T, int VEC, bool APPEND>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(const RotArgs a) {
  typedef T vec __attribute__((ext_vector_type(VEC)));
  const RotRows& r = a.r[blockIdx.z];
  const int64_t n0 = (int64_t)blockIdx.x * r.tok;
  const int h0 = blockIdx.y * r.hc;
  if (n0 >= a.n || h0 >= r.heads) return;
  const int ntok = (int)min((int64_t)r.tok, a.n - n0), tid = threadIdx.x;
  extern __shared__ __attribute__((aligned(16))) char rot_smem[];
  RotTok* const info = reinterpret_cast<RotTok*>(rot_smem);                      // [kRotMaxTok]
  float2* const cs = reinterpret_cast<float2*>(rot_smem + kRotMaxTok * sizeof(RotTok));  // [ntok][rot / 2]
  if constexpr (APPEND) {
    for (int t = tid >> 6; t < ntok; t += kRotThreads / 64) {
      const int64_t n = n0 + t;
      const int b = paged_seq_of(a.cu, a.nseq, n);
      RotTok k{0, n * r.x_token, n * r.y_token, 1};
      if (b < a.nseq) {
        const int lo = a.cu[b], hi = a.cu[b + 1];
        k.pos = (int64_t)a.lens[b] - hi + n;
        if (n >= lo && k.pos >= 0) k.state = 0;
      }
      if (r.paged) {
        const int64_t col = k.pos >> a.page_shift;
        int page = -1;
        if (k.state == 0 && col < a.table_width) page = a.table[b * a.table_row + col];
        const bool held = page >= 0 && page < a.pages;
        k.y_off = held ? page * r.y_batch + (k.pos & ((1 << a.page_shift) - 1)) * r.y_token : 0;
        if (!held) k.state = 2;
      }
      if ((tid & 63) == 0) info[t] = k;
    }
  } else {
    if (tid < ntok) {
      const int64_t n = n0 + tid, b = n / a.per_batch, t = n - b * a.per_batch;
      const int64_t p = a.pos64 ? static_cast<const int64_t*>(a.positions)[n] : static_cast<const int32_t*>(a.positions)[n];
      info[tid] = RotTok{p, b * r.x_batch + t * r.x_token, b * r.y_batch + t * r.y_token, 0};
    }
  }
  __syncthreads();
  const int half = a.rot >> 1;
  if (r.rotate) {
    for (int t = 0; t < ntok; ++t)
      for (int i = tid; i < half; i += kRotThreads) {
        float2 v = turn_cos_sin((uint64_t)info[t].pos * a.turns[i]);
        v.x *= a.amp;
        v.y *= a.inverse ? -a.amp : a.amp;
        cs[t * half + i] = v;
      }
    __syncthreads();
  }
  const int nh = min(r.hc, r.heads - h0);
  const int items = ntok * r.hc * a.units;
  const T* const x = static_cast<const T*>(r.x);
  T* const y = static_cast<T*>(r.y);
  for (int idx = tid; idx < items; idx += kRotThreads) {
    const int row = a.units == 1 ? idx : (int)__umulhi((uint32_t)idx, a.units_magic);
    const int u = idx - row * a.units;
    const int t = r.hc == 1 ? row : (int)__umulhi((uint32_t)row, r.hc_magic);
    const int h = row - t * r.hc;
    if (h >= nh) continue;
    const RotTok k = info[t];
    if (k.state == 2) continue;
    const T* const xr = x + k.x_off + (int64_t)(h0 + h) * r.x_head;
    T* const yr = y + k.y_off + (int64_t)(h0 + h) * r.y_head;
    if (u < a.pair_units) {
      const int e0 = a.inter ? 2 * VEC * u : VEC * u, e1 = a.inter ? e0 + VEC : half + VEC * u;
      vec v0 = *reinterpret_cast<const vec*>(xr + e0), v1 = *reinterpret_cast<const vec*>(xr + e1);
      if (r.rotate) {
        const float2* const c = cs + t * half + VEC * u;
        T in[2 * VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) in[e] = v0[e], in[VEC + e] = v1[e];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int ia = a.inter ? 2 * e : e, ib = a.inter ? 2 * e + 1 : VEC + e;
          const float p = (float)in[ia], q = (float)in[ib];
          in[ia] = (T)(p * c[e].x - q * c[e].y);
          in[ib] = (T)(q * c[e].x + p * c[e].y);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) v0[e] = in[e], v1[e] = in[VEC + e];
      }
      if (k.state == 1) v0 = vec{}, v1 = vec{};
      *reinterpret_cast<vec*>(yr + e0) = v0;
      *reinterpret_cast<vec*>(yr + e1) = v1;
    } else {
      const int e0 = a.rot + VEC * (u - a.pair_units);
      vec v0 = *reinterpret_cast<const vec*>(xr + e0);
      if (k.state == 1) v0 = vec{};
      *reinterpret_cast<vec*>(yr + e0) = v0;
    }
  }
}

static uint32_t magic_of(int d) { return (uint32_t)((((uint64_t)1 << 32) + d - 1) / d); }

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
  a.units_magic = magic_of(a.units);
  int64_t gx = 1;
  int gy = 1, tok = 1;
  for (int i = 0; i < nr; ++i) {
    RotRows& r = a.r[i];
    r.hc = std::min(r.heads, std::max(1, kRotItems / a.units));
    r.hc_magic = magic_of(r.hc);
    r.tok = std::max(1, std::min(kRotMaxTok, kRotItems / (r.hc * a.units)));
    gx = std::max(gx, (a.n + r.tok - 1) / r.tok);
    gy = std::max(gy, (r.heads + r.hc - 1) / r.hc);
    tok = std::max(tok, r.tok);
  }
  LOGO_REQUIRE(gx < ((int64_t)1 << 31) && gy <= 65535, "too many tokens or heads");
  const size_t smem = kRotMaxTok * sizeof(RotTok) + (size_t)tok * (a.rot / 2) * sizeof(float2);
  hipLaunchKernelGGL((rotary_kernel<T, VEC, APPEND>), dim3((unsigned)gx, gy, nr), dim3(kRotThreads), smem, st, a);
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
  LOGO_REQUIRE(n_tokens >= 0 && tokens_per_batch >= 1, "bad token counts");
  if (n_tokens == 0) return LOGO_OK;
  LOGO_REQUIRE(positions != nullptr, "null positions");
  RotArgs a{};
  bool inplace = true;
  for (int i = 0; i < n_rows; ++i) {
    const logo_rows& s = rows[i];
    LOGO_REQUIRE(s.x && s.y && s.heads >= 1, "tensor %d: null pointer or no heads", i);
    a.r[i] = RotRows{s.x, s.y, s.x_batch, s.x_token, s.x_head, s.y_batch, s.y_token, s.y_head, s.heads, 1, 1, 0, true,
                     false};
    // in place, what passes through stays where it is
    inplace = inplace && s.x == s.y && s.x_batch == s.y_batch && s.x_token == s.y_token && s.x_head == s.y_head;
  }
  if (inplace && rot == 0) return LOGO_OK;
  a.positions = positions;
  a.pos64 = position_bits == 64;
  a.n = n_tokens;
  a.per_batch = tokens_per_batch;
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
  LOGO_REQUIRE(n_tokens >= 0, "n_tokens must be >= 0");
  LOGO_REQUIRE((q == nullptr) == (q_out == nullptr) && (q == nullptr || hq >= 1), "q needs an output and heads");
  if (n_tokens == 0 || cache->nseq == 0) return LOGO_OK;
  LOGO_REQUIRE(k && v, "null pointer argument");
  const logo_paged_cache& c = *cache;
  RotArgs a{};
  a.r[0] = RotRows{k, c.k, 0, k_token, k_head, c.k_page, c.k_slot, c.k_head, c.heads, 1, 1, 0, rot > 0, true};
  a.r[1] = RotRows{v, c.v, 0, v_token, v_head, c.v_page, c.v_slot, c.v_head, c.heads, 1, 1, 0, false, true};
  a.r[2] = RotRows{q, q_out, 0, q_token, q_head, 0, (int64_t)hq * d, d, hq, 1, 1, 0, rot > 0, false};
  a.n = n_tokens;
  a.per_batch = n_tokens;
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
