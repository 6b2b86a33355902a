// Attention of new tokens over a paged key / value cache for gfx950.
//
// Sequence b has n_b new tokens (rows cu[b] .. cu[b + 1] - 1 of q) whose keys are
// the last n_b of its lens[b] cached ones: token i sits at p = lens[b] - n_b + i and
//   o = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q.k_j),  p - window <= j <= p.
// One pass over the keys with a running maximum m: l <- l e^(m - m') + sum w,
// O <- O e^(m - m') + sum w v, in fp32.  Key j of kv head h is slot j % page_size
// of page table[b, j / page_size].
//
// A key that a row does not see has weight zero, but zero times infinity or NaN is
// NaN.  Where a tile crosses the edge of some row's keys, its values are therefore
// tested, and if one is not finite they enter the product as zeros and only the
// rows that see such a key get NaN (paged_tile_finite, paged_pv_guarded).
//
// Tiles.  A tile of keys is copied to LDS by buffer_load ... lds in groups of 16
// keys: a page holds a multiple of 16, so a group's rows lie in one page and share
// one buffer descriptor, whose base is the 64-bit address of the rows and whose
// extent ends behind the group's last valid key.  Keys behind it read as zeros
// (whatever the page holds there, NaN included), as does a group whose table
// entry names no page.
#include <math.h>

#include <algorithm>

#include "capi.hpp"
#include "common.hpp"
#include "paged.hpp"

namespace logo {

struct PagedArgs {
  logo_paged_cache c;
  const bf16* q;
  int64_t q_token, q_head;
  bf16* out;             // [n, hq, D]
  const uint8_t* sel;    // [n] or null: every token
  float* part;           // [n, hq, npiece, D + 2]
  int64_t n;
  int hq, g, shift, npiece, chunk, window;
  float scale_log2;
  bool zero_rest;
};

constexpr int kPagedPad = 4;  // floats between the rows of an LDS block of partial outputs

// The rows of sequence b.
struct PagedSeq {
  int64_t lo;   // first token
  int nq, len;  // new tokens, keys
  __device__ __forceinline__ PagedSeq(const PagedArgs& a, int b) {
    lo = max(0, a.c.cu[b]);
    nq = (int)(min((int64_t)a.c.cu[b + 1], a.n) - lo);
    len = min(max(a.c.lens[b], 0), a.c.table_width << a.shift);
  }
};

// Keys [lo, hi) that positions [pmin, pmax] see of piece pc.
__device__ __forceinline__ void paged_range(const PagedArgs& a, int len, int pmin, int pmax, int pc, int& lo, int& hi) {
  lo = a.window >= 0 ? max(0, pmin - a.window) : 0;
  hi = min(len, pmax + 1);
  if (a.npiece > 1) {
    lo = max(lo, pc * a.chunk);
    if (pc < a.npiece - 1) hi = min(hi, (pc + 1) * a.chunk);
  }
}

// Page ids of a sequence by its wave: lane l holds entry first + l.
struct PagedIds {
  const int32_t* row;
  int width, first, id;
  int64_t pages;
  __device__ __forceinline__ void init(const PagedArgs& a, int b) {
    row = a.c.table + (int64_t)b * a.c.table_row;
    width = a.c.table_width;
    pages = a.c.pages;
    first = -64;
    id = -1;
  }
  // Entry e (wave-uniform), -1 where it names no page.
  __device__ __forceinline__ int get(int e) {
    if (e < first || e >= first + 64) {
      first = e;
      const int at = e + (int)(threadIdx.x & 63);
      id = at < width ? row[at] : -1;
      if (id >= pages) id = -1;
    }
    return max(__builtin_amdgcn_readlane(id, e - first), -1);
  }
};

// Copies of 16-key groups of one kv head's rows into a kSwz tile.
template <int D>
struct PagedDma {
  static constexpr int CH = D / 8, RPB = 64 / CH, BLOCKS = 16 / RPB;
  using Geo = TileGeom<D, kSwz>;
  const bf16* base;
  int64_t page_stride;
  int slot_stride;
  uint32_t o[BLOCKS];
  __device__ __forceinline__ void init(const void* pages, int64_t page, int64_t head, int64_t slot, int h) {
    base = static_cast<const bf16*>(pages) + h * head;
    page_stride = page;
    slot_stride = (int)slot;
    const int j = threadIdx.x & 63;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      const int row = RPB * b + j / CH;  // the swizzle has period 16
      o[b] = (uint32_t)(row * slot_stride + 8 * ((j % CH) ^ Geo::swz(row))) * 2u;
    }
  }
  // `rows` valid rows (at most 16; none: zeros) from slot `slot` of page `page` to tile rows 0 .. 15 of dst
  __device__ __forceinline__ void issue(bf16* dst, int page, int slot, int rows) const {
    const bf16* p = base + (int64_t)max(page, 0) * page_stride + (int64_t)slot * slot_stride;
    const int bytes = rows > 0 && page >= 0 ? ((min(rows, 16) - 1) * slot_stride + D) * 2 : 0;
    const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16*>(p), (short)0, bytes, kBufRsrcWord3);
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) buf_load_lds16(r, dst + RPB * b * D, o[b]);
  }
};

// Whether all values of `steps` 16-key steps of a V tile are finite: their products
// with zero, which are NaN for the others, summed by the matrix unit.
template <typename EL, int D, int STEPS>
__device__ __forceinline__ bool paged_tile_finite(const TileReader<D, kSwz>& rd, const bf16* vt) {
  using E8 = typename Elem<EL>::x8;
  f32x16 z = f32x16{};
#pragma unroll
  for (int ks = 0; ks < STEPS; ++ks)
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) z = mfma32(rd.template tr<EL>(vt, 16 * ks, dt), E8{}, z);
  float t = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) t += z[e];
  return __ballot(t != t) == 0;
}

// O += V^T P over one 16-key step whose values may be infinite or NaN: those count
// as zero, and elements of rows that see one become NaN.  seen: bit e, whether the
// row sees the lane's key e of the step.
template <typename EL, int D>
__device__ __forceinline__ void paged_pv_guarded(f32x16 (&oacc)[D / 32], const TileReader<D, kSwz>& rd, const bf16* vt,
                                                 int ks, const typename Elem<EL>::x8 pb, uint32_t seen) {
  using E8 = typename Elem<EL>::x8;
  E8 sees;
#pragma unroll
  for (int e = 0; e < 8; ++e) sees[e] = (EL)(seen >> e & 1 ? 1.f : 0.f);
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt) {
    const E8 v = rd.template tr<EL>(vt, 16 * ks, dt);
    E8 fin, odd;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool ok = fabsf((float)v[e]) < INFINITY;
      fin[e] = ok ? v[e] : (EL)0.f;
      odd[e] = (EL)(ok ? 0.f : 1.f);
    }
    oacc[dt] = mfma32(fin, pb, oacc[dt]);
    const f32x16 bad = mfma32(odd, sees, f32x16{});
#pragma unroll
    for (int e = 0; e < 16; ++e) oacc[dt][e] = bad[e] > 0.f ? __builtin_nanf("") : oacc[dt][e];
  }
}

// ---------------------------------------------------------------------------
// Few rows
// ---------------------------------------------------------------------------
// A workgroup takes one piece of a sequence's keys for one kv head; its rows are
// (token, query head of the group) pairs, 32 at a time.  The four waves split the
// keys in tiles of 32, each with a double-buffered K and V tile of its own and no
// barrier in the loop, and join at the end through LDS.
constexpr int kFewWaves = 4;

template <int D>
constexpr size_t few_smem() { return (size_t)kFewWaves * 2 * 2 * 32 * D * sizeof(bf16); }

template <typename EL, int D>
__global__ __launch_bounds__(64 * kFewWaves) __attribute__((amdgpu_waves_per_eu(1, 1)))
void paged_few_kernel(const PagedArgs a) {
  using E8 = typename Elem<EL>::x8;
  constexpr int DS = D / 16, DT = D / 32, TILE = 32 * D, NISSUE = 2 * 2 * PagedDma<D>::BLOCKS;
  constexpr int ORS = D + kPagedPad;
  extern __shared__ __attribute__((aligned(16))) char paged_smem[];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, i = l & 31, g = l >> 5;
  const int pc = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  if (b == a.c.nseq) {
    // tokens of no sequence: zero rows of this kv head's group
    const int64_t end = max(0, a.c.nseq > 0 ? a.c.cu[a.c.nseq] : 0), begin = a.c.nseq > 0 ? a.c.cu[0] : 0;
    for (int64_t n = pc; n < a.n; n += gridDim.x) {
      if (n >= begin && n < end) continue;
      for (int e = tid; e < a.g * D / 8; e += 64 * kFewWaves)
        reinterpret_cast<u32x4*>(a.out + (n * a.hq + h * a.g) * D)[e] = u32x4{};
    }
    return;
  }
  const PagedSeq s(a, b);
  const int rows = s.nq * a.g, pos0 = s.len - s.nq;
  PagedIds ids;
  ids.init(a, b);
  PagedDma<D> dk, dv;
  dk.init(a.c.k, a.c.k_page, a.c.k_head, a.c.k_slot, h);
  dv.init(a.c.v, a.c.v_page, a.c.v_head, a.c.v_slot, h);
  TileReader<D, kSwz> rd;
  rd.init();
  bf16* const tiles = reinterpret_cast<bf16*>(paged_smem) + wave * 4 * TILE;  // [stage][K, V]
  float* const so = reinterpret_cast<float*>(paged_smem);                     // [wave][32][ORS]
  __shared__ float sm[kFewWaves][32], sl[kFewWaves][32];
  const float c = a.scale_log2;

  for (int r0 = 0; r0 < rows; r0 += 32) {
    const int r = r0 + i, tok = min(r, rows - 1) / a.g;
    const bool valid = r < rows && (a.sel == nullptr || a.sel[s.lo + tok] != 0);
    const int p = valid ? pos0 + tok : -1;
    // the row block's positions (rows ascend by token)
    const int pmin = pos0 + r0 / a.g, pmax = pos0 + (min(r0 + 32, rows) - 1) / a.g;
    int lo, hi;
    paged_range(a, s.len, pmin, pmax, pc, lo, hi);
    const bool any = __ballot(valid && p >= 0) != 0;
    E8 qreg[DS];
    {
      const bf16* const qrow = a.q + (s.lo + tok) * a.q_token + (h * a.g + (min(r, rows - 1) - tok * a.g)) * a.q_head + 8 * g;
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) qreg[ds] = valid ? *reinterpret_cast<const E8*>(qrow + 16 * ds) : E8{};
    }
    f32x16 oacc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) oacc[dt] = f32x16{};
    float m_run = -INFINITY, l_run = 0.f;
    const int first = (lo & ~31) + 32 * wave;
    const int nt = any && first < hi ? (hi - first + 32 * kFewWaves - 1) / (32 * kFewWaves) : 0;
    uint32_t held = 0;  // bits 2 k, 2 k + 1: the groups of the tile in stage k have a page
    auto issue = [&](int t) {
      const int j0 = first + 32 * kFewWaves * t;
      bf16* const kt = tiles + (t & 1) * 2 * TILE;
      held &= ~(3u << (2 * (t & 1)));
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = j0 + 16 * u, rem = s.len - j;
        const int page = rem > 0 ? ids.get(j >> a.shift) : -1, slot = j & ((1 << a.shift) - 1);
        if (page >= 0) held |= 1u << (2 * (t & 1) + u);
        dk.issue(kt + 16 * u * D, page, slot, rem);
        dv.issue(kt + TILE + 16 * u * D, page, slot, rem);
      }
    };
    if (nt > 0) issue(0);
    for (int t = 0; t < nt; ++t) {
      if (t + 1 < nt) {
        // the tile's last reads are done before its copies overwrite it
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        issue(t + 1);
        asm volatile("s_waitcnt vmcnt(%0)" ::"i"(NISSUE) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      const int j0 = first + 32 * kFewWaves * t;
      const bf16* const kt = tiles + (t & 1) * 2 * TILE;
      const uint32_t has = held >> (2 * (t & 1)) & 3;
      f32x16 sc = f32x16{};
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) sc = mfma32(rd.template row<EL>(kt, 0, ds), qreg[ds], sc);
      float mx = -INFINITY;
      uint32_t seen = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = j0 + rowmap(g, e);
        const bool vis = key <= p && (a.window < 0 || key >= p - a.window) && (has >> (e >> 3) & 1);
        seen |= vis ? 1u << e : 0u;
        sc[e] = vis ? sc[e] * c : -INFINITY;
        mx = fmaxf(mx, sc[e]);
      }
      const float m_new = fmaxf(m_run, pair_max(mx));
      const float base = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = fast_exp2(m_run - base);
      m_run = m_new;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        sc[e] = fast_exp2(sc[e] - base);
        sum += sc[e];
      }
      l_run = l_run * alpha + sum;
      if (__ballot(alpha != 1.f)) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) oacc[dt] *= alpha;
      }
      // rows past the block's last (p = -1) see nothing and are not written
      const bool edge = __ballot(p >= 0 && seen != 0xffffu) != 0;
      if (edge && !paged_tile_finite<EL, D, 2>(rd, kt + TILE)) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
          paged_pv_guarded<EL, D>(oacc, rd, kt + TILE, ks, acc_to<EL>(sc, ks), seen >> (8 * ks));
      } else {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const E8 pb = acc_to<EL>(sc, ks);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
            oacc[dt] = mfma32(rd.template tr<EL>(kt + TILE, 16 * ks, dt), pb, oacc[dt]);
        }
      }
    }
    // join the waves
    const float l_tot = pair_sum(l_run);
    __syncthreads();  // every wave is done with its tiles (and with the block before)
    {
      float* const orow = so + (wave * 32 + i) * ORS;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = oacc[dt][4 * q4 + e];
          *reinterpret_cast<f32x4*>(orow + 32 * dt + 8 * q4 + 4 * g) = v;
        }
      if (g == 0) sm[wave][i] = m_run, sl[wave][i] = l_tot;
    }
    __syncthreads();
    constexpr int CH = D / 8;
    for (int e = tid; e < 32 * CH; e += 64 * kFewWaves) {
      const int rr = e / CH, ch = e % CH;
      if (r0 + rr >= rows) break;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) m = fmaxf(m, sm[w][rr]);
      const float base = m == -INFINITY ? 0.f : m;
      float lsum = 0.f, o[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = 0.f;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) {
        const float f = fast_exp2(sm[w][rr] - base);
        lsum = fmaf(f, sl[w][rr], lsum);
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = fmaf(f, so[(w * 32 + rr) * ORS + 8 * ch + k], o[k]);
      }
      const int tk = (r0 + rr) / a.g;
      const int64_t row = (s.lo + tk) * a.hq + h * a.g + (r0 + rr - tk * a.g);
      if (a.npiece == 1) {
        const float inv = lsum != 0.f ? 1.f / lsum : 0.f;
        E8 v;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (EL)(lsum != 0.f ? o[k] * inv : 0.f);
        *reinterpret_cast<E8*>(a.out + row * D + 8 * ch) = v;
      } else {
        float* const pp = a.part + (row * a.npiece + pc) * (D + 2);
#pragma unroll
        for (int k = 0; k < 8; ++k) pp[8 * ch + k] = o[k];
        if (ch == 0) pp[D] = m, pp[D + 1] = lsum;
      }
    }
    __syncthreads();
  }
}

// Joins the pieces of a row: one workgroup a (token, query head).
template <typename EL, int D>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedArgs a) {
  const int64_t row = blockIdx.x, n = row / a.hq;
  const int tid = threadIdx.x, l = tid & 63;
  int cnt = 0;
  for (int b0 = 0; b0 < a.c.nseq; b0 += 64) {
    const bool past = b0 + l < a.c.nseq && (int64_t)a.c.cu[b0 + l + 1] <= n;
    cnt += __builtin_popcountll(__ballot(past));
  }
  if (cnt == a.c.nseq || n < a.c.cu[cnt]) {
    if (a.zero_rest && tid < D / 8) reinterpret_cast<u32x4*>(a.out + row * D)[tid] = u32x4{};
    return;
  }
  const PagedSeq s(a, cnt);
  const int p = s.len - s.nq + (int)(n - s.lo);
  const bool valid = p >= 0 && (a.sel == nullptr || a.sel[n] != 0);
  // the pieces that hold keys which the row sees
  const int lo = a.window >= 0 ? max(0, p - a.window) : 0;
  const int p0 = min(lo / a.chunk, a.npiece - 1), p1 = valid ? min(p / a.chunk, a.npiece - 1) + 1 : p0;
  constexpr int CH = D / 4, GR = 256 / CH;
  const int ch = tid % CH, gr = tid / CH;
  const float* const pp = a.part + row * a.npiece * (D + 2);
  __shared__ float red[4];
  __shared__ float so[GR][D + 4];
  float m = -INFINITY;
  for (int k = p0 + tid; k < p1; k += 256) m = fmaxf(m, pp[(int64_t)k * (D + 2) + D]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
  if (l == 0) red[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float base = m == -INFINITY ? 0.f : m;
  f32x4 o = f32x4{};
  float ls = 0.f;
  for (int k = p0 + gr; k < p1; k += GR) {
    const float* const q = pp + (int64_t)k * (D + 2);
    const float f = fast_exp2(q[D] - base);
    ls = fmaf(f, q[D + 1], ls);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(f, q[4 * ch + e], o[e]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) so[gr][4 * ch + e] = o[e];
  if (ch == 0) so[gr][D] = ls;
  __syncthreads();
  if (tid < D) {
    float v = 0.f, sum = 0.f;
#pragma unroll
    for (int k = 0; k < GR; ++k) v += so[k][tid], sum += so[k][D];
    reinterpret_cast<EL*>(a.out)[row * D + tid] = (EL)(sum != 0.f ? v / sum : 0.f);
  }
}

// How the keys are cut: pieces per sequence and keys per piece (a multiple of 128).
static void paged_pieces(int nseq, int h, int max_len, int window, int max_q, int& npiece, int& chunk) {
  const int64_t wgs = (int64_t)std::max(nseq, 1) * h;
  const int64_t span = window >= 0 ? std::min<int64_t>(max_len, (int64_t)window + max_q) : max_len;
  int64_t want = std::min<int64_t>((1024 + wgs - 1) / wgs, (span + 255) / 256);
  if (window >= 0) want = 1;  // a window's keys are few
  want = std::max<int64_t>(want, 1);
  const int64_t per = std::max<int64_t>((max_len + want - 1) / want, 1);
  chunk = (int)std::min<int64_t>((per + 127) & ~(int64_t)127, (int64_t)1 << 30);
  npiece = std::max(1, (max_len + chunk - 1) / chunk);
}

template <typename EL, int D>
static int paged_launch(const PagedArgs& a, int h, hipStream_t st) {
  auto few = paged_few_kernel<EL, D>;
  LOGO_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(few), hipFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)few_smem<D>()));
  const bool rest = a.npiece == 1 && a.zero_rest;
  hipLaunchKernelGGL(few, dim3(a.npiece, h, a.c.nseq + (rest ? 1 : 0)), dim3(64 * kFewWaves), few_smem<D>(), st, a);
  LOGO_LAUNCH_CHECK("paged_few_kernel");
  if (a.npiece > 1) {
    hipLaunchKernelGGL((paged_join_kernel<EL, D>), dim3((unsigned)(a.n * a.hq)), dim3(256), 0, st, a);
    LOGO_LAUNCH_CHECK("paged_join_kernel");
  }
  return LOGO_OK;
}

}  // namespace logo

using namespace logo;

extern "C" size_t logo_paged_attn_workspace_bytes(int nseq, int h, int hq, int64_t n_tokens, int d, int max_q,
                                                  int max_len, int window) {
  if (nseq < 1 || h < 1 || hq < 1 || n_tokens < 1 || max_len < 1) return 0;
  int npiece, chunk;
  paged_pieces(nseq, h, max_len, window, max_q, npiece, chunk);
  return npiece > 1 ? (size_t)n_tokens * hq * npiece * (d + 2) * sizeof(float) : 0;
}

extern "C" int logo_paged_attn(const logo_paged_cache* cache, const void* q, int64_t q_token, int64_t q_head, void* out,
                               const uint8_t* selection, int hq, int64_t n_tokens, int d, int max_q, int max_len,
                               float scale, int window, int zero_rest, void* workspace, size_t workspace_bytes,
                               int dtype, void* stream) {
  LOGO_REQUIRE(dtype == LOGO_DTYPE_BF16 || dtype == LOGO_DTYPE_F16, "only 16-bit tensors are supported");
  const int rc = paged_check(cache, d);
  if (rc != LOGO_OK) return rc;
  const int h = cache->heads;
  LOGO_REQUIRE(hq >= 1 && hq % h == 0, "query heads (%d) must be a multiple of the cache's heads (%d)", hq, h);
  LOGO_REQUIRE(cache->nseq <= 65534, "at most 65534 sequences");
  LOGO_REQUIRE(n_tokens >= 0 && n_tokens * hq < ((int64_t)1 << 31), "too many query rows");
  LOGO_REQUIRE(max_q >= 0 && max_len >= 0 && window >= -1, "bad max_q, max_len or window");
  LOGO_REQUIRE(scale > 0.f && isfinite(scale), "scale must be positive and finite");
  LOGO_REQUIRE(q_token % 8 == 0 && q_head % 8 == 0 && ((uintptr_t)q | (uintptr_t)out) % 16 == 0,
               "q and out rows must be 16-byte aligned");
  if (n_tokens == 0 || (cache->nseq == 0 && !zero_rest)) return LOGO_OK;
  LOGO_REQUIRE(q && out, "null pointer argument");
  PagedArgs a{};
  a.c = *cache;
  a.q = static_cast<const bf16*>(q);
  a.q_token = q_token;
  a.q_head = q_head;
  a.out = static_cast<bf16*>(out);
  a.sel = selection;
  a.n = n_tokens;
  a.hq = hq;
  a.g = hq / h;
  a.shift = __builtin_ctz((unsigned)cache->page_size);
  a.window = window;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.zero_rest = zero_rest != 0;
  paged_pieces(a.c.nseq, h, std::max(1, max_len), window, max_q, a.npiece, a.chunk);
  const size_t need = logo_paged_attn_workspace_bytes(a.c.nseq, h, hq, n_tokens, d, max_q, max_len, window);
  LOGO_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), "the workspace is too small");
  a.part = static_cast<float*>(workspace);
  hipStream_t st = as_stream(stream);
  if (dtype == LOGO_DTYPE_BF16) return d == 128 ? paged_launch<bf16, 128>(a, h, st) : paged_launch<bf16, 64>(a, h, st);
  return d == 128 ? paged_launch<f16, 128>(a, h, st) : paged_launch<f16, 64>(a, h, st);
}
