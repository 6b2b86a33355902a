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
  const int b = paged_seq_of(a.c.cu, a.c.nseq, n);
  if (b == a.c.nseq || n < a.c.cu[b]) {
    if (a.zero_rest && tid < D / 8) reinterpret_cast<u32x4*>(a.out + row * D)[tid] = u32x4{};
    return;
  }
  const PagedSeq s(a, b);
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

// Whether a call's rows go 32 at a time through the kernel for few rows: where no
// sequence has more (by the caller's bound; others stay right, 32 after 32).
static bool paged_few(int max_q, int g) { return (int64_t)max_q * g <= 32; }

// How the keys are cut: pieces per sequence and keys per piece (a multiple of 128).
struct PagedPlan {
  bool few;
  int npiece, chunk;
  size_t part_bytes, bytes;
};

static PagedPlan paged_plan(int nseq, int h, int hq, int64_t n, int d, int max_q, int max_len, int window, bool sel) {
  PagedPlan p{};
  const int g = hq / h;
  p.few = paged_few(max_q, g);
  max_len = std::max(max_len, 1);
  int64_t want = 1;
  if (window < 0) {  // a window's keys are few
    const int64_t wgs = (p.few ? (int64_t)nseq : n * g / kTileRows + nseq) * h;
    if (p.few) want = std::min<int64_t>((1024 + wgs - 1) / wgs, (max_len + 255) / 256);
    else if (wgs < 384) want = std::min<int64_t>((1024 + wgs - 1) / wgs, (max_len + 511) / 512);
  }
  const int64_t per = (max_len + want - 1) / want;
  p.chunk = (int)std::min<int64_t>((per + 127) & ~(int64_t)127, (int64_t)1 << 30);
  p.npiece = (max_len + p.chunk - 1) / p.chunk;
  if (p.npiece > 1) p.part_bytes = ((size_t)n * hq * p.npiece * (d + 2) * sizeof(float) + 255) & ~(size_t)255;
  p.bytes = p.part_bytes + (sel && !p.few ? ((size_t)n + nseq) * sizeof(int32_t) : 0);
  return p;
}

template <typename EL, int D>
static int paged_launch(const PagedArgs& a, bool few, int h, hipStream_t st) {
  if (few) {
    auto kern = paged_few_kernel<EL, D>;
    LOGO_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kern),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)few_smem<D>()));
    const bool rest = a.npiece == 1 && a.zero_rest;
    hipLaunchKernelGGL(kern, dim3(a.npiece, h, a.c.nseq + (rest ? 1 : 0)), dim3(64 * kFewWaves), few_smem<D>(), st, a);
    LOGO_LAUNCH_CHECK("paged_few_kernel");
  } else {
    const int rc = paged_launch_tile(a, h, D, Elem<EL>::kHalf, st);
    if (rc != LOGO_OK) return rc;
  }
  if (a.npiece > 1) {
    hipLaunchKernelGGL((paged_join_kernel<EL, D>), dim3((unsigned)(a.n * a.hq)), dim3(256), 0, st, a);
    LOGO_LAUNCH_CHECK("paged_join_kernel");
  }
  return LOGO_OK;
}

}  // namespace logo

using namespace logo;

extern "C" size_t logo_paged_attn_workspace_bytes(int nseq, int h, int hq, int64_t n_tokens, int d, int max_q,
                                                  int max_len, int window, int selected) {
  if (nseq < 1 || h < 1 || hq < h || n_tokens < 1) return 0;
  return paged_plan(nseq, h, hq, n_tokens, d, max_q, max_len, window, selected != 0).bytes;
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
  const PagedPlan plan = paged_plan(std::max(a.c.nseq, 1), h, hq, n_tokens, d, max_q, max_len, window, selection != nullptr);
  LOGO_REQUIRE(a.c.nseq == 0 || plan.bytes == 0 || (workspace != nullptr && workspace_bytes >= plan.bytes),
               "the workspace is too small");
  a.npiece = a.c.nseq == 0 ? 1 : plan.npiece;
  a.chunk = plan.chunk;
  a.part = static_cast<float*>(workspace);
  a.idx = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + plan.part_bytes);
  a.count = a.idx + n_tokens;
  const bool few = plan.few || a.c.nseq == 0;
  hipStream_t st = as_stream(stream);
  if (dtype == LOGO_DTYPE_BF16) return d == 128 ? paged_launch<bf16, 128>(a, few, h, st) : paged_launch<bf16, 64>(a, few, h, st);
  return d == 128 ? paged_launch<f16, 128>(a, few, h, st) : paged_launch<f16, 64>(a, few, h, st);
}
