// Attention of chunks of new tokens over a paged cache: many rows share a tile of
// keys (the formulas and the layout of the cache: paged_attn.hip).
//
// A workgroup of four waves takes 128 rows of one sequence and kv head, (token,
// query head of the group) pairs in token order, 32 a wave, and walks the keys
// that they see in tiles of 64, K and V double-buffered in LDS.  Each wave copies one
// 16-key group of a tile.  S^T = K Q^T and O^T = V^T P^T on 32x32x16 MFMA, so a row's
// scores and outputs lie in one lane pair and its statistics need one exchange.
#include <algorithm>

#include "paged.hpp"

namespace logo {

constexpr int kTileWaves = kTileRows / 32;

template <int D>
constexpr size_t tile_smem() { return (size_t)4 * 64 * D * sizeof(bf16); }  // K and V, two of each

// Selected tokens of each sequence, in order: one workgroup a sequence, 16 tokens a
// thread and step.
constexpr int kSelThreads = 1024;
__global__ __launch_bounds__(kSelThreads) void paged_select_kernel(const PagedArgs a) {
  const int b = blockIdx.x, tid = threadIdx.x, l = tid & 63, wave = tid >> 6;
  const PagedSeq s(a, b);
  __shared__ int wsum[kSelThreads / 64];
  int done = 0;
  for (int t0 = 0; t0 < s.nq; t0 += 16 * kSelThreads) {
    const int t = t0 + 16 * tid;
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (t + e < s.nq && a.sel[s.lo + t + e] != 0) bits |= 1u << e;
    const int mine = __builtin_popcount(bits);
    int pre = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(pre, off);
      if (l >= off) pre += o;
    }
    if (l == 63) wsum[wave] = pre;
    __syncthreads();
    int at = done + pre - mine;
    for (int w = 0; w < kSelThreads / 64; ++w) {
      if (w < wave) at += wsum[w];
      done += wsum[w];
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (bits >> e & 1) a.idx[s.lo + at++] = t + e;
    __syncthreads();
  }
  if (tid == 0) a.count[b] = done;
}

// What a workgroup takes of the launch's (sequence, row tile, key piece) triples of
// one kv head: the rank-th of them.  By a whole wave.
struct TileWork {
  int b, tile, piece, rows;
  __device__ __forceinline__ bool find(const PagedArgs& a, int64_t rank) {
    const int lane = threadIdx.x & 63;
    for (int c = 0; c < a.c.nseq; c += 64) {
      int r = 0;
      if (c + lane < a.c.nseq) {
        const PagedSeq s(a, c + lane);
        r = max(0, a.sel ? a.count[c + lane] : s.nq) * a.g;
      }
      const int nt = (r + kTileRows - 1) / kTileRows * a.npiece;
      int pre = nt;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(pre, off);
        if (lane >= off) pre += o;
      }
      const unsigned long long past = __ballot(rank < pre);
      if (past != 0) {
        const int j = __builtin_ctzll(past);
        const int tiles = __shfl(nt, j);
        const int k = (int)rank - (__shfl(pre, j) - tiles);
        b = c + j;
        rows = __shfl(r, j);
        piece = k % a.npiece;
        tile = tiles / a.npiece - 1 - k / a.npiece;  // the latest rows, with the most keys, first
        return true;
      }
      rank -= __shfl(pre, 63);
    }
    return false;
  }
};

template <typename EL, int D, bool WINDOW>
__global__ __launch_bounds__(64 * kTileWaves) __attribute__((amdgpu_waves_per_eu(2, 2)))
void paged_tile_kernel(const PagedArgs a) {
  using E8 = typename Elem<EL>::x8;
  using E4 = typename Elem<EL>::x4;
  constexpr int NW = kTileWaves, DS = D / 16, DT = D / 32;
  using GT = TileGeom<D, kSwz>;
  extern __shared__ __attribute__((aligned(16))) char tile_mem[];
  bf16* const smem = reinterpret_cast<bf16*>(tile_mem);
  auto tileK = [&](int b) { return smem + b * GT::ELEMS; };
  auto tileV = [&](int b) { return smem + (2 + b) * GT::ELEMS; };
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, i = l & 31, g = l >> 5;
  int rank, h;
  xcd_remap(blockIdx.x, a.c.heads, rank, h);

  // zero rows: tokens that are not selected and those of no sequence, a slice of them a workgroup
  if (a.npiece == 1 && (a.sel != nullptr || a.zero_rest)) {
    const int slices = (int)(gridDim.x / a.c.heads), per = (int)((a.n + slices - 1) / slices);
    const int64_t n0 = (int64_t)rank * per, first = a.c.cu[0], end = a.c.cu[a.c.nseq];
    const int per_row = a.g * D / 8, cnt = (int)max((int64_t)0, min((int64_t)per, a.n - n0));
    // 16-byte chunks of the slice's rows, all lanes' tests in flight together
    for (int64_t e = tid; e < (int64_t)cnt * per_row; e += 64 * NW) {
      const int64_t n = n0 + e / per_row;
      const bool inside = n >= first && n < end;
      if (inside ? a.sel == nullptr || a.sel[n] != 0 : !a.zero_rest) continue;
      st_nt(reinterpret_cast<u32x4*>(a.out + (n * a.hq + h * a.g) * D) + e % per_row, u32x4{});
    }
  }
  TileWork w;
  if (!w.find(a, rank)) return;
  const PagedSeq s(a, w.b);
  const int r0 = w.tile * kTileRows, pos0 = s.len - s.nq;
  // token in the sequence of row r
  auto token = [&](int r) { return a.sel ? a.idx[s.lo + r / a.g] : r / a.g; };
  const int rl = min(r0 + kTileRows, w.rows) - 1;  // last row
  const int wr = r0 + 32 * wave, r = wr + i;
  const bool valid = r <= rl;
  const int tok = token(min(r, rl));
  const int p = valid ? pos0 + tok : -1;
  const bool active = wr <= rl;
  const int pmin = pos0 + __builtin_amdgcn_readfirstlane(token(min(wr, rl)));
  const int pmax = active ? pos0 + __builtin_amdgcn_readfirstlane(token(min(wr + 31, rl))) : -1;
  int kv_lo, kv_hi;
  paged_range(a, s.len, pos0 + __builtin_amdgcn_readfirstlane(token(r0)), pos0 + __builtin_amdgcn_readfirstlane(token(rl)),
              w.piece, kv_lo, kv_hi);
  kv_lo &= ~63;
  if (a.npiece > 1 && kv_lo >= kv_hi) return;
  const int W = a.window, nt = max(0, (kv_hi - kv_lo + 63) >> 6);
  const int hrow = min(r, rl) - min(r, rl) / a.g * a.g;  // query head in the group

  E8 qreg[DS];
  {
    const bf16* const qrow = a.q + (s.lo + tok) * a.q_token + (h * a.g + hrow) * a.q_head + 8 * g;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) qreg[ds] = valid ? *reinterpret_cast<const E8*>(qrow + 16 * ds) : E8{};
  }
  f32x16 oacc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) oacc[dt] = f32x16{};
  float m_run = -INFINITY, l_run = 0.f;
  const float c = a.scale_log2;

  TileReader<D, kSwz> rd;
  rd.init();
  PagedDma<D> dk, dv;
  dk.init(a.c.k, a.c.k_page, a.c.k_head, a.c.k_slot, h);
  dv.init(a.c.v, a.c.v_page, a.c.v_head, a.c.v_slot, h);
  PagedIds ids;
  ids.init(a, w.b);
  auto page_of = [&](int j) { return j < s.len ? ids.get(j >> a.shift) : -1; };
  auto load = [&](const PagedDma<D>& d, bf16* tile, int t) {
    const int j = kv_lo + 64 * t + 16 * wave;
    d.issue(tile + 16 * wave * D, page_of(j), j & ((1 << a.shift) - 1), s.len - j);
  };
  // the wave's tiles
  const int tw_hi = active ? min(nt, ((pmax - kv_lo) >> 6) + 1) : 0;
  const int tw_lo = WINDOW && active ? max(0, pmin - W - kv_lo) >> 6 : 0;
  if (nt > 0) load(dk, tileK(0), 0), load(dv, tileV(0), 0);
  for (int t = 0; t < nt; ++t) {
    if (t + 1 < nt) load(dk, tileK((t + 1) & 1), t + 1), load(dv, tileV((t + 1) & 1), t + 1);
    if (t + 1 < nt) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * PagedDma<D>::BLOCKS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t >= tw_lo && t < tw_hi) {
      const int j0 = kv_lo + 64 * t;
      const bf16 *kt = tileK(t & 1), *vt = tileV(t & 1);
      uint32_t has = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) has |= page_of(j0 + 16 * u) >= 0 ? 1u << u : 0u;
      f32x16 sc[2];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        sc[kk] = f32x16{};
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) sc[kk] = mfma32(rd.template row<EL>(kt, 32 * kk, ds), qreg[ds], sc[kk]);
      }
      uint32_t seen = 0;
      float mx = -INFINITY;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = j0 + 32 * kk + rowmap(g, e);
          const bool vis = key <= p && (!WINDOW || key >= p - W) && (has >> (2 * kk + e / 8) & 1);
          seen |= vis ? 1u << (16 * kk + e) : 0u;
          sc[kk][e] = vis ? sc[kk][e] * c : -INFINITY;
          mx = fmaxf(mx, sc[kk][e]);
        }
      const float m_new = fmaxf(m_run, pair_max(mx));
      const float base = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = fast_exp2(m_run - base);
      m_run = m_new;
      float sum = 0.f;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          sc[kk][e] = fast_exp2(sc[kk][e] - base);
          sum += sc[kk][e];
        }
      l_run = l_run * alpha + sum;
      if (__ballot(alpha != 1.f)) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) oacc[dt] *= alpha;
      }
      if (__ballot(p >= 0 && seen != 0xffffffffu) != 0 && !paged_tile_finite<EL, D, 4>(rd, vt)) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          paged_pv_guarded<EL, D>(oacc, rd, vt, ks, acc_to<EL>(sc[ks / 2], ks & 1), seen >> (8 * ks));
      } else {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const E8 pb = acc_to<EL>(sc[ks / 2], ks & 1);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) oacc[dt] = mfma32(rd.template tr<EL>(vt, 16 * ks, dt), pb, oacc[dt]);
        }
      }
    }
    __syncthreads();
  }
  const float l_tot = pair_sum(l_run);
  if (a.npiece > 1) {
    if (valid) {
      float* const pp = a.part + (((s.lo + tok) * a.hq + h * a.g + hrow) * a.npiece + w.piece) * (D + 2);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) pp[32 * dt + rowmap(g, e)] = oacc[dt][e];
      if (g == 0) pp[D] = m_run, pp[D + 1] = l_tot;
    }
    return;
  }
  // O leaves through LDS, so that a row's stores are contiguous
  const float inv = l_tot != 0.f ? 1.f / l_tot : 0.f;
  const int row = 32 * wave + i;
  bf16* const orow = smem + (row >> 6) * GT::ELEMS;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      E4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (EL)(l_tot != 0.f ? oacc[dt][4 * q4 + e] * inv : 0.f);
      *reinterpret_cast<E4*>(orow + GT::off(row & 63, 4 * dt + q4) + 4 * g) = v;
    }
  __syncthreads();
  constexpr int CH = D / 8;
  const int ch = tid % CH;
  for (int rr = tid / CH; r0 + rr <= rl; rr += 64 * NW / CH) {
    const int q = r0 + rr;
    const u32x4 v = *reinterpret_cast<const u32x4*>(smem + (rr >> 6) * GT::ELEMS + GT::off(rr & 63, ch));
    *reinterpret_cast<u32x4*>(a.out + ((s.lo + token(q)) * a.hq + h * a.g + q % a.g) * D + 8 * ch) = v;
  }
}

template <typename EL, int D>
static int tile_launch(const PagedArgs& a, int h, hipStream_t st) {
  if (a.sel != nullptr) {
    hipLaunchKernelGGL(paged_select_kernel, dim3(a.c.nseq), dim3(kSelThreads), 0, st, a);
    LOGO_LAUNCH_CHECK("paged_select_kernel");
  }
  // each sequence may end inside a tile
  const int64_t tiles = a.n * a.g / kTileRows + a.c.nseq, blocks = tiles * a.npiece * h;
  LOGO_REQUIRE(blocks < ((int64_t)1 << 31), "grid too large");
  auto kern = a.window >= 0 ? paged_tile_kernel<EL, D, true> : paged_tile_kernel<EL, D, false>;
  LOGO_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)tile_smem<D>()));
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(64 * kTileWaves), tile_smem<D>(), st, a);
  LOGO_LAUNCH_CHECK("paged_tile_kernel");
  return LOGO_OK;
}

int paged_launch_tile(const PagedArgs& a, int h, int d, bool half, hipStream_t st) {
  if (half) return d == 128 ? tile_launch<f16, 128>(a, h, st) : tile_launch<f16, 64>(a, h, st);
  return d == 128 ? tile_launch<bf16, 128>(a, h, st) : tile_launch<bf16, 64>(a, h, st);
}

}  // namespace logo
