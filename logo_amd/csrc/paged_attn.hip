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
// NaN, which stays in O.  So rows whose O is not finite at the end are worked out once
// more, guarded: in tiles that cross the edge of some row's keys, values that are not
// finite then count as zeros, and only the rows that see such a key get NaN
// (paged_pv_guarded).
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
// Bound by reading the keys and values once.  A row is a (token, query head of the
// group) pair of a sequence and kv head.  The workgroups that the device holds at
// once share out the keys of all sequences and kv heads evenly, whatever the
// sequences' lengths: laid end to end (in units of 64 keys, kv head by kv head; keys
// that no selected row sees are left out), each takes an equal stretch, and works it
// off sequence by sequence.  Every workgroup finds its stretch itself from cu, lens and
// selection.  A sequence that is cut leaves partial results, which
// paged_few_join_kernel joins; at most two of a workgroup's sequences are.
//
// Its waves split a sequence's keys in tiles of 32, each through a ring of tile slots
// of its own in LDS (K(0) V(0) K(1) V(1) ...), without a barrier in the loop: a slot is
// filled again as soon as its tile has been read, so most of a CU's 160 KB of LDS is in
// flight at any time, which HBM's latency needs.  Streaming loads: no other workgroup
// reads a key.
//
// The weights are rounded to the element type for the product with V (half a step of
// sum w |v|, as much as the result's own rounding), their sum is not.
//
// Measured (D = 128): 32 sequences of up to 16384 keys, 16 heads in bf16, half of them
// selected, 2.02 GB in 314 us (6.4 TB/s; a plain streaming read reaches 7.1); 3 x up to
// 100003 keys, 32 heads over 4 in fp16, 462 MB in 80 us (5.7 TB/s) and the join 5.5; 700 keys
// of 4 heads 15.6 us with the join, all of it latency.  Pieces of a fixed number of keys,
// each with two tiles in flight, took 435 and 120 us.
constexpr int kFewWaves = 2;
constexpr int kFewUnit = 64;      // keys (as PagedSeq::first_key)
// Keys up to which no sequence is cut.  A call takes 14.9 us uncut and 16.4 cut with its
// join for one sequence of 300 keys (4 heads), 18.3 and 15.4 for one of 512, 18.4 and 22.1
// for 16 of 512 (16 heads).  Beyond it a stretch may be as short as a unit: of four at least,
// 700 keys took 22.7 us and not 15.6, one sequence of 8000 22.4 and not 18.
constexpr int kFewWhole = 512;

template <int D>
constexpr int few_slots() { return D == 128 ? 5 : 10; }
template <int D>
constexpr size_t few_smem() { return (size_t)kFewWaves * few_slots<D>() * 32 * D * sizeof(bf16); }

// The sequences laid end to end, kv head by kv head.
struct FewCut {
  int total, share;  // units a kv head; units a workgroup
  int units, lo, b;  // the located sequence: its units, its first key, its index
  int start;         // its first unit
  int n, first, pre; // the lane's sequence of the last 64 looked at: units, first key, units up to its end

  // Looks at sequences c .. c + 63, a lane each: the units of the keys that some row of
  // theirs sees (at least one where there are new tokens).
  __device__ __forceinline__ void look(const PagedArgs& a, int c) {
    const int lane = threadIdx.x & 63, b = c + lane;
    n = first = 0;
    if (b < a.c.nseq) {
      const PagedSeq s(a, b);
      bool any = s.nq > 0;
      if (a.sel != nullptr) {
        any = false;
        for (int t = 0; t < s.nq && !any; ++t) any = a.sel[s.lo + t] != 0;
      }
      if (a.window >= 0) first = s.first_key(0, a.window);
      n = any ? max(1, (s.len - first + kFewUnit - 1) / kFewUnit) : s.nq > 0;
    }
    pre = n;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(pre, off);
      if (lane >= off) pre += o;
    }
  }
  // One pass over the sequences, by a whole wave: the sum of their units (rest < 0), or
  // the sequence that holds unit `rest` of a kv head (or is number `seq`).
  __device__ __forceinline__ void pass(const PagedArgs& a, int rest, int seq = -1) {
    int base = 0;
    for (int c = 0; c < a.c.nseq; c += 64) {
      if (rest < 0 || a.c.nseq > 64) look(a, c);
      const int lane = threadIdx.x & 63;
      const unsigned long long past = __ballot(rest >= 0 && (seq < 0 ? rest < base + pre : c + lane == seq));
      if (past != 0) {
        const int j = __builtin_ctzll(past);
        b = c + j;
        units = __builtin_amdgcn_readlane(n, j);
        lo = __builtin_amdgcn_readlane(first, j);
        start = base + __builtin_amdgcn_readlane(pre, j) - units;
        return;
      }
      base += __builtin_amdgcn_readlane(pre, 63);
    }
    total = base;
    share = max(1, (base * a.c.heads + a.target - 1) / a.target);
  }
};

template <typename EL, int D>
__global__ __launch_bounds__(64 * kFewWaves) __attribute__((amdgpu_waves_per_eu(1, 1)))
void paged_few_kernel(const PagedArgs a) {
  using E8 = typename Elem<EL>::x8;
  constexpr int NW = kFewWaves, DS = D / 16, DT = D / 32, TILE = 32 * D, SLOTS = few_slots<D>();
  constexpr int NI = 2 * PagedDma<D>::BLOCKS;  // copies a slot
  constexpr int AHEAD = (SLOTS - 1) * NI;      // copies behind the slot that is read
  constexpr int ORS = D + kPagedPad, CH = D / 8;
  static_assert(AHEAD < 64, "vmcnt holds 6 bits");
  static_assert(NW * (32 * ORS + 64) * sizeof(float) <= few_smem<D>(), "the join fits the slots");
  extern __shared__ __attribute__((aligned(16))) char paged_smem[];
  const int tid = threadIdx.x, wave = uniform(tid >> 6), l = tid & 63, i = l & 31, g = l >> 5;
  const int w = blockIdx.x;
  if (a.zero_rest) {
    // tokens of no sequence
    const int begin = a.c.nseq > 0 ? a.c.cu[0] : 0, behind = a.c.nseq > 0 ? a.c.cu[a.c.nseq] : 0;
    if (begin > 0 || behind < a.n)
#pragma unroll 1
      for (int64_t n = w; n < a.n; n += gridDim.x)
        if (n < begin || n >= behind)
#pragma unroll 1
          for (int e = tid; e < a.hq * CH; e += 64 * NW) reinterpret_cast<u32x4*>(a.out + n * a.hq * D)[e] = u32x4{};
  }
  TileReader<D, kSwz> rd;
  rd.init();
  bf16* const ring = reinterpret_cast<bf16*>(paged_smem) + wave * SLOTS * TILE;
  float* const so = reinterpret_cast<float*>(paged_smem);  // [wave][32][ORS], then [wave][32] maxima and sums
  float* const sm = so + NW * 32 * ORS;
  float* const sl = sm + NW * 32;
  const float c = a.scale_log2;

  FewCut cut;
  int pos = 0, end = 0, rest = -1, h = 0, n = 0;
  const bool direct = !a.split && a.c.heads * (int64_t)a.c.nseq <= gridDim.x;
#pragma unroll 1
  for (;; pos += n, rest += n) {
    if (pos >= end && rest >= 0) return;
    if (direct) {  // a sequence and kv head each, nothing to look for
      if (w >= a.c.heads * a.c.nseq) return;
      h = (uint32_t)w / (uint32_t)a.c.nseq;
      cut.b = w - h * a.c.nseq;
      cut.units = 1;
      cut.start = rest = pos = 0;
      end = 1;
      const PagedSeq s(a, cut.b);
      if (s.nq == 0) return;
      cut.lo = a.window >= 0 ? s.first_key(0, a.window) : 0;
    } else if (rest >= 0) {
      if (rest == cut.total) ++h, rest = 0;
      cut.pass(a, rest);
    } else {  // the first pass: the stretch
      cut.pass(a, -1);
      const int all = cut.total * a.c.heads;
      // the last one may end before it starts
      if ((int64_t)w * cut.share >= all) return;
      pos = w * cut.share;
      end = min(pos + cut.share, all);
      h = (uint32_t)pos / (uint32_t)cut.total;
      rest = pos - h * cut.total;
      n = 0;
      continue;
    }
    const int f = rest - cut.start;  // units of the sequence before this stretch
    n = min(cut.units - f, end - pos);
    const int b = uniform(cut.b);
    const PagedSeq s(a, b);
    const int rows = s.nq * a.g, pos0 = s.pos0;
    // not cut (also where nothing joins: keys or rows beyond the caller's bounds): all of it where it starts
    const bool whole = n == cut.units || !a.split || rows > a.part_rows;
    if (whole && f > 0) continue;
    const int lo = cut.lo + kFewUnit * f, hi_piece = whole ? s.len : min(s.len, lo + kFewUnit * n);
    PagedDma<D> dk, dv;
    dk.init(a.c.k, a.c.k_page, a.c.k_head, a.c.k_slot, h);
    dv.init(a.c.v, a.c.v_page, a.c.v_head, a.c.v_slot, h);
    // the table read through the scalar cache, whose waits leave the copies alone
    typedef const __attribute__((address_space(4))) int32_t* Table;
    const Table table = (Table)(uintptr_t)(a.c.table + (int64_t)b * a.c.table_row);

    for (int r0 = 0; r0 < rows; r0 += 32) {  // 32 rows at a time
      const int r = min(r0 + i, rows - 1), tok = r / a.g;
      const bool valid = r0 + i < rows && (a.sel == nullptr || a.sel[s.lo + tok] != 0);
      const int p = valid ? pos0 + tok : -1;
      const int pmin = pos0 + r0 / a.g, pmax = pos0 + (min(r0 + 32, rows) - 1) / a.g;
      const int hi = min(hi_piece, pmax + 1);
      E8 qreg[DS];
      {
        const bf16* const qrow = a.q + (s.lo + tok) * a.q_token + (h * a.g + (r - tok * a.g)) * a.q_head + 8 * g;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) qreg[ds] = valid ? *reinterpret_cast<const E8*>(qrow + 16 * ds) : E8{};
      }
      f32x16 oacc[DT];
      float m_run, l_run, base;
      const int first = lo + 32 * wave;
      const int nt = __ballot(p >= 0) != 0 && first < hi ? (hi - first + 32 * NW - 1) / (32 * NW) : 0;
      int page[2];        // of the groups of the tile whose copies go out next
      uint32_t held = 0;  // bits 2 (t % 16) + u: group u of tile t has a page
      auto look_up = [&](int t) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
          page[u] = table[min((first + 32 * NW * min(t, nt - 1) + 16 * u) >> a.shift, a.c.table_width - 1)];
      };
      // K of tile t, then V of it; past the last tile nothing is read, and the count of copies in flight stays
      auto issue = [&](const PagedDma<D>& d, bf16* slot, int t, bool is_v) {
        const int j0 = first + 32 * NW * t;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int j = j0 + 16 * u;
          const bool has = page[u] >= 0 && page[u] < a.c.pages && j < s.len;
          const uint32_t bit = 1u << (2 * (t & 15) + u);
          held = has ? held | bit : held & ~bit;
          d.template issue<true>(slot + 16 * u * D, has ? page[u] : -1, j & ((1 << a.shift) - 1), t < nt ? s.len - j : 0);
        }
        if (is_v) look_up(t + 1);
      };
      bool guard = false;
#pragma unroll 1
      for (;;) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) oacc[dt] = f32x16{};
        m_run = -INFINITY, l_run = base = 0.f;
        if (nt > 0) {
          look_up(0);
          // as a loop: the launch's first instructions come from memory, one line after the other
#pragma unroll 1
          for (int k = 0; k < SLOTS / 2; ++k) {
            issue(dk, ring + 2 * k * TILE, k, false);
            issue(dv, ring + (2 * k + 1) * TILE, k, true);
          }
          if (SLOTS & 1) issue(dk, ring + (SLOTS - 1) * TILE, SLOTS / 2, false);
        }
        // q has arrived here: waited for inside the loop, it would drain the copies each time
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) pin(qreg[ds]);
        int at = 0;  // ring slot of the tile that is read next
        for (int t = 0; t < nt; ++t) {
          const int j0 = first + 32 * NW * t;
          const uint32_t has = held >> (2 * (t & 15)) & 3;
          const bf16* const kt = ring + at * TILE;
          asm volatile("s_waitcnt vmcnt(%0)" ::"i"(AHEAD) : "memory");
          // all reads of the tile in flight at once; they are done before its slot's next copies
          E8 op[2 * DT > DS ? 2 * DT : DS];
#pragma unroll
          for (int ds = 0; ds < DS; ++ds) op[ds] = rd.template row<EL>(kt, 0, ds);
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_sched_barrier(0);
          f32x16 sc = f32x16{};
#pragma unroll
          for (int ds = 0; ds < DS; ++ds) sc = mfma32(op[ds], qreg[ds], sc);
          // slot 2 t + SLOTS takes the place of K(t): a V where the ring is odd
          issue(SLOTS & 1 ? dv : dk, ring + at * TILE, t + SLOTS / 2, SLOTS & 1);
          at = at + 1 == SLOTS ? 0 : at + 1;
          // V(t), read while S turns into P
          const bf16* const vt = ring + at * TILE;
          asm volatile("s_waitcnt vmcnt(%0)" ::"i"(AHEAD) : "memory");
#pragma unroll
          for (int k = 0; k < 2 * DT; ++k) op[k] = rd.template tr<EL>(vt, 16 * (k / DT), k % DT);
          __builtin_amdgcn_sched_barrier(0);
          float mx = -INFINITY;
          uint32_t seen = 0xffffu;
          // (rows that are not valid may see what they like: their results are dropped)
          if (j0 + 31 > pmin || a.window >= 0 || has != 3) {
            seen = 0;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int key = j0 + rowmap(g, e);
              const bool vis = key <= p && (a.window < 0 || key >= p - a.window) && (has >> (e >> 3) & 1);
              seen |= vis ? 1u << e : 0u;
              sc[e] = vis ? sc[e] : -INFINITY;
            }
          }
#pragma unroll
          for (int e = 0; e < 16; e += 2) mx = max3_f32(mx, sc[e], sc[e + 1]);
          // the reference maximum moves only when the row's grew by more than 2^8 (or on its first key)
          const float mxs = pair_max(mx) * c;
          if (__ballot(mxs - m_run > 8.f)) {
            const float m_new = fmaxf(m_run, mxs);
            base = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = fast_exp2(m_run - base);
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) oacc[dt] *= alpha;
          }
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            sc[e] = fast_exp2(fmaf(sc[e], c, -base));
            sum += sc[e];
          }
          l_run += sum;
          if (guard && __ballot(p >= 0 && seen != 0xffffu) != 0) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
              paged_pv_guarded<EL, D>(oacc, rd, vt, ks, acc_to<EL>(sc, ks), seen >> (8 * ks));
          } else {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
              const E8 pb = acc_to<EL>(sc, ks);
#pragma unroll
              for (int dt = 0; dt < DT; ++dt) oacc[dt] = mfma32(op[DT * ks + dt], pb, oacc[dt]);
            }
          }
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_sched_barrier(0);
          issue(SLOTS & 1 ? dk : dv, ring + at * TILE, t + (SLOTS + 1) / 2, !(SLOTS & 1));
          at = at + 1 == SLOTS ? 0 : at + 1;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (guard || !paged_any_nan<DT>(oacc, valid)) break;
        guard = true;
      }
      // join the waves
      const float l_tot = valid ? pair_sum(l_run) : 0.f;
      if (!valid) m_run = -INFINITY;
      __syncthreads();  // every wave is done with its slots
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
        if (g == 0) sm[wave * 32 + i] = m_run, sl[wave * 32 + i] = l_tot;
      }
      __syncthreads();
      for (int e = tid; e < 32 * CH; e += 64 * NW) {
        const int rr = e / CH, ch = e % CH;
        if (r0 + rr >= rows) break;
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < NW; ++k) m = fmaxf(m, sm[k * 32 + rr]);
        const float base = m == -INFINITY ? 0.f : m;
        float lsum = 0.f, o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = 0.f;
#pragma unroll
        for (int wv = 0; wv < NW; ++wv) {
          const float x = fast_exp2(sm[wv * 32 + rr] - base);
          lsum = fmaf(x, sl[wv * 32 + rr], lsum);
          if (sl[wv * 32 + rr] != 0.f)
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = fmaf(x, so[(wv * 32 + rr) * ORS + 8 * ch + k], o[k]);
        }
        if (whole) {
          const int tk = (r0 + rr) / a.g;
          const float inv = lsum != 0.f ? 1.f / lsum : 0.f;
          E8 v;
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = (EL)(lsum != 0.f ? o[k] * inv : 0.f);
          *reinterpret_cast<E8*>(a.out + ((s.lo + tk) * a.hq + h * a.g + (r0 + rr - tk * a.g)) * D + 8 * ch) = v;
        } else {
          // a stretch has one sequence that started before it and one that goes on behind it at most
          float* const pp = a.part + ((int64_t)(2 * w + (f == 0 ? 1 : 0)) * a.part_rows + rr) * paged_part_row(D);
          *reinterpret_cast<f32x4*>(pp + 8 * ch) = f32x4{o[0], o[1], o[2], o[3]};
          *reinterpret_cast<f32x4*>(pp + 8 * ch + 4) = f32x4{o[4], o[5], o[6], o[7]};
          if (ch == 0) pp[D] = m, pp[D + 1] = lsum;
        }
      }
      __syncthreads();
    }
  }
}

// Joins the parts of a row (blockIdx.y) of a sequence that is cut: blockIdx.x runs
// over the sequences of all kv heads (by_seq), or, where these are more, over the
// boundaries between the stretches, the first inside a sequence standing for it.
template <typename EL, int D>
__global__ __launch_bounds__(256) void paged_few_join_kernel(const PagedArgs a, const bool by_seq) {
  const int row = blockIdx.y, tid = threadIdx.x, l = tid & 63;
  int w = blockIdx.x + 1;  // the stretch in which the sequence's second part lies
  FewCut cut;
  int h, f;  // f: units of its first part
  cut.pass(a, -1);
  if (cut.total == 0) return;
  if (by_seq) {
    h = blockIdx.x / a.c.nseq;
    cut.pass(a, 0, blockIdx.x - h * a.c.nseq);
    const int pos = h * cut.total + cut.start;
    w = (uint32_t)pos / (uint32_t)cut.share + 1;
    f = w * cut.share - pos;
    if (f >= cut.units) return;
  } else {
    if ((int64_t)w * cut.share >= cut.total * a.c.heads) return;
    h = (uint32_t)(w * cut.share) / (uint32_t)cut.total;
    const int rest = w * cut.share - h * cut.total;
    cut.pass(a, rest);
    f = rest - cut.start;
    if (f == 0 || f > cut.share) return;
  }
  const PagedSeq s(a, cut.b);
  const int rows = s.nq * a.g;
  if (row >= rows || rows > a.part_rows) return;
  const int np = 1 + (cut.units - f + cut.share - 1) / cut.share;
  constexpr int CL = D / 4, GR = 256 / CL;
  const int ch = tid % CL, gr = tid / CL;
  auto part = [&](int k) { return a.part + ((int64_t)(2 * (w - 1 + k) + (k == 0 ? 1 : 0)) * a.part_rows + row) * paged_part_row(D); };
  __shared__ float red[4];
  __shared__ float so[GR][D + 4];
  float m = -INFINITY;
  for (int k = tid; k < np; k += 256) m = fmaxf(m, part(k)[D]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
  if (l == 0) red[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float base = m == -INFINITY ? 0.f : m;
  f32x4 o = f32x4{};
  float ls = 0.f;
#pragma unroll 4
  for (int k = gr; k < np; k += GR) {
    const float* const q = part(k);
    const float x = fast_exp2(q[D] - base);
    ls = fmaf(x, q[D + 1], ls);
    const f32x4 y = *reinterpret_cast<const f32x4*>(q + 4 * ch);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(x, y[e], o[e]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) so[gr][4 * ch + e] = o[e];
  if (ch == 0) so[gr][D] = ls;
  __syncthreads();
  if (tid < D) {
    float v = 0.f, sum = 0.f;
#pragma unroll
    for (int k = 0; k < GR; ++k) v += so[k][tid], sum += so[k][D];
    const int tk = row / a.g;
    reinterpret_cast<EL*>(a.out)[((s.lo + tk) * a.hq + h * a.g + row - tk * a.g) * D + tid] =
        (EL)(sum != 0.f ? v / sum : 0.f);
  }
}

// How a call runs: the kernel, whether and how finely keys may be cut, and the workspace.
struct PagedPlan {
  bool few, split;
  int target, cap, part_rows, nw;
  size_t part_bytes, bytes;
};

static PagedPlan paged_plan(int nseq, int h, int hq, int64_t n, int d, int max_q, int max_len, int window, bool sel) {
  PagedPlan p{};
  const int g = hq / h, cus = std::max(1, device_cus());
  // up to 32 rows a sequence (by the caller's bound) share one pass of its keys
  p.few = (int64_t)max_q * g <= 32;
  const int64_t span = window >= 0 ? std::min<int64_t>(max_len, (int64_t)window + max_q) : max_len;
  int64_t parts;
  if (p.few) {
    p.split = span > kFewWhole;
    p.target = cus * (int)(160 * 1024 / (d == 128 ? few_smem<128>() : few_smem<64>()));
    p.part_rows = std::max(1, max_q * g);
    parts = 2 * p.target;
  } else {
    tile_plan(nseq, h, g, n, span, cus, sel, p.split, p.target, p.cap, p.nw);
    p.part_rows = 32 * p.nw;
    parts = (int64_t)p.cap * h;
  }
  if (p.split) p.part_bytes = ((size_t)parts * p.part_rows * paged_part_row(d) * sizeof(float) + 255) & ~(size_t)255;
  p.bytes = p.part_bytes + (sel && !p.few ? ((size_t)n + nseq) * sizeof(int32_t) : 0);
  return p;
}

template <typename EL, int D>
static int few_launch(const PagedArgs& a, hipStream_t st) {
  auto kern = paged_few_kernel<EL, D>;
  LOGO_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)few_smem<D>()));
  hipLaunchKernelGGL(kern, dim3(a.target), dim3(64 * kFewWaves), few_smem<D>(), st, a);
  LOGO_LAUNCH_CHECK("paged_few_kernel");
  if (a.split) {
    const int64_t seqs = (int64_t)a.c.heads * a.c.nseq;
    const bool by_seq = seqs < a.target;
    hipLaunchKernelGGL((paged_few_join_kernel<EL, D>), dim3(by_seq ? (int)seqs : a.target, a.part_rows), dim3(256), 0, st,
                       a, by_seq);
    LOGO_LAUNCH_CHECK("paged_few_join_kernel");
  }
  return LOGO_OK;
}

}  // namespace logo

using namespace logo;

extern "C" size_t logo_paged_attn_workspace_bytes(int nseq, int h, int hq, int64_t n_tokens, int d, int max_q,
                                                  int max_len, int window, int selected) {
  if (nseq < 1 || h < 1 || hq < h || n_tokens < 1 || max_q < 0 || max_len < 0) return 0;
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
  LOGO_REQUIRE((int64_t)cache->nseq * ((int64_t)cache->table_width * cache->page_size / kFewUnit + 1) * h < ((int64_t)1 << 31),
               "sequences x table x heads must stay below 2^31 units of %d keys", kFewUnit);
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
  PagedPlan plan{};
  plan.few = true;
  plan.target = std::max(1, device_cus());
  if (a.c.nseq > 0) plan = paged_plan(a.c.nseq, h, hq, n_tokens, d, max_q, max_len, window, selection != nullptr);
  LOGO_REQUIRE(plan.bytes == 0 || (workspace != nullptr && workspace_bytes >= plan.bytes), "the workspace is too small");
  a.split = plan.split;
  a.target = plan.target;
  a.cap = plan.cap;
  a.part_rows = plan.part_rows;
  a.part = static_cast<float*>(workspace);
  a.idx = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + plan.part_bytes);
  a.count = a.idx + n_tokens;
  hipStream_t st = as_stream(stream);
  const bool half = dtype == LOGO_DTYPE_F16;
  if (!plan.few) return paged_launch_tile(a, h, d, half, plan.nw, st);
  if (half) return d == 128 ? few_launch<f16, 128>(a, st) : few_launch<f16, 64>(a, st);
  return d == 128 ? few_launch<bf16, 128>(a, st) : few_launch<bf16, 64>(a, st);
}
