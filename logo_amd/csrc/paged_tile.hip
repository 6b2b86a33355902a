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

template <int D>
constexpr size_t tile_smem() { return (size_t)4 * 64 * D * sizeof(bf16); }  // K and V, two of each

// Selected tokens of each sequence, in order: one workgroup a sequence, 16 tokens a
// thread and step (5 us for 8192 tokens, a launch's own time).
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

// The cut of a launch's rows and keys.  Where the row tiles leave the device idle, each
// tile's keys are cut into pieces of equal size for all sequences.  How many: a launch
// lasts about as many rounds of workgroups as its pieces fill, each as long as a full
// piece with what a workgroup costs beside (kPieceCost, in keys: its start, its partial
// results); the number with the shortest sum is taken.  Every workgroup works out the
// same from cu, lens and the selected tokens' counts.  Against pieces for two rounds
// wherever the tiles fill less than three quarters of one: 512 tokens behind 7680 (16
// heads over 4, D = 128) 79 -> 59 us, four of them 164 -> 155, a quarter of 8192 tokens
// behind 24576 (16 heads) 640 -> 560; twelve single tokens beside four such chunks the same.
constexpr int kMaxPieces = 16;
constexpr int kTileMinChunk = 512;  // keys
constexpr float kPieceCost = 400.f;
constexpr int kOneByOne = 16;       // sequences up to which each is looked at for the cut and the order
constexpr int kPieceRounds = 2;  // pieces that the partial results have room for, in rounds of workgroups

struct TileWork {
  int b, tile, rows;   // sequence, row tile, the sequence's rows
  int npiece, chunk;   // pieces a row tile, keys a piece
  int piece, total;    // total (split): row tiles of a kv head
  __device__ __forceinline__ static int rows_of(const PagedArgs& a, int b, int& len, int& nq) {
    len = nq = 0;
    if (b >= a.c.nseq) return 0;
    const PagedSeq s(a, b);
    len = s.len;
    nq = s.nq;
    return max(0, a.sel ? min(a.count[b], s.nq) : s.nq) * a.g;
  }
  // The rank-th (piece, row tile) of a kv head: first pieces of all tiles, then second
  // ones, so that those that the ends of sequences shorten come last; the latest rows of
  // a sequence first (they see the most keys).  With pieces = false the rank-th row tile.
  // Against all pieces of a tile together: 1000 tokens each at the ends of 1000, 2000 and
  // 3000 keys (16 heads, D = 128) 96 -> 78 us, a quarter of 8192 tokens behind 24576
  // 650 -> 605, 300, 700 and 120 tokens at the ends of 5000, 9000 and 2000 keys (16 heads
  // over 4) 115 -> 113.
  // By a whole wave; false: none.
  __device__ __forceinline__ bool find(const PagedArgs& a, int rank, int tile_rows, bool pieces) {
    const int lane = threadIdx.x & 63;
    int len, nq, r = rows_of(a, lane, len, nq), nt = (r + tile_rows - 1) / tile_rows;
    npiece = 1;
    piece = total = 0;
    chunk = 0x7fffffff;
    if (a.split) {
      int longest = nt > 0 ? len : 0;
      total = nt;
      float keys = nt * (len - 0.5f * nq);  // of all tiles, about
      for (int c = 64; c < a.c.nseq; c += 64) {
        int x, y;
        const int k = (rows_of(a, c + lane, x, y) + tile_rows - 1) / tile_rows;
        total += k;
        if (k > 0) longest = max(longest, x);
        keys += k * (x - 0.5f * y);
      }
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) {
        total += __shfl_xor(total, off);
        longest = max(longest, __shfl_xor(longest, off));
        keys += __shfl_xor(keys, off);
      }
      total = uniform(total);
      const float wgs = (float)total * a.c.heads;
      // a lane a number of pieces, as far as the partial results have room
      const int n = lane % kMaxPieces + 1, size = ((longest + n - 1) / n + 127) & ~127;
      const bool fits = n == 1 || (size >= kTileMinChunk && n * wgs <= (float)kPieceRounds * a.target);
      const float per_key = __builtin_amdgcn_rcpf((float)size);
      float count = keys * per_key + 0.5f * total;
      if (a.c.nseq <= kOneByOne) {  // few sequences: counted, by the pieces of a middle row
        const float middle = len - 0.5f * nq;
        count = 0.f;
        for (int k = 0; k < a.c.nseq; ++k) {
          const int x = __builtin_amdgcn_readlane(__float_as_int(middle), k);
          count = fmaf((float)__builtin_amdgcn_readlane(nt, k), ceilf(__int_as_float(x) * per_key), count);
        }
      }
      count = n == 1 ? wgs : count * a.c.heads;
      // whole rounds where the tiles are about as long as the longest; others end one by one
      const float rounds = count * __builtin_amdgcn_rcpf((float)a.target);
      const float lasts = keys > 0.8f * total * longest ? ceilf(rounds) : fmaxf(1.f, rounds + 0.5f);
      float cost = fits ? lasts * (size + kPieceCost) : INFINITY;
      int best = n;
#pragma unroll
      for (int off = kMaxPieces / 2; off > 0; off >>= 1) {
        const float o = __shfl_xor(cost, off);
        const int ob = __shfl_xor(best, off);
        if (o < cost || (o == cost && ob < best)) cost = o, best = ob;
      }
      npiece = a.window < 0 ? uniform(best) : 1;
      if (npiece > 1) chunk = ((uniform(longest) + npiece - 1) / npiece + 127) & ~127;
    }
    if (pieces && npiece > 1) {
      piece = rank / total;
      if (piece >= npiece) return false;
      rank -= piece * total;
    }
    for (int c = 0; c < a.c.nseq; c += 64) {
      if (c > 0) r = rows_of(a, c + lane, len, nq), nt = (r + tile_rows - 1) / tile_rows;
      // Uncut tiles of more than a round: the sequences with the longest tiles first.
      // Against their own order: 2048 tokens each at the ends of 2048, 4096, 6144 and 8192
      // keys (16 heads, D = 128) 312 -> 274 us (D = 64: 238 -> 198), 4096 tokens before 15
      // single ones (16 heads over 4, 8192 keys) 334 -> 275; among 51 sequences the looking
      // costs what it gains (349 -> 362).
      int pre = nt;  // tiles up to the end of the lane's sequence
      if (npiece == 1 && a.c.nseq <= kOneByOne && (!a.split || total * a.c.heads > a.target)) {
        const int keys = len - nq / 2;  // of a middle row
        for (int k = 0; k < a.c.nseq; ++k) {
          const int x = __builtin_amdgcn_readlane(keys, k), y = __builtin_amdgcn_readlane(nt, k);
          pre += x > keys || (x == keys && k < lane) ? y : 0;
        }
      } else {
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const int o = __shfl_up(pre, off);
          if (lane >= off) pre += o;
        }
      }
      const unsigned long long past = __ballot(rank < pre && rank >= pre - nt);
      if (past != 0) {
        const int j = __builtin_ctzll(past);
        const int tiles = __builtin_amdgcn_readlane(nt, j);
        const int k = rank - (__builtin_amdgcn_readlane(pre, j) - tiles);
        b = c + j;
        rows = __builtin_amdgcn_readlane(r, j);
        tile = tiles - 1 - k;  // the latest rows, with the most keys, first
        return true;
      }
      rank -= __builtin_amdgcn_readlane(pre, 63);
    }
    return false;
  }
};

// Page ids of the rows that a wave copies, for 64 tiles at a time (lane l: tile
// 64 block + l), and which 16-key groups of those tiles have a page at all.
struct TilePages {
  const int32_t* row;
  int64_t pages;
  int width, shift, kv_lo, len, own, block, id;
  unsigned long long ok[4];
  __device__ __forceinline__ void init(const PagedArgs& a, int b, int lo, int length, int first_row) {
    row = a.c.table + (int64_t)b * a.c.table_row;
    pages = a.c.pages;
    width = a.c.table_width;
    shift = a.shift;
    kv_lo = lo;
    len = length;
    own = first_row >> 4;
    block = -1;
  }
  // Page of the wave's rows of tile x (negative: none), and in `bad` the groups of the tile without one.
  __device__ __forceinline__ int get(int x, uint32_t& bad) {
    if (x >> 6 != block) {
      block = x >> 6;
      const int j0 = kv_lo + 64 * (64 * block + (int)(threadIdx.x & 63));
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = j0 + 16 * u, e = j >> shift;
        int v = -1;
        if (j < len && e < width) v = row[e];
        const bool held = v >= 0 && v < pages;
        ok[u] = __ballot(held);
        if (u == own) id = held ? v : -1;
      }
    }
    const int at = x & 63;
    bad = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) bad |= (ok[u] >> at & 1) ? 0u : 1u << u;
    return __builtin_amdgcn_readlane(id, at);
  }
};

// The loop over key tiles is software-pipelined inside each wave, as in sq_fwd.hip:
// step t runs the MFMAs of S(t + 1) and of O += V(t)^T P(t) slot by slot, with the
// exponentials of P(t) spread over the first three quarters of the slots, the mask and
// row maximum of S(t + 1) over the second half, and operand reads four slots ahead.
// K is copied one tile further ahead than V.  A row's reference maximum moves only when
// its maximum grew by more than 2^8 (or on its first key), so O is rarely rescaled.  The
// weights are rounded to the element type for the product with V (half a step of sum
// w |v|, as much as the result's own rounding), their sum is not.
//
// Bound by the MFMAs and the vector work beside them: 16384 tokens behind 16384 (16 heads
// over 4, D = 128) take 3.1 ms, 1060 TFLOP/s, with the MFMAs 51% busy, the vector units 49%
// and 32% of wave time waiting; the dense causal kernel of this library reaches 1100 at
// 16384 tokens of 16 heads.  At D = 64 a score has half the MFMA work for the same vector
// work: 590 TFLOP/s (four chunks of 512 behind 7680).  Windows and short pieces are bound
// by a workgroup's start (3 to 6 us: its place, its pages, the first tiles) and the
// latency of a step: 4 x 2048 tokens with a window of 128 (16 heads) 49 us.  The same loop
// without the pipeline: 7.4 ms for the first, 97 us for the last.
template <typename EL, int D, bool WINDOW, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 2)))
void paged_tile_kernel(const PagedArgs a) {
  using E8 = typename Elem<EL>::x8;
  using E4 = typename Elem<EL>::x4;
  constexpr int ROWS = 32 * NW, RPW = 64 / NW, DS = D / 16, DT = D / 32;
  constexpr int NX = 2 * DS, NY = 4 * DT;     // MFMA slots of S and of PV
  constexpr int IY = 32 / NY;                 // mask / maximum items per Y slot
  constexpr int NPS = NX + 3 * DT - 1;        // slots that carry items of P
  constexpr auto pfirst = [](int s) constexpr { return (32 * s + NPS - 1) / NPS < 32 ? (32 * s + NPS - 1) / NPS : 32; };
  constexpr auto pslot = [](int it) constexpr { return it * NPS / 32; };
  constexpr int kMaxPerSlot = (32 + NPS - 1) / NPS;
  static_assert(pfirst(NPS) == 32 && pslot(7) + 1 < NX && pslot(15) + 1 < NX + DT && pslot(23) + 1 < NX + 2 * DT &&
                    pslot(31) + 1 < NX + 3 * DT,
                "each group of eight items of P is packed before its PV MFMAs");
  constexpr int PF = 4;                       // operand reads, in slots ahead
  using GT = TileGeom<D, kSwz>;
  extern __shared__ __attribute__((aligned(16))) char tile_mem[];
  bf16* const smem = reinterpret_cast<bf16*>(tile_mem);
  auto tileK = [&](int b) { return smem + b * GT::ELEMS; };
  auto tileV = [&](int b) { return smem + (2 + b) * GT::ELEMS; };
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, i = l & 31, g = l >> 5;
  int rank, h;
  xcd_remap(blockIdx.x, a.c.heads, rank, h);

  // zero rows: tokens that are not selected and those of no sequence, a slice of them a
  // workgroup, D / 8 lanes a row
  if (a.sel != nullptr || (a.zero_rest && (a.c.cu[0] > 0 || a.c.cu[a.c.nseq] < a.n))) {
    constexpr int CH = D / 8;
    const int slices = (int)(gridDim.x / a.c.heads), per = (int)((a.n + slices - 1) / slices);
    const int64_t n0 = (int64_t)rank * per, first = a.c.cu[0], end = a.c.cu[a.c.nseq];
    const int cnt = (int)max((int64_t)0, min((int64_t)per, a.n - n0)) * a.g;
    for (int e = tid / CH; e < cnt; e += 64 * NW / CH) {
      const int64_t n = n0 + e / a.g;
      const bool inside = n >= first && n < end;
      if (inside ? a.sel == nullptr || a.sel[n] != 0 : !a.zero_rest) continue;
      st_nt(reinterpret_cast<u32x4*>(a.out + (n * a.hq + h * a.g + e % a.g) * D) + tid % CH, u32x4{});
    }
  }
  TileWork w;
  if (!w.find(a, rank, ROWS, true)) return;
  const PagedSeq s(a, w.b);
  const int r0 = w.tile * ROWS, pos0 = s.pos0;
  // token in the sequence of row r
  auto token = [&](int r) {
    const int t = a.g == 1 ? r : (int)((uint32_t)r / (uint32_t)a.g);
    return a.sel ? a.idx[s.lo + t] : t;
  };
  const int rl = min(r0 + ROWS, w.rows) - 1;  // last row
  const int wr = r0 + 32 * wave, r = min(wr + i, rl);
  const bool valid = wr + i <= rl, active = wr <= rl;
  const int tok = token(r), hrow = a.g == 1 ? 0 : r % a.g;   // and its query head in the group
  const int p = valid ? pos0 + tok : -1;
  // held as lane values: with scalar branches around the pipelined bodies the register
  // allocator spills hundreds of values between them
  int pmin = pos0 + token(min(wr, rl)), pmax = active ? pos0 + token(min(wr + 31, rl)) : -1;
  pin(pmin);
  pin(pmax);
  // the keys that the workgroup's rows see, of its piece
  const int W = a.window;
  int kv_lo = WINDOW ? s.first_key(uniform(token(r0)), W) : 0;
  int kv_hi = min(s.len, pos0 + uniform(token(rl)) + 1);
  if (w.npiece > 1) {
    kv_lo = w.piece * w.chunk;
    if (w.piece < w.npiece - 1) kv_hi = min(kv_hi, kv_lo + w.chunk);
    if (kv_lo >= kv_hi) return;
  }
  const int nt = max(0, (kv_hi - kv_lo + 63) >> 6);

  E8 qreg[DS];
  {
    const bf16* const qrow = a.q + (s.lo + tok) * a.q_token + (h * a.g + hrow) * a.q_head + 8 * g;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) qreg[ds] = valid ? *reinterpret_cast<const E8*>(qrow + 16 * ds) : E8{};
  }
  f32x16 oacc[DT];
  f32x16 sbuf[2][2];  // [t & 1][32-key half]: scores of this tile and the next
  E8 pb[4];           // P(t) as the PV MFMAs' operand
  float m_run, l_run, base;
  const float c = a.scale_log2;

  TileReader<D, kSwz> rd;  // K read along rows, V transposed
  rd.init();
  PagedDma<D, RPW> dk, dv;
  dk.init(a.c.k, a.c.k_page, a.c.k_head, a.c.k_slot, h, RPW * wave & 15);
  dv.init(a.c.v, a.c.v_page, a.c.v_head, a.c.v_slot, h, RPW * wave & 15);
  TilePages pages;
  pages.init(a, w.b, kv_lo, s.len, RPW * wave);
  auto load = [&](const PagedDma<D, RPW>& d, bf16* tile, int t, int page) {
    const int j = kv_lo + 64 * t + RPW * wave;
    d.issue(tile + RPW * wave * D, page, j & ((1 << a.shift) - 1), s.len - j);
  };
  const int tw_hi = active ? min(nt, ((pmax - kv_lo) >> 6) + 1) : 0;  // the wave's tiles
  const int tw_lo = WINDOW && active ? max(0, max(pmin, 0) - W - kv_lo) >> 6 : 0;
  int page_v = -1;              // page of the wave's rows of tile t + 1
  uint32_t bad1 = 0, bad2 = 0;  // groups without a page of tiles t + 1 and t + 2
  bool edge = false;            // tile t crosses the edge of some row's keys
  bool guard = false;           // a second run, for values that are not finite behind an edge

  auto step = [&](auto par_tag, int t) {
    constexpr int PAR = decltype(par_tag)::value;  // t & 1
    if (t + 1 < nt) load(dv, tileV(PAR ^ 1), t + 1, page_v);
    bad1 = bad2;
    if (t + 2 < nt) {
      page_v = pages.get(t + 2, bad2);
      load(dk, tileK(PAR), t + 2, page_v);
    }
    const bf16* const kb = tileK(PAR ^ 1);
    const bf16* const vb = tileV(PAR);
    const int j0n = kv_lo + 64 * (t + 1);

    auto body = [&](auto dos_tag, auto dopv_tag, auto mask_tag) {
      constexpr bool DOS = decltype(dos_tag)::value;    // S(t + 1) and its statistics
      constexpr bool DOPV = decltype(dopv_tag)::value;  // P(t) and O += V^T P
      constexpr bool MASK = decltype(mask_tag)::value;  // S(t + 1) crosses an edge
      E8 op[NX + NY];
      auto load_op = [&](auto s_c) {
        constexpr int S = decltype(s_c)::value;
        if constexpr (S < NX) {
          if constexpr (DOS) op[S] = rd.template row<EL>(kb, 32 * (S / DS), S % DS);
        } else {
          if constexpr (DOPV) op[S] = rd.template tr<EL>(vb, 16 * ((S - NX) / DT), (S - NX) % DT);
        }
      };
      static_for<PF>([&](auto s_c) { load_op(s_c); });
      const int hi = p - j0n - 4 * g;  // key offsets in [hi - W, hi] are seen
      float mx = -INFINITY, psum = 0.f;
      static_for<NX + NY>([&](auto s_c) {
        constexpr int S = decltype(s_c)::value;
        __builtin_amdgcn_sched_barrier(0);
        constexpr int I0 = pfirst(S), NI = pfirst(S + 1) - I0;
        float spv[kMaxPerSlot];
        if constexpr (DOPV)
          static_for<NI>([&](auto i_c) {
            constexpr int I = decltype(i_c)::value, IT = I0 + I;
            spv[I] = sbuf[PAR][IT / 16][IT % 16];
            pin(spv[I]);
          });
        if constexpr (S < NX) {
          if constexpr (DOS) {
            constexpr int KK = S / DS, DSI = S % DS;
            const E8 o = op[S];
            sbuf[PAR ^ 1][KK] = mfma32(o, qreg[DSI], DSI == 0 ? f32x16{} : sbuf[PAR ^ 1][KK]);
          }
        } else {
          constexpr int Y = S - NX;
          if constexpr (DOPV) {
            const E8 o = op[S];
            oacc[Y % DT] = mfma32(o, pb[Y / DT], oacc[Y % DT]);
          }
          if constexpr (DOS) {
            float sv[IY];
            static_for<IY>([&](auto e_c) {
              constexpr int E = decltype(e_c)::value, IT = Y * IY + E, KK = IT / 16, JJ = IT % 16;
              sv[E] = sbuf[PAR ^ 1][KK][JJ];
              if constexpr (MASK) {
                pin(sv[E]);
                constexpr int off = 32 * KK + 8 * (JJ / 4) + (JJ % 4);
                bool vis = off <= hi && !(bad1 >> (2 * KK + JJ / 8) & 1);
                if (WINDOW) vis = vis && off >= hi - W;
                if (!vis) sv[E] = -INFINITY;
                sbuf[PAR ^ 1][KK][JJ] = sv[E];
              }
            });
#pragma unroll
            for (int e = 0; e < IY; e += 2) mx = max3_f32(mx, sv[e], sv[e + 1]);
          }
        }
        if constexpr (DOPV) {
          static_for<NI>([&](auto i_c) {
            constexpr int I = decltype(i_c)::value, IT = I0 + I;
            float pv = fast_exp2(fmaf(spv[I], c, -base));
            pin(pv);
            sbuf[PAR][IT / 16][IT % 16] = pv;
          });
          if constexpr (S >= 1) {
            constexpr int J0 = pfirst(S - 1), NJ = I0 - J0;
            static_for<NJ>([&](auto i_c) {
              constexpr int IT = J0 + decltype(i_c)::value;
              psum += sbuf[PAR][IT / 16][IT % 16];
              if constexpr (IT % 8 == 7) pb[IT / 8] = acc_to<EL>(sbuf[PAR][IT / 16], (IT / 8) & 1);
            });
            if constexpr (NJ > 0) pin(psum);
          }
        }
        if constexpr (S + PF < NX + NY) load_op(std::integral_constant<int, S + PF>{});
      });
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (DOPV) l_run += psum;
      if constexpr (DOS) {
        const float mxs = pair_max(mx) * c;
        const bool any_grow = __ballot(mxs - m_run > 8.f);
        const float m_new = any_grow ? fmaxf(m_run, mxs) : m_run;
        const float nbase = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = fast_exp2(m_run - nbase);
        l_run *= alpha;
        m_run = m_new;
        base = nbase;
        if (__ballot(alpha != 1.f)) {
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) oacc[dt] *= alpha;
        }
      }
    };
    using T_ = std::true_type;
    using F_ = std::false_type;
    const bool doS = t + 1 >= tw_lo && t + 1 < tw_hi;
    bool doPV = t >= tw_lo && t < tw_hi;
    if (guard && doPV && edge) {
      // this tile by itself
      const int hi = p - (j0n - 64) - 4 * g;
      uint32_t bad0;
      pages.get(t, bad0);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        uint32_t seen = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int jj = 8 * (ks & 1) + e, off = 32 * (ks / 2) + 8 * (jj / 4) + (jj & 3);
          const float x = fast_exp2(fmaf(sbuf[PAR][ks / 2][jj], c, -base));
          sbuf[PAR][ks / 2][jj] = x;
          l_run += x;
          if (off <= hi && !(bad0 >> ks & 1) && (!WINDOW || off >= hi - W)) seen |= 1u << e;
        }
        paged_pv_guarded<EL, D>(oacc, rd, vb, ks, acc_to<EL>(sbuf[PAR][ks / 2], ks & 1), seen);
      }
      doPV = false;
    }
    const bool maskn = j0n + 63 > pmin || (WINDOW && j0n < pmax - W) || bad1 != 0;
    if (doS && doPV) {
      if (maskn) body(T_{}, T_{}, T_{});
      else body(T_{}, T_{}, F_{});
    } else if (doS) {
      body(T_{}, F_{}, T_{});
    } else if (doPV) {
      body(F_{}, T_{}, F_{});
    }
    edge = maskn;
    wait_vmem();
    __syncthreads();
  };

  __shared__ int redo;
#pragma unroll 1
  for (;;) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) oacc[dt] = f32x16{};
    m_run = -INFINITY, l_run = base = 0.f;
    if (nt > 0) {
      page_v = pages.get(0, bad2);
      load(dk, tileK(0), 0, page_v);
      if (tid == 0) redo = 0;
      // q has arrived here too: waited for inside the loop, it would drain its copies each time
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) pin(qreg[ds]);
      wait_vmem();
      __syncthreads();
      // step -1 copies V(0) and K(1)
      for (int t = -1; t < nt; t += 2) {
        step(std::integral_constant<int, 1>{}, t);
        if (t + 1 < nt) step(std::integral_constant<int, 0>{}, t + 1);
      }
    }
    if (guard || nt == 0) break;
    if (paged_any_nan<DT>(oacc, valid) && l == 0) redo = 1;
    __syncthreads();
    if (redo == 0) break;
    guard = true;
    __syncthreads();
  }
  const float l_tot = pair_sum(l_run);
  if (w.npiece > 1) {
    if (valid) {
      float* const pp = a.part + (((int64_t)h * a.cap + rank) * ROWS + 32 * wave + i) * paged_part_row(D);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = oacc[dt][4 * q4 + e];
          *reinterpret_cast<f32x4*>(pp + 32 * dt + 8 * q4 + 4 * g) = v;
        }
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

// Joins the pieces of some rows of a row tile a workgroup, eight lanes a row.  Each
// workgroup first finds its tile (some 3 us), so it takes 32 rows and not fewer: at 8 the
// launch took 18.9 us for a batch of 12 single tokens and four chunks of 500 behind up to
// 8192 keys (16 heads, D = 64; 24 MB of partial results), at 32 9.2 us.
constexpr int kJoinRows = 32;
template <typename EL, int D, int NW>
__global__ __launch_bounds__(256) void paged_tile_join_kernel(const PagedArgs a) {
  constexpr int ROWS = 32 * NW, LANES = 256 / kJoinRows, CT = D / (4 * LANES);  // four columns of CT a lane
  using E4 = typename Elem<EL>::x4;
  const int h = blockIdx.y;
  TileWork w;
  if (!w.find(a, blockIdx.x / (ROWS / kJoinRows), ROWS, false) || w.npiece == 1) return;
  const PagedSeq s(a, w.b);
  const int r = w.tile * ROWS + blockIdx.x % (ROWS / kJoinRows) * kJoinRows + threadIdx.x / LANES;
  const int col = threadIdx.x % LANES * 4;
  if (r >= w.rows) return;
  const int tok = a.sel ? a.idx[s.lo + r / a.g] : r / a.g, p = min(s.len - 1, s.pos0 + tok);
  // pieces that hold keys which the row sees
  const int np = p < 0 ? 0 : min(p / w.chunk, w.npiece - 1) + 1;
  const int64_t size = (int64_t)ROWS * paged_part_row(D), step = w.total * size;
  const float* const pp = a.part + ((int64_t)h * a.cap + blockIdx.x / (ROWS / kJoinRows)) * size +
                          (r - w.tile * ROWS) * paged_part_row(D);
  float m = -INFINITY;
  for (int k = 0; k < np; ++k) m = fmaxf(m, pp[k * step + D]);
  const float base = m == -INFINITY ? 0.f : m;
  f32x4 o[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) o[c] = f32x4{};
  float sum = 0.f;
#pragma unroll 2
  for (int k = 0; k < np; ++k) {
    const float* const pk = pp + k * step;
    const float f = fast_exp2(pk[D] - base);
    sum = fmaf(f, pk[D + 1], sum);
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(pk + 4 * LANES * c + col);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[c][e] = fmaf(f, x[e], o[c][e]);
    }
  }
  EL* const orow = reinterpret_cast<EL*>(a.out) + ((s.lo + tok) * a.hq + h * a.g + r % a.g) * D + col;
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    E4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (EL)(sum != 0.f ? o[c][e] / sum : 0.f);
    *reinterpret_cast<E4*>(orow + 4 * LANES * c) = v;
  }
}

template <typename EL, int D, int NW>
static int tile_launch(const PagedArgs& a, int h, hipStream_t st) {
  if (a.sel != nullptr) {
    hipLaunchKernelGGL(paged_select_kernel, dim3(a.c.nseq), dim3(kSelThreads), 0, st, a);
    LOGO_LAUNCH_CHECK("paged_select_kernel");
  }
  // each sequence may end inside a tile
  const int64_t tiles = a.n * a.g / (32 * NW) + a.c.nseq, ranks = std::max<int64_t>(tiles, a.split ? a.cap : 0);
  LOGO_REQUIRE(ranks * h < ((int64_t)1 << 31), "grid too large");
  auto kern = a.window >= 0 ? paged_tile_kernel<EL, D, true, NW> : paged_tile_kernel<EL, D, false, NW>;
  LOGO_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)tile_smem<D>()));
  hipLaunchKernelGGL(kern, dim3((unsigned)(ranks * h)), dim3(64 * NW), tile_smem<D>(), st, a);
  LOGO_LAUNCH_CHECK("paged_tile_kernel");
  if (a.split) {
    // only tiles that are cut: their pieces fit a.cap
    const int64_t cut = std::min<int64_t>(tiles, a.cap / 2);
    hipLaunchKernelGGL((paged_tile_join_kernel<EL, D, NW>), dim3((unsigned)(cut * (32 * NW / kJoinRows)), h), dim3(256), 0,
                       st, a);
    LOGO_LAUNCH_CHECK("paged_tile_join_kernel");
  }
  return LOGO_OK;
}

template <typename EL, int D>
static int tile_dispatch(const PagedArgs& a, int h, int nw, hipStream_t st) {
  return nw == 8 ? tile_launch<EL, D, 8>(a, h, st) : tile_launch<EL, D, 4>(a, h, st);
}

// Eight waves (256 rows share a tile's copies) where at least two rounds of such
// workgroups are sure, one on a CU; four elsewhere, two on a CU.  16384 tokens behind
// 16384 (16 heads over 4, D = 128): 3140 us with eight, 3530 with four.
void tile_plan(int nseq, int h, int g, int64_t n, int64_t span, int cus, bool sel, bool& split, int& target, int& cap,
               int& nw) {
  const int64_t rows = n * g;
  nw = !sel && rows / 256 * h >= 2 * cus ? 8 : 4;
  target = cus * 8 / nw;
  // the selected rows may be few of all, else the row tiles are known but for the sequences' ends
  split = span >= 2 * kTileMinChunk && (sel || rows / (32 * nw) * h < (int64_t)target);
  const int64_t tiles = rows / (32 * nw) + nseq;
  cap = split ? (int)std::max<int64_t>(1, std::min<int64_t>(kPieceRounds * target / h, tiles * kMaxPieces)) : 0;
}

int paged_launch_tile(const PagedArgs& a, int h, int d, bool half, int nw, hipStream_t st) {
  if (half) return d == 128 ? tile_dispatch<f16, 128>(a, h, nw, st) : tile_dispatch<f16, 64>(a, h, nw, st);
  return d == 128 ? tile_dispatch<bf16, 128>(a, h, nw, st) : tile_dispatch<bf16, 64>(a, h, nw, st);
}

}  // namespace logo
