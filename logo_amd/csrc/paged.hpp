// The paged key / value cache as the kernels that write and read it see it.
#pragma once

#include <math.h>

#include "capi.hpp"
#include "common.hpp"

namespace logo {

// Refuses what neither kernel takes.
inline int paged_check(const logo_paged_cache* c, int d) {
  LOGO_REQUIRE(c != nullptr, "null cache");
  LOGO_REQUIRE(d == 64 || d == 128, "head dim %d unsupported (64 or 128)", d);
  LOGO_REQUIRE(c->heads >= 1 && c->heads <= 65535, "bad head count");
  LOGO_REQUIRE(c->page_size >= 16 && c->page_size <= 65536 && (c->page_size & (c->page_size - 1)) == 0,
               "page_size (%d) must be a power of two in [16, 65536]", c->page_size);
  LOGO_REQUIRE(c->nseq >= 0 && c->table_width >= 0 && c->pages >= 0 && c->table_row >= c->table_width,
               "bad sequence, table or page counts");
  LOGO_REQUIRE((int64_t)c->table_width * c->page_size <= ((int64_t)1 << 30), "a sequence must stay within 2^30 keys");
  const int64_t strides[6] = {c->k_page, c->k_head, c->k_slot, c->v_page, c->v_head, c->v_slot};
  for (int64_t s : strides) LOGO_REQUIRE(s % 8 == 0 && s >= 0, "page strides must be multiples of 8 elements");
  // a page's rows are addressed by 32-bit byte offsets
  LOGO_REQUIRE(c->k_slot >= d && c->v_slot >= d && c->k_slot * c->page_size < ((int64_t)1 << 30) &&
                   c->v_slot * c->page_size < ((int64_t)1 << 30),
               "slots must hold a row, and a page stay below 2 GB");
  LOGO_REQUIRE(((uintptr_t)c->k | (uintptr_t)c->v) % 16 == 0, "pages must be 16-byte aligned");
  LOGO_REQUIRE(c->pages == 0 || (c->k && c->v), "null pages");
  LOGO_REQUIRE(c->nseq == 0 || (c->cu && c->lens && (c->table || c->table_width == 0)), "null table, cu or lens");
  return LOGO_OK;
}

struct PagedArgs {
  logo_paged_cache c;
  const bf16* q;
  int64_t q_token, q_head;
  bf16* out;             // [n, hq, D]
  const uint8_t* sel;    // [n] or null: every token
  int32_t* idx;          // [n] with sel (many rows): the selected tokens of each sequence, from its first token's place on
  int32_t* count;        // [nseq] with sel (many rows): how many
  float* part;           // partial results, paged_part_row(D) floats a row
  int64_t n;
  int hq, g, shift, window;
  float scale_log2;
  bool zero_rest;
  bool split;            // a sequence's keys may be cut into pieces
  int target;            // workgroups the device holds at once
  int cap;               // many rows: pieces per kv head that part holds
  int part_rows;         // rows of a piece in part
};

// A row's partial result: O unnormalised, its reference maximum, its sum (16-byte aligned).
__host__ __device__ constexpr int paged_part_row(int d) { return d + 4; }

constexpr int kPagedPad = 4;  // floats between the rows of an LDS block of partial outputs

// Compute units of the current device (cached per device).
int device_cus();

// A value that all lanes of the wave hold, as a scalar: what is derived from it (buffer
// descriptors above all) then stays in scalar registers.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The rows of sequence b.
struct PagedSeq {
  int64_t lo;   // first token
  int nq, len;  // new tokens, keys that the table reaches
  int pos0;     // position of the first token
  __device__ __forceinline__ PagedSeq(const PagedArgs& a, int b) {
    lo = max(0, a.c.cu[b]);
    nq = (int)max((int64_t)0, min((int64_t)a.c.cu[b + 1], a.n) - lo);
    const int all = max(a.c.lens[b], 0);
    len = min(all, a.c.table_width << a.shift);
    pos0 = all - nq;
  }
  // The first key that the token at position pos0 + t sees, in whole units of 64, at most len.
  __device__ __forceinline__ int first_key(int t, int window) const {
    return (int)max((int64_t)0, min((int64_t)pos0 + t - window, (int64_t)len)) & ~63;
  }
};

// Copies of one kv head's rows into a kSwz tile, ROWS (8 or 16) at a time: rows row0
// .. row0 + ROWS - 1 of a 16-key group.
template <int D, int ROWS = 16>
struct PagedDma {
  static constexpr int CH = D / 8, RPB = 64 / CH, BLOCKS = ROWS / RPB;
  using Geo = TileGeom<D, kSwz>;
  const bf16* base;
  int64_t page_stride;
  int slot_stride;
  uint32_t o[BLOCKS];
  __device__ __forceinline__ void init(const void* pages, int64_t page, int64_t head, int64_t slot, int h, int row0 = 0) {
    base = static_cast<const bf16*>(pages) + h * head;
    page_stride = page;
    slot_stride = (int)slot;
    const int j = threadIdx.x & 63;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      const int row = RPB * b + j / CH;  // the swizzle has period 16
      o[b] = (uint32_t)(row * slot_stride + 8 * ((j % CH) ^ Geo::swz(row0 + row))) * 2u;
    }
  }
  // `rows` valid rows (none or less: zeros) from slot `slot` of page `page` (negative: zeros) on, to dst
  // (NT: streaming loads, for rows that no other workgroup reads)
  template <bool NT = false>
  __device__ __forceinline__ void issue(bf16* dst, int page, int slot, int rows) const {
    const bf16* p = base + (int64_t)max(page, 0) * page_stride + (int64_t)slot * slot_stride;
    const int bytes = rows > 0 && page >= 0 ? ((min(rows, ROWS) - 1) * slot_stride + D) * 2 : 0;
    const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16*>(p), (short)0, bytes, kBufRsrcWord3);
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      if constexpr (NT) buf_load_lds16_nt(r, dst + RPB * b * D, o[b]);
      else buf_load_lds16(r, dst + RPB * b * D, o[b]);
    }
  }
};

// Whether some element of a lane's outputs is NaN, for any lane whose row is valid.
template <int DT>
__device__ __forceinline__ bool paged_any_nan(const f32x16 (&oacc)[DT], bool valid) {
  float t = 0.f;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) t += oacc[dt][e] * 0.f;  // NaN for infinities too
  return __ballot(valid && t != 0.f) != 0;
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

// Sequence that token n belongs to, or nseq.  By a whole wave.
__device__ __forceinline__ int paged_seq_of(const int32_t* cu, int nseq, int64_t n) {
  const int lane = threadIdx.x & 63;
  int cnt = 0;  // ends at or before n
  for (int c = 0; c < nseq; c += 64) {
    const bool past = c + lane < nseq && (int64_t)cu[c + lane + 1] <= n;
    cnt += __builtin_popcountll(__ballot(past));
  }
  return cnt;
}

// The kernel for chunks of many rows (paged_tile.hip): how a call of n tokens that see
// at most `span` keys each is cut, and its launcher (nw: waves of a workgroup, 32 rows each).
void tile_plan(int nseq, int h, int g, int64_t n, int64_t span, int cus, bool sel, bool& split, int& target, int& cap,
               int& nw);
int paged_launch_tile(const PagedArgs& a, int h, int d, bool half, int nw, hipStream_t st);

}  // namespace logo
