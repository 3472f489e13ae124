// Attention of a step's new tokens over a paged key-value cache on gfx950.
//
// Query i of row b (i < T) sees keys [0, lengths[b] + i) of the row's pages:
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q.k_j,  m = max_j s_j, zeros where there is no key.
// The unit of work is (row, kv head, block of 16 query columns): the T * group queries that read one kv head's keys are
// its columns, column i * group + j being token i's head kv * group + j, so that grouped heads and drafts share one read of
// the keys.
//
// What bounds it is the HBM stream of the keys, so every CU is to stream the same share from start to end.  The 32-key
// tiles of all units stand in one line (row after row, unit after unit), cut into equal shares, one for each workgroup of
// four waves, whatever the rows' lengths: a share is the end of one unit, whole units, and the beginning of another.  A
// unit's start counts as some more tiles (paged_start), about what it costs.  A wave holds 128 dimensions, so the waves
// take a unit's tiles in turn at head dim 128, in pairs at 256 and together at 512, where their partial scores are added
// through LDS; each has the next tiles' loads in flight in registers.  A unit within one share is written at once; of the others each
// share leaves (O, m, l) in fp32, and a second launch joins them:
//   w_s = exp(m_s - max m), out = sum w_s O_s / sum w_s l_s.
// All of it is found from the lengths on the device, so one launch shape serves every length (graphs), and results do not
// depend on timing.
#include <math.h>

#include "attn_chunks.h"

namespace omni {

constexpr int kPaWaves = 4;
constexpr int kPaLeast = 3;  // places of a share, at least

struct PagedAttn {
  const uint16_t* q;  // [rows * T, H, D]
  PagedCache cache;
  const int64_t* lengths;
  int rows, T, H, group, cols, qblocks;
  int units;  // of a row: kv heads x qblocks
  int start;  // tiles that a unit's start counts as
  float scale_log2;
  float* part_o;   // [2 * workgroups][16 NB][D]: share w's unit begun before it at 2 w, its unit that goes on at 2 w + 1
  float* part_ml;  // [2 * workgroups][16 NB][2]
  int* ahead;      // [rows + 1]: places ahead of each row, and all; from the first launch for the second
  uint16_t* out;   // [rows * T, H, D]
};

// Workgroups of a launch at most: as many as run at once, two on each of 256 CUs.  (One at head dim 256 with two blocks of
// columns, whose LDS, 83456 bytes, fits a CU once: there the shares take two rounds.)
constexpr int kPaSlots = 512;

// Keys that the row's first and last query see.
struct PagedReach {
  int first, last;
};
__device__ __forceinline__ PagedReach paged_reach(const PagedAttn& a, int b) {
  const int n = (int)clamp64(a.lengths[b], 0, a.cache.positions);
  const int64_t last = (int64_t)n + a.T - 1;
  return {n, (int)(last < a.cache.positions ? last : a.cache.positions)};
}

// The line: 64 rows at a time in the lanes of a wave, lane's row with ``tiles`` for each of its units, after ``before``
// places of the rows ahead of it.
struct PagedLine {
  int b0, n, tiles, before, places;  // places: of a unit
  // Rows b0 .. b0 + 63, the first after ``ahead`` places; returns the places up to their end.
  __device__ int take(const PagedAttn& a, int lane, int first, int ahead) {
    b0 = first;
    n = tiles = places = 0;
    if (first + lane < a.rows) {
      const PagedReach r = paged_reach(a, first + lane);
      n = r.first;
      tiles = (r.last + 31) >> 5;
      places = tiles > 0 ? tiles + a.start : 0;
    }
    const int mine = places * a.units, sum = wave_scan(mine);
    before = ahead + sum - mine;
    return ahead + __builtin_amdgcn_readlane(sum, kWave - 1);
  }
};

// All rows' places; ``line`` is left at the last 64 rows.  One wave keeps them (``keep``) for the second launch, whose
// workgroups, one for each query and head, would each have to pass over all rows.
__device__ __forceinline__ int paged_total(const PagedAttn& a, int lane, PagedLine& line, bool keep) {
  int total = 0;
  for (int b0 = 0; b0 < a.rows; b0 += kWave) {
    total = line.take(a, lane, b0, total);
    if (keep && b0 + lane < a.rows) a.ahead[b0 + lane] = line.before;
  }
  if (keep && lane == 0) a.ahead[a.rows] = total;
  return total;
}

// Places of a share: an even part of all for each workgroup, but not so few that what the second launch has to read
// outweighs them.  Measured, shares of 2, 3, 4, 8 places and more, us: 1 slot x 1433 keys, 8 x 512 e4m3 12.5, 13.3, 14.4, 18.2
// (a tile after the other takes 1.1 us there); 32 over 8 x 128 9.8, 9.3, 9.4, 12.1.
__device__ __forceinline__ int paged_share(int total) { return max((total + kPaSlots - 1) / kPaSlots, kPaLeast); }

// A unit, and where its tiles are in the line: [from, from + tiles).
struct PagedUnit {
  int b, n, unit, tiles, from;
};

// The unit that holds place ``x`` (in its start or its tiles).  A workgroup's places follow each other, so the search goes
// on from the rows it is at and passes over all of them once.
__device__ __forceinline__ PagedUnit paged_find(const PagedAttn& a, int lane, PagedLine& line, int x) {
  if (x < __builtin_amdgcn_readlane(line.before, 0)) line.take(a, lane, 0, 0);
  for (;;) {
    const uint64_t hit = __ballot(x >= line.before && x < line.before + line.places * a.units);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      PagedUnit u;
      u.b = line.b0 + l;
      u.n = __builtin_amdgcn_readlane(line.n, l);
      u.tiles = __builtin_amdgcn_readlane(line.tiles, l);
      const int start = __builtin_amdgcn_readlane(line.before, l), places = u.tiles + a.start;
      u.unit = (int)((uint32_t)(x - start) / (uint32_t)places);
      u.from = start + u.unit * places + a.start;
      return u;
    }
    // (Past the last row only where another stream changed the lengths meanwhile: no unit, so that the search ends.)
    if (line.b0 + kWave >= a.rows) return PagedUnit{0, 0, 0, 0, x};
    line.take(a, lane, line.b0 + kWave, __builtin_amdgcn_readlane(line.before + line.places * a.units, kWave - 1));
  }
}

// Tiles ahead that a wave's loads run: what its registers hold beside the accumulators.
template <bool kF8, int NB>
constexpr int paged_ahead() {
  return NB <= (kF8 ? 2 : 1) ? 2 : 1;
}

// What a lane holds of a tile's 128 dimensions: K, V and, e4m3, exponent bytes (V's for its 8 keys).
template <bool kF8>
struct PagedTile {
  KvChunk<kF8> k, v;
  uint32_t ks[2];
  u32x2_t vs;
};

// A value that the compiler does not know to be the same in every pass of a loop: what follows from it is worked out where
// it is used, not kept in registers around the loop.
__device__ __forceinline__ int afresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// A share's part of a unit: tiles t0 .. t1 - 1, of which this wave takes ``mine``: first, first + step, ...
struct PagedPiece {
  PagedUnit u;
  int last;  // keys that the row's last query sees (u.n: its first)
  int t0, t1, head, qblk, first, mine;
  const int32_t* table;
};

// NB: blocks of 16 query columns that share a read of the keys.  Two at most: four spill registers (64
// columns, 42 us against 31 in twos).  Measured, with the second launch's 4-5 us: 8 slots x 5 of 750-2400 keys, 8 heads
// x 512 e4m3 26 us (the stream at 4.1 TB/s), 32 x 128 bf16 37; 16 slots of 4000-8188, 32 over 8 x 128 e4m3 43 (5.5 TB/s).
// Three tiles ahead in place of two 28.6 against 27.1 us; 1024, 768 and 256 workgroups 31, 29 and 27 against 27.  Loads that
// are not kept in the caches, over more caches than those hold: the first of these 28.6 to 27.1, the second 45.6 to 42.8, the
// third 48.7 to 44.6 (in bf16 83.8 to 75.3), 8 x 512 bf16 43.3 to 40.6; but 16 tokens, 16 over 2 heads x 256, whose keys four
// units read, 35.9 to 39.2, and K's at head dim 512 28.2 in place of 27.1 (a wave reads a line of K in two halves).
template <int D, bool kF8, int NB>
__global__ __launch_bounds__(64 * kPaWaves) __attribute__((amdgpu_waves_per_eu(2))) void paged_attn_kernel(PagedAttn a) {
  constexpr int kRowB = D * (kF8 ? 1 : 2), kAhead = paged_ahead<kF8, NB>();
  // Two blocks may be a part of more than 32 columns, whose other units read the same keys.  (17 to 32 columns are one unit's,
  // and kept in the caches all the same.)
  constexpr bool kOnce = NB == 1;
  constexpr int kSlices = D / 128, kStep = kPaWaves / kSlices;  // waves to a tile, tiles at a time
  constexpr int kQRow = D * 2 + 16;  // LDS bytes of a query, padded against bank conflicts
  constexpr int kQPieces = 16 * NB * (D / 8) / (64 * kPaWaves);  // of 16 bytes, of the blocks' queries, for a thread
  __shared__ __attribute__((aligned(16))) char qs[16 * NB * kQRow];
  __shared__ f32x4_t parts[kSlices > 1 ? 2 : 1][kSlices > 1 ? kPaWaves : 1][NB][2][64];  // scores by tile parity and wave
  __shared__ __attribute__((aligned(16))) float os[kStep > 1 ? kStep : 1][kStep > 1 ? 16 : 1][D];
  __shared__ float mls[kPaWaves][16 * NB][2];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), sl = w % kSlices, stream = w / kSlices;

  PagedLine line;
  const int total = paged_total(a, lane, line, blockIdx.x == 0 && w == 0), share = paged_share(total);
  int x = blockIdx.x * share;
  if (x >= total) return;
  const int x_end = min(x + share, total);

  // The next piece from place x on, false if there is none.
  auto next = [&](PagedPiece& p) {
    if (x >= x_end) return false;
    p.u = paged_find(a, lane, line, x);
    p.t0 = max(x - p.u.from, 0);
    p.t1 = min(x_end - p.u.from, p.u.tiles);
    x = p.u.from + p.u.tiles;
    if (p.t1 <= p.t0) return false;  // only the start of a unit whose tiles are the next share's
    p.head = (int)((uint32_t)p.u.unit / (uint32_t)a.qblocks);
    p.qblk = p.u.unit - p.head * a.qblocks;
    p.last = (int)min((int64_t)p.u.n + a.T - 1, a.cache.positions);
    p.table = a.cache.table + p.u.b * a.cache.table_stride;
    p.first = p.t0 + stream;
    p.mine = p.first < p.t1 ? (p.t1 - p.first + kStep - 1) / kStep : 0;
    return true;
  };
  // 8 keys in a row are on one page.  Groups of 8 past the one with the last key are read as it; keys behind the last one
  // are read where they share its group, and masked like those a query does not see.  A page number out of the pool is
  // held in it.
  struct Pages {
    int k, v;
  };
  auto group_of = [&](const PagedPiece& p, int i, int eighth) {
    return min((p.first + kStep * i) * 4 + eighth, (p.last - 1) >> 3);
  };
  auto page_of = [&](const PagedPiece& p, int group) { return p.table[(group * 8) >> a.cache.page_log2]; };
  auto cell = [&](const PagedPiece& p, int group, int page) {
    const int64_t held = min(max(page, 0), a.cache.pages - 1);
    return ((held * a.cache.kv + p.head) << a.cache.page_log2) + ((group * 8) & ((1 << a.cache.page_log2) - 1));
  };
  auto look = [&](const PagedPiece& p, int i) {
    return Pages{page_of(p, group_of(p, i, c >> 2)), page_of(p, group_of(p, i, g))};
  };
  PagedTile<kF8> tile[kAhead];
  Pages pages;  // of the next tile to be loaded
  // Loads of the wave's tile i: K with its exponents at once, V from ``vrow``.  Loads past the wave's last tile are made all
  // the same, of one line for all lanes, and not used: without a branch around them no wait has to cover the case that they
  // were not made.
  auto load_k = [&](PagedTile<kF8>& t, const PagedPiece& p, int i, Pages at, const char*& vrow, u32x2_t& vs) {
    const int64_t kc = cell(p, group_of(p, i, c >> 2), at.k) + (c & 3), vc = cell(p, group_of(p, i, g), at.v);
    if constexpr (kF8) {
      t.ks[0] = a.cache.k_scale[kc];
      t.ks[1] = a.cache.k_scale[kc + 4];
      vs = *reinterpret_cast<const u32x2_t*>(a.cache.v_scale + vc);
    }
    constexpr int kSliceB = 128 * (kF8 ? 1 : 2);
    vrow = i < p.mine ? a.cache.v + vc * kRowB + sl * kSliceB + c * (kF8 ? 8 : 16) : a.cache.v;
    load_k_chunk<kF8, kRowB, kOnce && D == 128>(t.k, i < p.mine ? a.cache.k + kc * kRowB + sl * kSliceB + g * 16 : a.cache.k);
  };

  PagedPiece p;
  while (next(p)) {
    // The blocks' queries (0 past the last column) and the first tiles on their way; the queries to LDS.
    {
      const int t = afresh(tid);
      u32x4_t qv[kQPieces];
#pragma unroll
      for (int k = 0; k < kQPieces; ++k) {
        const int i = t + k * 64 * kPaWaves, col = 16 * NB * p.qblk + i / (D / 8), e = i % (D / 8) * 8;
        const int held = min(col, a.cols - 1), token = (int)((uint32_t)held / (uint32_t)a.group);
        qv[k] = *reinterpret_cast<const u32x4_t*>(
            a.q + (((int64_t)p.u.b * a.T + token) * a.H + p.head * a.group + held - token * a.group) * D + e);
        if (col != held) qv[k] = u32x4_t{0u, 0u, 0u, 0u};
      }
      Pages at[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) at[i] = look(p, i);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const char* vrow;
        load_k(tile[i], p, i, at[i], vrow, tile[i].vs);
        load_v_chunk<kF8, kRowB, kOnce>(tile[i].v, vrow);
      }
      pages = look(p, kAhead);
#pragma unroll
      for (int k = 0; k < kQPieces; ++k) {
        const int i = t + k * 64 * kPaWaves;
        *reinterpret_cast<u32x4_t*>(&qs[i / (D / 8) * kQRow + i % (D / 8) * 16]) = qv[k];
      }
    }
    lds_barrier();
    int lim[NB];  // keys that the lane's query columns see
    f32x4_t o[NB][8];
    SoftmaxState st[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int col = 16 * (NB * p.qblk + nb) + c;
      lim[nb] = col < a.cols ? min(p.u.n + (int)((uint32_t)col / (uint32_t)a.group), p.last) : 0;
      st[nb] = SoftmaxState{-INFINITY, -INFINITY, 0.f};
#pragma unroll
      for (int e = 0; e < 8; ++e) o[nb][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    bool bad = false;
    // The wave's tile i, and the loads of tile i + kAhead into its registers as they fall free.
    auto attend = [&](PagedTile<kF8>& t, int i) __attribute__((always_inline)) {
      f32x4_t acc[NB][2];
      {
        const float kscale[2] = {scale_of(t.ks[0]), scale_of(t.ks[1])};
        u32x4_t q[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int s = 0; s < 4; ++s)
            q[nb][s] = *reinterpret_cast<const u32x4_t*>(
                &qs[(16 * nb + c) * kQRow + sl * 256 + (kF8 ? 128 * (s >> 1) + 32 * g + 16 * (s & 1) : 64 * s + 16 * g)]);
        chunk_scores<kF8, NB>(t.k, q, kscale, acc);
      }
      __builtin_amdgcn_sched_barrier(0);
      const char* vrow;
      u32x2_t vs;
      load_k(t, p, i + kAhead, pages, vrow, vs);
      pages = look(p, i + kAhead + 1);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kSlices > 1) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int mb = 0; mb < 2; ++mb) parts[i & 1][w][nb][mb][lane] = acc[nb][mb];
        lds_barrier();
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int mb = 0; mb < 2; ++mb) {
            acc[nb][mb] = parts[i & 1][w - sl][nb][mb][lane];  // the slices in one order in every wave
#pragma unroll
            for (int s = 1; s < kSlices; ++s) acc[nb][mb] += parts[i & 1][w - sl + s][nb][mb][lane];
          }
      }
      if (i < p.mine) {
        const int at = (p.first + kStep * i) * 32;
        float vscale[8];
        u32x4_t pop[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          pop[nb] = tile_softmax<8>(acc[nb], a.scale_log2, st[nb], o[nb], g, lim[nb] - at - 8 * g);
        // Only the wave's last tile of the unit can hold keys that a query does not see where the waves' tiles are kStep
        // apart, its last two otherwise: such keys are the last T - 1 <= 15 and the end of the last tile.
        if (at + 31 >= p.u.n) bad |= only_finite<kF8>(t.v, t.vs);
#pragma unroll
        for (int j = 0; j < 8; ++j) vscale[j] = scale_of((t.vs[j >> 2] >> (8 * (j & 3))) & 0xffu);
        chunk_values<kF8, NB>(t.v, pop, vscale, o);
      }
      load_v_chunk<kF8, kRowB, kOnce>(t.v, vrow);
      t.vs = vs;
      __builtin_amdgcn_sched_barrier(0);
    };
    // The waves of a tile, and those beside them, meet at its barrier: as many rounds for all.
    const int rounds = kSlices > 1 ? (p.t1 - p.t0 + kStep - 1) / kStep : p.mine;
    if (rounds > 0) {
      for (int i = 0;;) {
        attend(tile[0], i);
        if (++i == rounds) break;
        if constexpr (kAhead == 2) {
          attend(tile[1], i);
          if (++i == rounds) break;
        }
      }
    }
    if (__any(bad)) {  // infinities and NaN of V that the products of the last tiles left out (the ballot keeps it one branch)
      for (int i = max(p.mine - 2, 0); i < p.mine; ++i) {
        const int at = (p.first + kStep * i) * 32;
        if (at + 31 < p.u.n) continue;
        for (int key = at; key < min(at + 32, p.last); ++key) {
          const int64_t at_cell = cell(p, key >> 3, page_of(p, key >> 3)) + (key & 7), row = at_cell * D + 128 * sl + 8 * c;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float v;
            if constexpr (kF8) {
              v = __builtin_amdgcn_cvt_f32_fp8((uint8_t)a.cache.v[row + e], 0) * scale_of(a.cache.v_scale[at_cell]);
            } else {
              v = bf16_to_f32(reinterpret_cast<const uint16_t*>(a.cache.v)[row + e]);
            }
            if (v - v == 0.f) continue;  // finite
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int col = 16 * (NB * p.qblk + nb) + 4 * g + r;
                if (col < a.cols && key < p.u.n + col / a.group) o[nb][e][r] += v;
              }
          }
        }
      }
    }

    // ---- the waves' parts: those of one slice joined through LDS
    const int tj = afresh(tid), cj = tj & 15, gj = (tj & 63) >> 4;
    const bool whole = p.t0 == 0 && p.t1 == p.u.tiles;
    const int64_t slot = (2 * (int64_t)blockIdx.x + (p.t0 == 0 ? 1 : 0)) * 16 * NB;
    // 8 dimensions from ``e`` of the piece's column ``r`` (relative to m, weights' sum l), out or left for the second launch.
    auto keep = [&](int r, int e, f32x4_t lo, f32x4_t hi, float m, float l) {
      const int col = 16 * NB * p.qblk + r;
      if (whole) {
        const float div = l == 0.f ? 1.f : l;
        const u32x4_t v = {pack_bf16x2(lo[0] / div, lo[1] / div), pack_bf16x2(lo[2] / div, lo[3] / div),
                           pack_bf16x2(hi[0] / div, hi[1] / div), pack_bf16x2(hi[2] / div, hi[3] / div)};
        const int token = (int)((uint32_t)col / (uint32_t)a.group);
        *reinterpret_cast<u32x4_t*>(
            a.out + (((int64_t)p.u.b * a.T + token) * a.H + p.head * a.group + col - token * a.group) * D + e) = v;
      } else {
        float* po = a.part_o + (slot + r) * D + e;
        *reinterpret_cast<f32x4_t*>(po) = lo;
        *reinterpret_cast<f32x4_t*>(po + 4) = hi;
        if (e == 0) {
          a.part_ml[(slot + r) * 2] = m;
          a.part_ml[(slot + r) * 2 + 1] = l;
        }
      }
    };
    const int live = min(a.cols - 16 * NB * p.qblk, 16 * NB);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float l = column_sum(st[nb].l_run);
      if (16 * nb >= live) break;
      if constexpr (kStep == 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 4 * gj + i;
          const float mr = __shfl(st[nb].m_ref, r, kWave), lr = __shfl(l, r, kWave);
          if (16 * nb + r >= live) continue;
          keep(16 * nb + r, 128 * sl + 8 * cj, f32x4_t{o[nb][0][i], o[nb][1][i], o[nb][2][i], o[nb][3][i]},
               f32x4_t{o[nb][4][i], o[nb][5][i], o[nb][6][i], o[nb][7][i]}, mr, lr);
        }
      } else {
        if (nb > 0) lds_barrier();  // the block before has been read
        if (gj == 0) {
          mls[w][16 * nb + cj][0] = st[nb].m_ref;
          mls[w][16 * nb + cj][1] = l;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (16 * nb + 4 * gj + i >= live) continue;
          float* row = &os[stream][4 * gj + i][128 * sl + 8 * cj];
          *reinterpret_cast<f32x4_t*>(row) = f32x4_t{o[nb][0][i], o[nb][1][i], o[nb][2][i], o[nb][3][i]};
          *reinterpret_cast<f32x4_t*>(row + 4) = f32x4_t{o[nb][4][i], o[nb][5][i], o[nb][6][i], o[nb][7][i]};
        }
        lds_barrier();
        for (int i = tj; i < min(live - 16 * nb, 16) * (D / 8); i += 64 * kPaWaves) {
          const int r = i / (D / 8), e = i % (D / 8) * 8;
          float m = -INFINITY, ls = 0.f;
          f32x4_t sum[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int s = 0; s < kStep; ++s) m = fmaxf(m, mls[s * kSlices][16 * nb + r][0]);
#pragma unroll
          for (int s = 0; s < kStep; ++s) {
            const float ms = mls[s * kSlices][16 * nb + r][0];
            const float f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - m);
            ls += f * mls[s * kSlices][16 * nb + r][1];
            sum[0] += f * *reinterpret_cast<const f32x4_t*>(&os[s][r][e]);
            sum[1] += f * *reinterpret_cast<const f32x4_t*>(&os[s][r][e + 4]);
          }
          keep(16 * nb + r, e, sum[0], sum[1], m, ls);
        }
      }
    }
    // The next piece's queries and scores go where this one's were read, and its parts where these were summed.
    lds_barrier();
  }
}

// One workgroup per (query, head): its unit's parts joined where more than one share holds it, zeros where it has no tile.
// Each wave takes every fourth part, several at a time, and the waves join through LDS.
template <int D, int NB>
__global__ __launch_bounds__(64 * kPaWaves) void paged_attn_merge_kernel(PagedAttn a) {
  constexpr int kPer = D / 64, kBatch = 4;  // dimensions of a lane, parts in flight
  __shared__ float os[kPaWaves][D], ls[kPaWaves], ms[kPaWaves];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x, b = row / a.T, h = blockIdx.y;
  const int col = (row - b * a.T) * a.group + h % a.group, unit = h / a.group * a.qblocks + col / (16 * NB);
  const int total = a.ahead[a.rows], before = a.ahead[b], places = (int)((uint32_t)(a.ahead[b + 1] - before) / (uint32_t)a.units);
  const int tiles = places > 0 ? places - a.start : 0;
  uint16_t* out = a.out + ((int64_t)row * a.H + h) * D;
  if (tiles == 0) {
    for (int e = threadIdx.x; e < D; e += 64 * kPaWaves) out[e] = 0;
    return;
  }
  const uint32_t from = before + unit * places + a.start, share = paged_share(total);
  const int w0 = from / share, w1 = (from + tiles - 1) / share;
  if (w0 == w1) return;
  auto slot = [&](int part) { return (2 * (int64_t)part + (part == w0 ? 1 : 0)) * 16 * NB + col % (16 * NB); };
  float m = -INFINITY, l = 0.f, o[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) o[e] = 0.f;
  for (int p0 = w0 + w; p0 <= w1; p0 += kPaWaves * kBatch) {
    float mp[kBatch], lp[kBatch], op[kBatch][kPer];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int part = p0 + k * kPaWaves;
      const int64_t s = slot(min(part, w1));
      mp[k] = part <= w1 ? a.part_ml[s * 2] : -INFINITY;  // (past the last part: its loads again, not used)
      lp[k] = a.part_ml[s * 2 + 1];
#pragma unroll
      for (int e = 0; e < kPer; ++e) op[k][e] = a.part_o[s * D + kPer * lane + e];
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) top = fmaxf(top, mp[k]);
    const float f0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    l *= f0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] *= f0;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (p0 + k * kPaWaves > w1) break;
      // -inf: no key seen, or scores that are all NaN, which 0 times the part's sums keeps.
      const float f = mp[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mp[k] - top);
      l += f * lp[k];
#pragma unroll
      for (int e = 0; e < kPer; ++e) o[e] += f * op[k][e];
    }
    m = top;
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) os[w][kPer * lane + e] = o[e];
  if (lane == 0) {
    ms[w] = m;
    ls[w] = l;
  }
  __syncthreads();
  float top = -INFINITY, sum = 0.f, f[kPaWaves];
#pragma unroll
  for (int k = 0; k < kPaWaves; ++k) top = fmaxf(top, ms[k]);
#pragma unroll
  for (int k = 0; k < kPaWaves; ++k) {
    f[k] = ms[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms[k] - top);
    sum += f[k] * ls[k];
  }
  const float div = sum == 0.f ? 1.f : sum;
  for (int e = threadIdx.x * 2; e < D; e += 128 * kPaWaves) {
    float v[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kPaWaves; ++k) {
      v[0] += f[k] * os[k][e];
      v[1] += f[k] * os[k][e + 1];
    }
    *reinterpret_cast<uint32_t*>(out + e) = pack_bf16x2(v[0] / div, v[1] / div);
  }
}

// Tiles that a unit's start counts as: more at head dim 128, where each of the four waves has tiles of its own, and more of
// them of e4m3, which are shorter.  Measured, 3, 6 and 8, us: 8 slots x 5 of 750-2400 keys, 32 x 128 e4m3 35.7, 28.1, 25.9, bf16
// 42.3, 37.2, 37.9; 8 slots, 32 over 8 x 128 e4m3 15.6, 13.7, 13.6; 16 over 2 x 256 bf16 13.7, 16.3, 16.2; 8 x 512 bf16 40.4,
// 42.2, 42.1.
inline int paged_start(int head_dim, bool f8) { return head_dim > 128 ? 3 : f8 ? 8 : 6; }

// Workgroups of a call: what runs at once, but none that a full table would leave without a share.
inline int paged_workgroups(int64_t units, int64_t positions, int start) {
  const int64_t places = units * ((positions + 31) / 32 + start), want = (places + kPaLeast - 1) / kPaLeast;
  return (int)(want < kPaSlots ? want : kPaSlots);
}

// Blocks of 16 columns that share a read of the keys, as far as the registers go.
inline int paged_blocks(int cols) { return cols <= 16 ? 1 : 2; }

template <int D, int NB>
inline void paged_launch(const PagedAttn& a, bool f8, int workgroups, hipStream_t s) {
  if (f8) paged_attn_kernel<D, true, NB><<<workgroups, 64 * kPaWaves, 0, s>>>(a);
  else paged_attn_kernel<D, false, NB><<<workgroups, 64 * kPaWaves, 0, s>>>(a);
  paged_attn_merge_kernel<D, NB><<<dim3((unsigned)(a.rows * a.T), a.H), 64 * kPaWaves, 0, s>>>(a);
}

}  // namespace omni

using namespace omni;

extern "C" size_t omni_paged_attention_workspace(int64_t rows, int32_t tokens, int32_t heads, int32_t kv_heads,
                                                 int32_t head_dim, int32_t page, int32_t width) {
  if (rows <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
  const int cols = tokens * (heads / kv_heads), wide = 16 * paged_blocks(cols);
  const int64_t units = rows * kv_heads * ((cols + wide - 1) / wide);
  const int64_t parts = 2LL * paged_workgroups(units, (int64_t)width * page, paged_start(head_dim, true)) * wide;
  return (size_t)(parts * (head_dim + 2) * 4 + (rows + 1) * 4);
}

extern "C" int omni_paged_attention(const void* q, const void* k_pages, const void* v_pages, const void* k_scale,
                                    const void* v_scale, int32_t pages, int32_t page, const int32_t* table,
                                    int64_t table_stride, int32_t width, const int64_t* lengths, int32_t rows,
                                    int32_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim, float scale,
                                    void* out, void* workspace, size_t workspace_bytes, int32_t cache_dtype,
                                    int32_t dtype, void* stream) {
  if (dtype != OMNI_BF16) return OMNI_ERR_DTYPE;
  if (rows < 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return OMNI_ERR_INVALID;
  if (tokens > 16 || heads > 4096) return OMNI_ERR_SHAPE;
  if (!(scale > 0.f) || scale == INFINITY) return OMNI_ERR_INVALID;
  if (rows == 0) return OMNI_OK;
  const int status = omni_check_pages(k_pages, v_pages, k_scale, v_scale, pages, page, kv_heads, head_dim, table,
                                      table_stride, rows, width, cache_dtype);
  if (status != OMNI_OK) return status;
  if (pages == 0 || width == 0) return OMNI_ERR_INVALID;
  if (!q || !lengths || !out || (((uintptr_t)q | (uintptr_t)out) & 15u)) return OMNI_ERR_INVALID;
  if ((int64_t)rows * tokens > 0xffffff) return OMNI_ERR_SHAPE;  // the second launch's threads along x: 256 to a query
  if (!workspace || ((uintptr_t)workspace & 255u) ||
      workspace_bytes < omni_paged_attention_workspace(rows, tokens, heads, kv_heads, head_dim, page, width))
    return OMNI_ERR_WORKSPACE;
  PagedAttn a;
  a.q = (const uint16_t*)q;
  a.cache = omni_paged_cache(k_pages, v_pages, k_scale, v_scale, pages, page, kv_heads, table, table_stride, rows, width);
  a.lengths = lengths;
  a.T = tokens;
  a.H = heads;
  a.rows = rows;
  a.group = heads / kv_heads;
  a.cols = tokens * a.group;
  const int blocks = paged_blocks(a.cols), wide = 16 * blocks;
  a.qblocks = (a.cols + wide - 1) / wide;
  a.units = kv_heads * a.qblocks;
  const int64_t units = (int64_t)rows * a.units;
  // Places of the line, keys and groups are counted in 31 bits.
  if (a.cache.positions > 0x7fffff00LL || units > 0x7fffff00LL ||
      units * ((a.cache.positions + 31) / 32 + 8) > 0x7fff0000LL)
    return OMNI_ERR_SHAPE;
  const bool f8 = cache_dtype == OMNI_E4M3;
  a.start = paged_start(head_dim, f8);
  const int workgroups = paged_workgroups(units, a.cache.positions, a.start);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + 2LL * workgroups * wide * head_dim;
  a.ahead = (int*)(a.part_ml + 2LL * workgroups * wide * 2);
  a.out = (uint16_t*)out;
  const hipStream_t s = (hipStream_t)stream;
  if (head_dim == 128) {
    if (blocks == 1) paged_launch<128, 1>(a, f8, workgroups, s);
    else paged_launch<128, 2>(a, f8, workgroups, s);
  } else if (head_dim == 256) {
    if (blocks == 1) paged_launch<256, 1>(a, f8, workgroups, s);
    else paged_launch<256, 2>(a, f8, workgroups, s);
  } else {
    if (blocks == 1) paged_launch<512, 1>(a, f8, workgroups, s);
    else paged_launch<512, 2>(a, f8, workgroups, s);
  }
  return omni_launch_status();
}
