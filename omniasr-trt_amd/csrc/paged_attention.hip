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
// unit's start counts as kPaStart more tiles, about what it costs.  A share's waves take a unit's tiles in turn, each with
// the next tiles' loads in flight in registers, and join through LDS, while the loads of the share's next unit are already
// on their way.  A unit within one share is written at once; of the others each share leaves (O, m, l) in fp32, and a second
// launch joins them:  w_s = exp(m_s - max m), out = sum w_s O_s / sum w_s l_s.
// All of it is found from the lengths on the device, so one launch shape serves every length (graphs), and results do not
// depend on timing.
#include <math.h>

#include "attn_chunks.h"

namespace omni {

constexpr int kPaWaves = 4;
constexpr int kPaStart = 6;

struct PagedAttn {
  const uint16_t* q;  // [rows * T, H, D]
  PagedCache cache;
  const int64_t* lengths;
  int rows, T, H, group, cols, qblocks;
  int units;  // of a row: kv heads x qblocks
  float scale_log2;
  float* part_o;   // [2 * workgroups][16][D]: share w's unit begun before it at 2 w, its unit that goes on at 2 w + 1
  float* part_ml;  // [2 * workgroups][16][2]
  uint16_t* out;   // [rows * T, H, D]
};

// Workgroups that run at once on 256 CUs: what the registers allow, a power of two.
template <int D>
constexpr int paged_slots_log2() {
  return D == 512 ? 8 : 9;
}

// Keys that the row's first and last query see.
struct PagedReach {
  int first, last;
};
__device__ __forceinline__ PagedReach paged_reach(const PagedAttn& a, int b) {
  const int n = (int)clamp64(a.lengths[b], 0, a.cache.positions);
  const int64_t last = (int64_t)n + a.T - 1;
  return {n, (int)(last < a.cache.positions ? last : a.cache.positions)};
}

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, true);  // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, true);
  return v;
}

// The line: 64 rows at a time in the lanes of a wave, lane's row with ``tiles`` for each of its units, after ``before``
// places of the rows ahead of it.
struct PagedLine {
  int b0, tiles, before;
  __device__ int places() const { return tiles > 0 ? tiles + kPaStart : 0; }  // of a unit
  // Rows b0 .. b0 + 63, the first after ``ahead`` places; returns the places up to their end.
  __device__ int take(const PagedAttn& a, int lane, int first, int ahead) {
    b0 = first;
    const int b = first + lane;
    tiles = b < a.rows ? (paged_reach(a, b).last + 31) >> 5 : 0;
    const int mine = places() * a.units, sum = wave_scan(mine);
    before = ahead + sum - mine;
    return ahead + __builtin_amdgcn_readlane(sum, kWave - 1);
  }
};

// All rows' places; ``line`` is left at the last 64 rows.
__device__ __forceinline__ int paged_total(const PagedAttn& a, int lane, PagedLine& line) {
  int total = 0;
  for (int b0 = 0; b0 < a.rows; b0 += kWave) total = line.take(a, lane, b0, total);
  return total;
}

// Places of a share: an even part of all for each workgroup, at least two tiles for each wave.
template <int D>
__device__ __forceinline__ int paged_share(int total) {
  return max((total + (1 << paged_slots_log2<D>()) - 1) >> paged_slots_log2<D>(), 2 * kPaWaves);
}

// A unit, and where its tiles are in the line: [from, from + tiles).
struct PagedUnit {
  int b, unit, tiles, from;
};

// The unit that holds place ``x`` (in its start or its tiles).
__device__ __forceinline__ PagedUnit paged_find(const PagedAttn& a, int lane, PagedLine& line, int x) {
  int ahead = 0;
  if (a.rows > kWave) ahead = line.take(a, lane, 0, 0);
  for (;;) {
    const uint64_t hit = __ballot(x >= line.before && x < line.before + line.places() * a.units);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      PagedUnit u;
      u.b = line.b0 + l;
      u.tiles = __builtin_amdgcn_readlane(line.tiles, l);
      const int start = __builtin_amdgcn_readlane(line.before, l), places = u.tiles + kPaStart;
      u.unit = (int)((uint32_t)(x - start) / (uint32_t)places);
      u.from = start + u.unit * places + kPaStart;
      return u;
    }
    ahead = line.take(a, lane, line.b0 + kWave, ahead);
  }
}

// Tiles ahead that a wave's loads run: what fits its registers beside the accumulators.
template <int D, bool kF8>
constexpr int paged_ahead() {
  return D == 128 ? 2 : 1;
}

// What a lane holds of a tile: K, V and, e4m3, exponent bytes (V's for its 8 keys).
template <int D, bool kF8>
struct PagedTile {
  KvChunk<kF8> k[D / 128], v[D / 128];
  uint32_t ks[2];
  u32x2_t vs;
};

// A value that the compiler does not know to be the same in every pass of a loop: what follows from it is worked out where
// it is used, not kept in registers around the loop.
__device__ __forceinline__ int afresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// A share's part of a unit: tiles t0 .. t1 - 1, of which this wave takes first, first + kPaWaves, ...
struct PagedPiece {
  PagedUnit u;
  PagedReach reach;
  int t0, t1, head, qblk, first, mine;
  const int32_t* table;
  __device__ int nth(int i) const { return first + kPaWaves * min(i, mine - 1); }
};

template <int D, bool kF8>
__global__ __launch_bounds__(64 * kPaWaves) __attribute__((amdgpu_waves_per_eu(D == 512 ? 1 : 2))) void
paged_attn_kernel(PagedAttn a) {
  constexpr int kChunks = D / 128, kRowB = D * (kF8 ? 1 : 2), kAhead = paged_ahead<D, kF8>();
  constexpr int kQRow = D * 2 + 16;  // LDS bytes of a query, padded against bank conflicts
  constexpr int kQPieces = 16 * (D / 8) / (64 * kPaWaves);  // of 16 bytes, of the block's queries, for a thread
  __shared__ __attribute__((aligned(16))) char qs[16 * kQRow];
  __shared__ __attribute__((aligned(16))) float os[kPaWaves][16][D];
  __shared__ float mls[kPaWaves][16][2];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  PagedLine line;
  const int total = paged_total(a, lane, line), share = paged_share<D>(total);
  int x = blockIdx.x * share;
  if (x >= total) return;
  const int x_end = min(x + share, total);

  // The next piece from place x on, false if there is none.
  auto next = [&](PagedPiece& p) {
    while (x < x_end) {
      p.u = paged_find(a, lane, line, x);
      p.t0 = max(x - p.u.from, 0);
      p.t1 = min(x_end - p.u.from, p.u.tiles);
      x = p.u.from + p.u.tiles;
      if (p.t1 <= p.t0) return false;  // only the start of a unit whose tiles are the next share's
      p.head = p.u.unit / a.qblocks;
      p.qblk = p.u.unit - p.head * a.qblocks;
      p.reach = paged_reach(a, p.u.b);
      p.table = a.cache.table + p.u.b * a.cache.table_stride;
      p.first = p.t0 + w;
      p.mine = p.first < p.t1 ? (p.t1 - p.first + kPaWaves - 1) / kPaWaves : 0;
      return true;
    }
    return false;
  };
  // 8 keys in a row are on one page.  Groups of 8 past the one with the last key are read as it; keys behind the last one
  // are read where they share its group, and masked like those a query does not see.  A page number out of the pool is
  // held in it.
  struct Pages {
    int k, v;
  };
  auto group_of = [&](const PagedPiece& p, int t, int eighth) { return min(t * 4 + eighth, (p.reach.last - 1) >> 3); };
  auto page_of = [&](const PagedPiece& p, int group) { return p.table[(group * 8) >> a.cache.page_log2]; };
  auto cell = [&](const PagedPiece& p, int group, int page) {
    const int64_t held = min(max(page, 0), a.cache.pages - 1);
    return ((held * a.cache.kv + p.head) << a.cache.page_log2) + ((group * 8) & ((1 << a.cache.page_log2) - 1));
  };
  auto look = [&](const PagedPiece& p, int i) {
    const int t = p.nth(i);
    return Pages{page_of(p, group_of(p, t, c >> 2)), page_of(p, group_of(p, t, g))};
  };
  PagedTile<D, kF8> tile[kAhead];
  Pages pages;  // of the next tile to be loaded
  // Loads of the wave's tile i: K with its exponents at once, V's chunks one by one from ``vrow``.  Loads past the wave's
  // last tile are made all the same, of one line for all lanes, and not used: without a branch around them no wait has to
  // cover the case that they were not made.
  auto load_k = [&](PagedTile<D, kF8>& t, const PagedPiece& p, int i, Pages at, const char*& vrow, u32x2_t& vs) {
    const int n = p.nth(i);
    const int64_t kc = cell(p, group_of(p, n, c >> 2), at.k) + (c & 3), vc = cell(p, group_of(p, n, g), at.v);
    if constexpr (kF8) {
      t.ks[0] = a.cache.k_scale[kc];
      t.ks[1] = a.cache.k_scale[kc + 4];
      vs = *reinterpret_cast<const u32x2_t*>(a.cache.v_scale + vc);
    }
    vrow = i < p.mine ? a.cache.v + vc * kRowB + c * (kF8 ? 8 : 16) : a.cache.v;
    const char* krow = i < p.mine ? a.cache.k + kc * kRowB + g * 16 : a.cache.k;
#pragma unroll
    for (int ch = 0; ch < kChunks; ++ch) load_k_chunk<kF8, kRowB>(t.k[ch], krow, ch);
  };
  // A piece's queries (0 past the last column) and first tiles on their way; the queries to LDS when they have come.
  u32x4_t qv[kQPieces];
  auto begin = [&](const PagedPiece& p) {
    const int t = afresh(tid);
#pragma unroll
    for (int k = 0; k < kQPieces; ++k) {
      const int i = t + k * 64 * kPaWaves, cc = 16 * p.qblk + i / (D / 8), e = i % (D / 8) * 8;
      const int held = min(cc, a.cols - 1);
      qv[k] = *reinterpret_cast<const u32x4_t*>(
          a.q + (((int64_t)p.u.b * a.T + held / a.group) * a.H + p.head * a.group + held % a.group) * D + e);
      if (cc != held) qv[k] = u32x4_t{0u, 0u, 0u, 0u};
    }
    if (p.mine == 0) return;
    Pages at[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) at[i] = look(p, i);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const char* vrow;
      load_k(tile[i], p, i, at[i], vrow, tile[i].vs);
#pragma unroll
      for (int ch = 0; ch < kChunks; ++ch) load_v_chunk<kF8, kRowB>(tile[i].v[ch], vrow, ch);
    }
    pages = look(p, kAhead);
  };

  PagedPiece p;
  while (next(p)) {
    begin(p);
    const int tq = afresh(tid);
#pragma unroll
    for (int k = 0; k < kQPieces; ++k) {
      const int i = tq + k * 64 * kPaWaves;
      *reinterpret_cast<u32x4_t*>(&qs[i / (D / 8) * kQRow + i % (D / 8) * 16]) = qv[k];
    }
    lds_barrier();
    const int col = 16 * p.qblk + c;
    const int lim = col < a.cols ? min(p.reach.first + col / a.group, p.reach.last) : 0;
    f32x4_t o[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    SoftmaxState st{-INFINITY, -INFINITY, 0.f};
    bool bad = false;
    // The wave's tile i, and the loads of tile i + kAhead into its registers as they fall free.
    auto attend = [&](PagedTile<D, kF8>& t, int i) __attribute__((always_inline)) {
      float kscale[2] = {1.f, 1.f}, vscale[8];
      if constexpr (kF8) {
        kscale[0] = scale_of(t.ks[0]);
        kscale[1] = scale_of(t.ks[1]);
#pragma unroll
        for (int j = 0; j < 8; ++j) vscale[j] = scale_of((t.vs[j >> 2] >> (8 * (j & 3))) & 0xffu);
      }
      f32x4_t acc[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int ch = 0; ch < kChunks; ++ch) {
        u32x4_t q[4];
#pragma unroll
        for (int s = 0; s < 4; ++s)
          q[s] = *reinterpret_cast<const u32x4_t*>(
              &qs[c * kQRow + ch * 256 + (kF8 ? 128 * (s >> 1) + 32 * g + 16 * (s & 1) : 64 * s + 16 * g)]);
        chunk_scores<kF8>(t.k[ch], q, kscale, acc);
        __builtin_amdgcn_sched_barrier(0);
      }
      const char* vrow;
      u32x2_t vs;
      load_k(t, p, i + kAhead, pages, vrow, vs);
      pages = look(p, i + kAhead + 1);
      __builtin_amdgcn_sched_barrier(0);
      float pr[8];
      const int at = p.nth(i) * 32;
      tile_softmax<D / 16>(acc, a.scale_log2, st, o, g, lim - at - 8 * g, pr);
      // Only the wave's last tile of the unit can hold keys that a query does not see: T <= 16 such keys and the end of a
      // tile lie within two tiles, of two waves.  (Columns that are no query's see none.)
      if (at + 31 >= p.reach.first) {
#pragma unroll
        for (int ch = 0; ch < kChunks; ++ch) bad |= only_finite<kF8>(t.v[ch]);
      }
#pragma unroll
      for (int ch = 0; ch < kChunks; ++ch) {
        chunk_values<kF8>(t.v[ch], pr, vscale, o + 8 * ch);
        load_v_chunk<kF8, kRowB>(t.v[ch], vrow, ch);
        __builtin_amdgcn_sched_barrier(0);
      }
      t.vs = vs;
    };
    if (p.mine > 0) {
      for (int i = 0;;) {
        attend(tile[0], i);
        if (++i == p.mine) break;
        if constexpr (kAhead == 2) {
          attend(tile[1], i);
          if (++i == p.mine) break;
        }
      }
    }
    // ---- the four waves' parts, joined through LDS
    const int tj = afresh(tid), cj = tj & 15, gj = (tj & 63) >> 4;
    const float l = column_sum(st.l_run);
    if (gj == 0) {
      mls[w][cj][0] = st.m_ref;
      mls[w][cj][1] = l;
    }
    const int live = min(a.cols - 16 * p.qblk, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (4 * gj + i >= live) continue;
#pragma unroll
      for (int ch = 0; ch < kChunks; ++ch)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<f32x4_t*>(&os[w][4 * gj + i][128 * ch + 8 * cj + 4 * h]) = f32x4_t{
              o[8 * ch + 4 * h][i], o[8 * ch + 4 * h + 1][i], o[8 * ch + 4 * h + 2][i], o[8 * ch + 4 * h + 3][i]};
    }
    if (__any(bad)) {  // infinities and NaN of V that the product of the wave's last tile left out
      const int at = p.nth(p.mine - 1) * 32;
      for (int key = at; key < min(at + 32, p.reach.last); ++key) {
        const int64_t row = (cell(p, key >> 3, page_of(p, key >> 3)) + (key & 7)) * D;
        for (int e = tj & 63; e < D; e += kWave) {
          const float v = kF8 ? ((a.cache.v[row + e] & 0x7f) == 0x7f ? NAN : 0.f)
                              : bf16_to_f32(reinterpret_cast<const uint16_t*>(a.cache.v)[row + e]);
          if (v - v == 0.f) continue;  // finite
          for (int r = 0; r < live; ++r)
            if (key < p.reach.first + (16 * p.qblk + r) / a.group) os[w][r][e] += v;
        }
      }
    }
    lds_barrier();
    const bool whole = p.t0 == 0 && p.t1 == p.u.tiles;
    const int64_t slot = (2 * (int64_t)blockIdx.x + (p.t0 == 0 ? 1 : 0)) * 16;
    for (int i = tj; i < live * (D / 8); i += 64 * kPaWaves) {
      const int r = i / (D / 8), e = i % (D / 8) * 8;
      float m = -INFINITY, ls = 0.f;
      f32x4_t sum[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int s = 0; s < kPaWaves; ++s) m = fmaxf(m, mls[s][r][0]);
#pragma unroll
      for (int s = 0; s < kPaWaves; ++s) {
        const float ms = mls[s][r][0];
        const float f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - m);
        ls += f * mls[s][r][1];
        sum[0] += f * *reinterpret_cast<const f32x4_t*>(&os[s][r][e]);
        sum[1] += f * *reinterpret_cast<const f32x4_t*>(&os[s][r][e + 4]);
      }
      if (whole) {
        const int cc = 16 * p.qblk + r;
        const float div = ls == 0.f ? 1.f : ls;
        u32x4_t v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = pack_bf16x2(sum[k >> 1][2 * (k & 1)] / div, sum[k >> 1][2 * (k & 1) + 1] / div);
        *reinterpret_cast<u32x4_t*>(
            a.out + (((int64_t)p.u.b * a.T + cc / a.group) * a.H + p.head * a.group + cc % a.group) * D + e) = v;
      } else {
        float* po = a.part_o + (slot + r) * D + e;
        *reinterpret_cast<f32x4_t*>(po) = sum[0];
        *reinterpret_cast<f32x4_t*>(po + 4) = sum[1];
        if (e == 0) {
          a.part_ml[(slot + r) * 2] = m;
          a.part_ml[(slot + r) * 2 + 1] = ls;
        }
      }
    }
  }
}

// One workgroup per (query, head): its unit's parts joined where more than one share holds it, zeros where it has no tile.
// Each wave takes every fourth part, several at a time, and the waves join through LDS.
template <int D>
__global__ __launch_bounds__(64 * kPaWaves) void paged_attn_merge_kernel(PagedAttn a) {
  constexpr int kPer = D / 64, kBatch = 4;  // dimensions of a lane, parts in flight
  __shared__ float os[kPaWaves][D], ls[kPaWaves], ms[kPaWaves];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.x, b = row / a.T, h = blockIdx.y;
  const int col = (row - b * a.T) * a.group + h % a.group, unit = h / a.group * a.qblocks + col / 16;
  PagedLine line;
  int total = 0, tiles = 0, before = 0;
  for (int b0 = 0; b0 < a.rows; b0 += kWave) {
    total = line.take(a, lane, b0, total);
    if (b >= b0 && b < b0 + kWave) {
      tiles = __builtin_amdgcn_readlane(line.tiles, b - b0);
      before = __builtin_amdgcn_readlane(line.before, b - b0);
    }
  }
  uint16_t* out = a.out + ((int64_t)row * a.H + h) * D;
  if (tiles == 0) {
    for (int e = threadIdx.x; e < D; e += 64 * kPaWaves) out[e] = 0;
    return;
  }
  const uint32_t from = before + unit * (tiles + kPaStart) + kPaStart, share = paged_share<D>(total);
  const int w0 = from / share, w1 = (from + tiles - 1) / share;
  if (w0 == w1) return;
  auto slot = [&](int part) { return (2 * (int64_t)part + (part == w0 ? 1 : 0)) * 16 + col % 16; };
  float m = -INFINITY, l = 0.f, o[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) o[e] = 0.f;
  for (int p0 = w0 + w; p0 <= w1; p0 += kPaWaves * kBatch) {
    float mp[kBatch], lp[kBatch], op[kBatch][kPer];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int part = p0 + k * kPaWaves;
      const int64_t s = slot(min(part, w1));
      mp[k] = part <= w1 ? a.part_ml[s * 2] : -INFINITY;
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
      if (mp[k] == -INFINITY) continue;  // no key seen
      const float f = __builtin_amdgcn_exp2f(mp[k] - top);
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

// Workgroups of a call: what runs at once, but none that a full table would leave without a share.
inline int paged_workgroups(int64_t units, int64_t positions, int head_dim) {
  const int64_t most = 1 << (head_dim == 512 ? paged_slots_log2<512>() : paged_slots_log2<128>());
  const int64_t places = units * ((positions + 31) / 32 + kPaStart), want = (places + 2 * kPaWaves - 1) / (2 * kPaWaves);
  return (int)(want < most ? want : most);
}

}  // namespace omni

using namespace omni;

static int64_t paged_attn_units(int64_t rows, int32_t tokens, int32_t heads, int32_t kv_heads) {
  const int64_t cols = (int64_t)tokens * (heads / kv_heads);
  return rows * kv_heads * ((cols + 15) / 16);
}

extern "C" size_t omni_paged_attention_workspace(int64_t rows, int32_t tokens, int32_t heads, int32_t kv_heads,
                                                 int32_t head_dim, int32_t page, int32_t width) {
  if (rows <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
  const int64_t units = paged_attn_units(rows, tokens, heads, kv_heads);
  return (size_t)(2LL * paged_workgroups(units, (int64_t)width * page, head_dim) * 16 * (head_dim + 2) * 4);
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
  if (rows > 65535) return OMNI_ERR_SHAPE;
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
  a.qblocks = (a.cols + 15) / 16;
  a.units = kv_heads * a.qblocks;
  const int64_t units = (int64_t)rows * a.units;
  // Places of the line, keys and groups are counted in 31 bits.
  if (a.cache.positions > 0x7fffff00LL || units > 0x7fffff00LL ||
      units * ((a.cache.positions + 31) / 32 + kPaStart) > 0x7fffff00LL)
    return OMNI_ERR_SHAPE;
  const int workgroups = paged_workgroups(units, a.cache.positions, head_dim);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + 2LL * workgroups * 16 * head_dim;
  a.out = (uint16_t*)out;
  const hipStream_t s = (hipStream_t)stream;
  const dim3 merge((unsigned)(rows * tokens), heads);
  const bool f8 = cache_dtype == OMNI_E4M3;
  if (head_dim == 128) {
    if (f8) paged_attn_kernel<128, true><<<workgroups, 64 * kPaWaves, 0, s>>>(a);
    else paged_attn_kernel<128, false><<<workgroups, 64 * kPaWaves, 0, s>>>(a);
    paged_attn_merge_kernel<128><<<merge, 64 * kPaWaves, 0, s>>>(a);
  } else if (head_dim == 256) {
    if (f8) paged_attn_kernel<256, true><<<workgroups, 64 * kPaWaves, 0, s>>>(a);
    else paged_attn_kernel<256, false><<<workgroups, 64 * kPaWaves, 0, s>>>(a);
    paged_attn_merge_kernel<256><<<merge, 64 * kPaWaves, 0, s>>>(a);
  } else {
    if (f8) paged_attn_kernel<512, true><<<workgroups, 64 * kPaWaves, 0, s>>>(a);
    else paged_attn_kernel<512, false><<<workgroups, 64 * kPaWaves, 0, s>>>(a);
    paged_attn_merge_kernel<512><<<merge, 64 * kPaWaves, 0, s>>>(a);
  }
  return omni_launch_status();
}
