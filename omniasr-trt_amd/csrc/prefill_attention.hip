// Causal attention over whole contexts for gfx950: the prefill's
//     F.scaled_dot_product_attention(q, k, v, is_causal=True)
// (src/omniasr_trt/decode.py:163-164) over the cache rows ``kernels.rope_kv`` has just written.  Query p of context
// b attends to keys [0, p] of its cache row; fp32 accumulation, bf16 in and out, head_dim 128, 256 or 512.
//
// The same kernels (kPacked) attend packed prompts of different lengths with grouped heads over k and v as a projection
// leaves them: sequence s has queries starts[s] .. of q and keys k_starts[s] .. of k / v, and its query i of nq sees its
// keys [0, i + nk - nq] of nk.  What bounds a tile is the same; what they add is lengths from the device, rows of any stride, a
// mask on every tile that not all of a wave's queries see, and at head dim 128 up to four heads of a kv head in a block (64
// queries of each: a short prompt fills a block, and the heads share its tiles).  Measured, us: 8 prompts of 750-2400, 8 heads
// x 512 197 (700 TFLOP/s), 32 over 8 x 128 175; 16 of up to 500 behind up to 900 keys, 32 over 8 x 128 76-80 (a head to a
// block 113); one of 1433, 32 x 128 42.
#include <math.h>

#include <algorithm>

#include "attn_chunks.h"
#include "common.h"

namespace omni {

// Query p of context b attends to keys [0, p] of its cache row; one workgroup per (query block, head, context), the
// longest blocks first; every kernel keeps a lazy softmax reference and masks only the tiles on the diagonal.
typedef short v4i16_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) v4i16_t lds_v4i16;
typedef __attribute__((address_space(3))) const char lds_char;

struct PrefillArgs {
  const uint16_t* q;    // [B * width, H, D] bf16
  const uint16_t* k;    // cache rows: element strides s_row / s_head, key rows contiguous (D elements)
  const uint16_t* v;
  const int64_t* slots;  // [B] cache row of each context
  int64_t s_row, s_head, cache_rows;
  int width, H;
  float scale_log2;
  uint16_t* out;  // [B * width, H, D] bf16
  int units8, group;  // head dim 512 in chains: heads x contexts / 8, and how many of them are listed together
  // Packed prompts (width: the longest's queries); element strides of a key and of a head in k and v.
  const int64_t* starts = nullptr;    // [sequences + 1]
  const int64_t* k_starts = nullptr;  // [sequences + 1]
  int64_t queries = 0, keys = 0;      // rows of q, of k and v
  int64_t k_pos = 0, k_head = 0, v_pos = 0, v_head = 0;
  int heads_per_kv = 1;
  int together = 1;  // head dims 128 and 256: heads of a kv head in one block (1, 2 or 4)
  int block = 0;     // head dims 128 and 256: queries of each head in a block
  // Blocks in parts (pf_part): at most ``parts``, each with room for its O and its queries' (m, l).
  int parts = 1;
  float* part_o = nullptr;   // [part][value wave][query half u][r][e][k][lane][4]
  float* part_ml = nullptr;  // [part][score wave][lane half][query][2]
  int sequences = 0;  // in chains
};
constexpr int kPartO = 4 * 32 * 256, kPartMl = 4 * 2 * 64 * 2;  // floats

// A context's or sequence's part of a call for one head: queries q0 .. q0 + nq - 1, keys 0 .. nk - 1 of k / v, rows
// k_bytes / v_bytes apart; query i sees keys [0, i + before].
struct PfSpan {
  int64_t q0;
  int nq, nk, before;
  const uint16_t* k;
  const uint16_t* v;
  uint32_t k_bytes, v_bytes;
};

template <int D>
__device__ __forceinline__ PfSpan pf_span(const PrefillArgs& a, int h, int b) {
  const int64_t slot = clamp64(a.slots[b], 0, a.cache_rows - 1);
  PfSpan p;
  p.q0 = (int64_t)b * a.width;
  p.nq = p.nk = a.width;
  p.before = 0;
  p.k = a.k + slot * a.s_row + h * a.s_head;
  p.v = a.v + slot * a.s_row + h * a.s_head;
  p.k_bytes = p.v_bytes = D * 2;
  return p;
}

// A packed sequence: its first query and key, and how many there are, within q and k.
struct PfSequence {
  int64_t q0, k0;
  int nq, nk;
};
__device__ __forceinline__ PfSequence pf_sequence(const PrefillArgs& a, int s) {
  PfSequence p;
  p.q0 = clamp64(a.starts[s], 0, a.queries);
  p.k0 = clamp64(a.k_starts[s], 0, a.keys);
  p.nq = (int)(clamp64(a.starts[s + 1], p.q0, a.queries) - p.q0);
  p.nk = (int)(clamp64(a.k_starts[s + 1], p.k0, a.keys) - p.k0);
  return p;
}

__device__ __forceinline__ PfSpan pf_packed_span(const PrefillArgs& a, int h, const PfSequence& s) {
  const int kv = h / a.heads_per_kv;
  PfSpan p;
  p.q0 = s.q0;
  p.nq = min(s.nq, a.width);
  p.nk = s.nk;
  p.before = s.nk - s.nq;
  p.k = a.k + s.k0 * a.k_pos + kv * a.k_head;
  p.v = a.v + s.k0 * a.v_pos + kv * a.v_head;
  p.k_bytes = (uint32_t)a.k_pos * 2;
  p.v_bytes = (uint32_t)a.v_pos * 2;
  return p;
}

// Zeros in rows [q0, q1) of one head: queries that see no key.
template <int D>
__device__ __forceinline__ void pf_zeros(const PrefillArgs& a, int64_t q0, int64_t q1, int h) {
  for (int64_t i = threadIdx.x; i < (q1 - q0) * (D / 8); i += blockDim.x)
    *reinterpret_cast<u32x4_t*>(a.out + ((q0 + i / (D / 8)) * a.H + h) * D + i % (D / 8) * 8) = u32x4_t{0u, 0u, 0u, 0u};
}

// Workgroup -> (query block j counted from the longest, head h, context b).  The dispatcher hands consecutive
// workgroups to the 8 XCDs in turn; when heads x contexts is a multiple of 8, XCD x gets units (head, context)
// x, x + 8, ... one after another, all query blocks of a unit together (longest first), so each unit's K / V rows
// are brought into one XCD's L2 rather than into all eight.  Only speed depends on the dispatch order.
constexpr bool kPfXcd = true;
struct PfBlock {
  int j, h, b;
};
__device__ __forceinline__ PfBlock pf_block(int nqb, int H, int B) {
  if (!kPfXcd || (H * B) % 8 != 0) return PfBlock{(int)blockIdx.x, (int)blockIdx.y, (int)blockIdx.z};
  const int L = (int)blockIdx.x + nqb * ((int)blockIdx.y + H * (int)blockIdx.z);
  const int x = L % 8, k = L / 8;
  const int unit = (k / nqb) * 8 + x;
  return PfBlock{k % nqb, unit % H, unit / H};
}

__device__ __forceinline__ int64_t pf_readlane64(int64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane), hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// Few blocks behind many keys: the longest block is the launch, ~1.4 us for each of its 64-key tiles, while other CUs have
// nothing.  So a block is cut along its keys into parts, each a workgroup's, and a second launch (packed_attn_join_kernel)
// joins their (O, m, l).  A part costs its start and end (~8 us) and 128 KB of O written and read (~1 us of the join, which
// takes 3 by itself): parts of kPartLeast tiles and more, at most kPartMost of a block; where CUs are plenty of 0.8 sqrt(the
// block's tiles), so that a part and the join of all take the least together.  Only where the longest block has kPartLong
// tiles and 1.5 times what all have for each CU, or kPartBlock and four times.  Measured, us, whole and in parts: 20 queries
// behind 1000 keys, 8 heads x 512 30.0 / 21.9, 32 over 8 x 128 29.0 / 19.4, 16 over 2 x 256 29.1 / 19.9; behind 4000, 8 x
// 512 72 / 31.0, 32 over 8 x 128 75 / 29.5; 64 behind 8000, 8 x 512 200 / 57; 300 behind 1000 38.3 / 30.8; 500 behind 6000
// 116 / 80.  Parts of 2 tiles and more, of any block: one prompt of 1433 45 / 57, four of 200-800 28 / 46.
constexpr int kPartCus = 256, kPartLeast = 4, kPartBlock = 12, kPartLong = 24, kPartMost = 16;

// The rank of a lane's sequence by work (queries x keys, less what causality hides), the most first.
__device__ __forceinline__ int pf_rank(const PfSequence& mine, int sequences) {
  const int lane = lane_id();
  const float work = lane < sequences ? (float)mine.nq * (2.f * (float)mine.nk - (float)mine.nq) : -INFINITY;
  int rank = 0;
  for (int t = 0; t < sequences; ++t) {
    const float other = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(work), t));
    rank += other > work || (other == work && t < lane) ? 1 : 0;
  }
  return rank;
}

// The sequence of rank r by work, the most first: so the last blocks of a launch, whose CUs wait for each other, are the
// short ones.  Past 64 sequences, more than a wave has lanes, the order of the call.
// ``share``, where blocks (of ``queries``, ``heads`` for each) may be in parts: the key tiles of a part, about what all blocks
// have for each CU, or what no block is longer than.
__device__ __forceinline__ PfSequence pf_ranked(const PrefillArgs& a, int sequences, int r, int queries, int heads,
                                                int& share) {
  if (sequences > kWave) return pf_sequence(a, r);
  const int lane = lane_id();
  const PfSequence mine = pf_sequence(a, min(lane, sequences - 1));
  if (a.parts > 1) {
    const int nq = min(mine.nq, a.width), blocks = (nq + queries - 1) / queries;
    // Keys of the first block and, about, of a block's mean.  With more queries than keys and a block's worth the first ones
    // see none: only the last nk queries' blocks have any, nk / 2 about.
    const int64_t first = (int64_t)min(nq, queries) + mine.nk - mine.nq;
    const int64_t mean = first > 0 ? (first + mine.nk) / 2 : (mine.nk + 1) / 2;
    const int seeing = first > 0 ? blocks : (int)(((int64_t)mine.nk + queries - 1) / queries);
    const int64_t tiles = blocks > 0 ? seeing * ((mean + 63) / 64) : 0;
    int all = lane < sequences ? (int)(tiles < 65536 ? tiles : 65536) : 0;
    int longest = all > 0 ? (mine.nk + 63) / 64 : 0, count = lane < sequences ? blocks : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      all += __shfl_xor(all, o, kWave);
      count += __shfl_xor(count, o, kWave);
      longest = max(longest, __shfl_xor(longest, o, kWave));
    }
    longest = __builtin_amdgcn_readfirstlane(longest);
    // Parts are whole tiles: half a part of each block's is lost.
    const int room = max(kPartCus - __builtin_amdgcn_readfirstlane(count) * heads / 2, kPartCus / 4);
    const int even = ((int)((uint32_t)__builtin_amdgcn_readfirstlane(all) * (uint32_t)heads) + room - 1) / room;
    int least = kPartLeast;
    while (25 * least * least < 16 * longest && least < 64) ++least;
    const bool cut = longest >= kPartLong ? 2 * longest >= 3 * even : longest >= kPartBlock && longest >= 4 * even;
    share = cut ? max(even, least) : max(longest, 1);
  }
  const int l = __builtin_ctzll(__ballot(lane < sequences && pf_rank(mine, sequences) == r));
  PfSequence p;
  p.q0 = pf_readlane64(mine.q0, l);
  p.k0 = pf_readlane64(mine.k0, l);
  p.nq = __builtin_amdgcn_readlane(mine.nq, l);
  p.nk = __builtin_amdgcn_readlane(mine.nk, l);
  return p;
}

// The workgroup's block for packed prompts, with ``heads`` blocks of heads: XCD x's are x * heads / 8 .., so that heads of
// one kv head stay in one L2.
struct PfPacked {
  int j, h;
  PfSequence s;
  int part, parts, slot, share;  // which of how many, the first one's place in part_o and part_ml
};
__device__ __forceinline__ PfPacked pf_packed_block(const PrefillArgs& a, int nqb, int queries, int heads, int sequences) {
  // The first parts of all blocks, then the second ones, ...: most of the later ones are none, and end at once.
  const int part = a.parts > 1 ? (int)blockIdx.z / sequences : 0, z = (int)blockIdx.z - part * sequences;
  const int L = (int)blockIdx.x + nqb * ((int)blockIdx.y + heads * z);
  PfBlock p = {(int)blockIdx.x, (int)blockIdx.y, z};
  if (heads % 8 == 0) {
    const int k = L / 8, unit = k / nqb;
    p = PfBlock{k % nqb, L % 8 * (heads / 8) + unit % (heads / 8), unit / (heads / 8)};
  } else if (heads * sequences % 8 == 0) {  // as pf_block
    const int k = L / 8, unit = k / nqb * 8 + L % 8;
    p = PfBlock{k % nqb, unit % heads, unit / heads};
  }
  PfPacked one = {p.j, p.h, {}, part, 1, ((p.b * heads + p.h) * nqb + p.j) * a.parts, 0};
  one.s = pf_ranked(a, sequences, p.b, queries, heads, one.share);
  return one;
}

// Parts of a block that sees ``keys`` keys, of about ``share`` tiles.
__device__ __forceinline__ int pf_parts(const PrefillArgs& a, int keys, int share) {
  return a.parts == 1 ? 1 : min(((keys + 63) / 64 + share - 1) / share, a.parts);
}

// This workgroup's part of its block, which sees ``keys`` keys: ``sp`` and ``keys`` narrowed to it; false: there is none.
__device__ __forceinline__ bool pf_part(const PrefillArgs& a, PfPacked& blk, PfSpan& sp, int& keys) {
  if (a.parts == 1) return true;
  const int parts = keys > 0 ? pf_parts(a, keys, blk.share) : 1;
  if (blk.part >= parts) return false;
  if (parts == 1) return true;
  blk.parts = parts;
  const int nt = (keys + 63) / 64, t0 = (int)((uint32_t)nt * (uint32_t)blk.part / (uint32_t)parts);
  const int k0 = 64 * t0, k1 = min(64 * (int)((uint32_t)nt * (uint32_t)(blk.part + 1) / (uint32_t)parts), keys);
  sp.k += k0 * a.k_pos;
  sp.v += k0 * a.v_pos;
  sp.nk = min(sp.nk, k1) - k0;
  sp.before -= k0;
  keys = k1 - k0;
  return true;
}

// Whether the workgroup has a part of a block: the same in every lane, so that neither way out waits for the other.
__device__ __forceinline__ bool pf_in_parts(const PfPacked& blk) { return __builtin_amdgcn_readfirstlane(blk.parts) > 1; }

// A part's queries' (m, l) from its score wave w: query i of lane half g.
__device__ __forceinline__ void pf_leave_ml(const PrefillArgs& a, const PfPacked& blk, int w, int g, int i, float m, float l) {
  *reinterpret_cast<f32x2_t*>(a.part_ml + (int64_t)(blk.slot + blk.part) * kPartMl + ((w * 2 + g) * 64 + i) * 2) =
      f32x2_t{m, l};
}

// A part's O from its value wave vw, of the ``n`` queries there are of its 64.
__device__ __forceinline__ void pf_leave_o(const PrefillArgs& a, const PfPacked& blk, int vw, int lane, int n,
                                           const f32x16_t (&o)[2][4]) {
  float* to = a.part_o + (int64_t)(blk.slot + blk.part) * kPartO + vw * (32 * 256) + lane * 4;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if (32 * u + (lane & 31) >= n) return;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = 4 * (r + 2 * k);
          *reinterpret_cast<f32x4_t*>(to + (((u * 2 + r) * 4 + e) * 2 + k) * 256) =
              f32x4_t{o[u][e][at], o[u][e][at + 1], o[u][e][at + 2], o[u][e][at + 3]};
        }
  }
}

// On a tile with keys that some query does not see, their probability is 0, but 0 times an infinity or NaN of V would
// reach the query's output.  Looking for such values tile by tile costs the kernels registers that they do not have, so
// the outputs are looked at instead: a wave with one that is not finite works its queries out again, 16 at a time and 128
// dimensions of the result (``out`` and ``v`` point at them), leaving what is not finite out of the products of those tiles
// and adding it to the queries that see it -- whose output it makes infinite or NaN whatever its weight.  Rare, and slow.
// ``q`` / ``out``: the first of the ``n`` <= 16 queries, rows q_pos apart; the first sees keys [0, whole] of nk.
template <int D>
__device__ __noinline__ void pf_again_16(const uint16_t* q, const uint16_t* k, const uint16_t* v, uint16_t* out,
                                         int64_t q_pos, int64_t k_pos, int64_t v_pos, int n, int whole, int nk,
                                         float scale_log2, uint32_t wanted) {
  const int lane = lane_id(), c = lane & 15, g = lane >> 4;
  const int end = whole + n, query = min(c, n - 1), lim = whole + query + 1;
  const uint16_t* qrow = q + query * q_pos + 8 * g;
  f32x4_t o[1][8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[0][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  SoftmaxState st{-INFINITY, -INFINITY, 0.f};
  for (int t = 0; t < end; t += 32) {
    f32x4_t acc[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
    for (int s = 0; s < D; s += 32) {
      const u32x4_t qs = *reinterpret_cast<const u32x4_t*>(qrow + s);
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
        const int key = min(t + 8 * (c >> 2) + 4 * mb + (c & 3), nk - 1);
        const u32x4_t ks = *reinterpret_cast<const u32x4_t*>(k + key * k_pos + s + 8 * g);
        acc[mb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, ks), __builtin_bit_cast(bf16x8_t, qs),
                                                          acc[mb], 0, 0, 0);
      }
    }
    const u32x4_t pop[1] = {tile_softmax<8>(acc, scale_log2, st, o[0], g, lim - t - 8 * g)};
    KvChunk<false> vt;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      vt.r[j] = ld16(reinterpret_cast<const char*>(v + min(t + 8 * g + j, nk - 1) * v_pos + 8 * c));
    u32x2_t none = {0u, 0u};
    if (t + 31 > whole && only_finite<false>(vt, none)) {
      for (int key = t; key < min(t + 32, end); ++key)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float value = bf16_to_f32(v[key * v_pos + 8 * c + e]);
          const float extra = value - value == 0.f ? 0.f : value;
#pragma unroll
          for (int i = 0; i < 4; ++i) o[0][e][i] += key <= whole + 4 * g + i ? extra : 0.f;
        }
    }
    const float one[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    chunk_values<false, 1>(vt, pop, one, o);
  }
  const float l = column_sum(st.l_run);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float li = __shfl(l, 4 * g + i, kWave), div = li == 0.f ? 1.f : li;
    if (4 * g + i >= n || !(wanted >> c & 1)) continue;
    u32x4_t w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(o[0][2 * e][i] / div, o[0][2 * e + 1][i] / div);
    *reinterpret_cast<u32x4_t*>(out + (4 * g + i) * q_pos + 8 * c) = w;
  }
}

// Queries q_first .. q_first + 16 groups - 1 of a head again, of dimensions slice .. + 127 the ``wanted`` eights.
template <int D>
__device__ __forceinline__ void pf_again(const PrefillArgs& a, const PfSpan& sp, int h, int q_first, int groups, int slice,
                                         uint32_t wanted = 0xffff) {
  for (int i = 0; i < groups; ++i) {
    const int q0 = q_first + 16 * i, n = min(sp.nq - q0, 16);
    if (n <= 0) return;
    const int64_t row = ((sp.q0 + q0) * a.H + h) * D;
    pf_again_16<D>(a.q + row, sp.k, sp.v + slice, a.out + row + slice, (int64_t)a.H * D, a.k_pos, a.v_pos, n,
                   q0 + sp.before, sp.nk, a.scale_log2, wanted);
  }
}

// Whether a word of two bf16 holds an infinity or NaN: an exponent of ones carries into the sign's place.
__device__ __forceinline__ bool pf_nonfinite(uint32_t w) {
  return (((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0;
}

// Head dim 256: one workgroup of kPwWaves waves per (query block, head, context).  The block's
// NG = kPwSub * M groups of 16 queries (M = kPwWaves / (D/128)): group gi holds queries qb + 16 gi .. + 15.  Wave w
// holds the 128-dimension slice sl = w % (D/128) of q and O for the groups m + M u (m = w / (D/128), u < kPwSub).
// Per 32-key tile (K and V through LDS once for all waves):
//   1. each wave writes its slice's partial scores S^T = K_sl Q_sl^T of its groups to LDS;  barrier;
//   2. wave w runs the softmax of groups w, w + kPwWaves, ...: adds the D/128 partials in slice order, moves the
//      lazy reference max when needed, and publishes the group's P operand (bf16) and, when the reference max
//      moved, its 16 rescale factors;  barrier;
//   3. each wave rescales its O_sl of a group when told to and adds P V_sl.
// So each group's softmax runs once, not once per slice.  K has one LDS buffer (the next tile's goes in after
// barrier 1, when every wave has read this one), V two (the next tile's goes in during step 3 of this one, into the
// buffer the previous tile's P V read before barrier 1).
constexpr int kPwWaves = 8;
constexpr int kPwSub = 3;  // 16-query groups per wave

__global__ __launch_bounds__(64 * kPwWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void prefill_attn_wide_kernel(
    PrefillArgs a) {
  constexpr int D = 256;
  constexpr int NSL = D / 128, M = kPwWaves / NSL, NG = kPwSub * M, QW = 16 * NG;
  constexpr int OWN = (NG + kPwWaves - 1) / kPwWaves;  // groups whose softmax one wave runs, at most
  constexpr int kRowB = D * 2 + 16;                     // LDS bytes per key row, padded against bank conflicts
  constexpr int kRowChunks = D / 8;                     // 16-byte chunks per key row
  constexpr int kChunks = 32 * kRowChunks / (64 * kPwWaves);  // chunks of K (or of V) per thread per tile
  static_assert(NSL * M == kPwWaves && kChunks * 64 * kPwWaves == 32 * kRowChunks, "whole slices and chunks");
  __shared__ __attribute__((aligned(16))) char kl[32 * kRowB];     // K: 32 key rows
  __shared__ __attribute__((aligned(16))) char vl[2][32 * kRowB];  // V: two tiles
  __shared__ f32x4_t part[NG][NSL][2][64];  // partial scores: [group][slice][block mb][lane]
  __shared__ u32x4_t pex[NG][64];           // P operand of each group: [group][lane]
  __shared__ float alx[NG][16];             // rescale factor of each query of a group (when rflag)
  __shared__ int rflag[NG];                 // the group's reference max moved on this tile
  __shared__ float lsum[NG][16];            // probability sum of each query, at the end
  const int nqb = (a.width + QW - 1) / QW;
  const PfBlock blk = pf_block(nqb, a.H, (int)gridDim.z);
  const int qb = (nqb - 1 - blk.j) * QW;  // the longest blocks first
  const int h = blk.h, b = blk.b;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int sl = w % NSL, m = w / NSL;
  const int64_t slot = clamp64(a.slots[b], 0, a.cache_rows - 1);
  const uint16_t* kbase = a.k + slot * a.s_row + h * a.s_head;
  const uint16_t* vbase = a.v + slot * a.s_row + h * a.s_head;
  const int kend = min(qb + QW, a.width);
  const int nt = (kend + 31) / 32;

  // Global -> LDS through one set of staging registers: thread tid moves 16-byte chunks tid, tid + 64 kPwWaves, ...
  // of a tile's K or V rows.  Rows past the context read its last key (finite: masked by the causal limit).
  u32x4_t stage[kChunks];
  auto fetch = [&](int t, const uint16_t* base) {
#pragma unroll
    for (int e = 0; e < kChunks; ++e) {
      const int ci = tid + e * 64 * kPwWaves, r = ci / kRowChunks, col = ci % kRowChunks;
      const int key = min(t * 32 + r, a.width - 1);
      stage[e] = *reinterpret_cast<const u32x4_t*>(base + (int64_t)key * D + col * 8);
    }
  };
  auto put = [&](char* dst) {
#pragma unroll
    for (int e = 0; e < kChunks; ++e) {
      const int ci = tid + e * 64 * kPwWaves, r = ci / kRowChunks, col = ci % kRowChunks;
      *reinterpret_cast<u32x4_t*>(dst + r * kRowB + col * 16) = stage[e];
    }
  };
  // Whether group gi sees the tile starting at key0: a live group whose last query reaches the tile's first key.
  auto sees = [&](int gi, int key0) { return qb + 16 * gi < a.width && key0 <= qb + 16 * gi + 15; };

  u32x4_t qop[kPwSub][4];  // lane (c, g): q[qb + 16 gi + c][128 sl + 32 s2 + 8g .. +7] (0 past the end)
  f32x4_t o[kPwSub][8];    // output column c of block e: dimension 128 sl + 16 e + c
#pragma unroll
  for (int u = 0; u < kPwSub; ++u) {
    const int row = qb + 16 * (m + M * u) + c;
    const bool live = row < a.width;
    const uint16_t* qrow = a.q + ((int64_t)(b * a.width + (live ? row : 0)) * a.H + h) * D + 128 * sl + g * 8;
#pragma unroll
    for (int s2 = 0; s2 < 4; ++s2)
      qop[u][s2] = live ? *reinterpret_cast<const u32x4_t*>(qrow + s2 * 32) : u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) o[u][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  SoftmaxState st[OWN];  // the softmax state of groups w + kPwWaves r
#pragma unroll
  for (int r = 0; r < OWN; ++r) st[r] = SoftmaxState{-INFINITY, -INFINITY, 0.f};

  fetch(0, kbase);
  put(kl);
  fetch(0, vbase);
  put(vl[0]);
  if (nt > 1) fetch(1, kbase);
  lds_barrier();
  for (int t = 0; t < nt; ++t) {
    const int key0 = t * 32;
    // 1. partial scores of this wave's groups over its slice
    {
      u32x4_t kf[2][4];
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
        const int rk = 8 * (c >> 2) + 4 * mb + (c & 3);
#pragma unroll
        for (int s2 = 0; s2 < 4; ++s2)
          kf[mb][s2] = *reinterpret_cast<const u32x4_t*>(&kl[rk * kRowB + 256 * sl + g * 16 + s2 * 64]);
      }
#pragma unroll
      for (int u = 0; u < kPwSub; ++u) {
        const int gi = m + M * u;
        if (!sees(gi, key0)) continue;
#pragma unroll
        for (int mb = 0; mb < 2; ++mb) {
          f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s2 = 0; s2 < 4; ++s2)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kf[mb][s2]),
                                                          __builtin_bit_cast(bf16x8_t, qop[u][s2]), acc, 0, 0, 0);
          part[gi][sl][mb][lane] = acc;
        }
      }
    }
    lds_barrier();
    if (t + 1 < nt) {
      put(kl);             // every wave has read this tile's K
      fetch(t + 1, vbase);  // the next V, in flight during steps 2 and 3
    }
    // 2. the softmax of this wave's own groups
#pragma unroll
    for (int r = 0; r < OWN; ++r) {
      const int gi = w + kPwWaves * r;
      if (gi >= NG || !sees(gi, key0)) continue;
      const int q0 = qb + 16 * gi;
      f32x4_t sum[2];
#pragma unroll
      for (int mb = 0; mb < 2; ++mb) {
        sum[mb] = part[gi][0][mb][lane];
#pragma unroll
        for (int s3 = 1; s3 < NSL; ++s3) sum[mb] += part[gi][s3][mb][lane];
      }
      float sv[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) sv[j] = sum[j >> 2][j & 3];
      const int lim = q0 + c + 1;
      if (!(key0 + 31 <= q0)) {  // not every query of the group sees the whole tile
#pragma unroll
        for (int j = 0; j < 8; ++j) sv[j] = key0 + 8 * g + j < lim ? sv[j] : -INFINITY;
      }
      bool over = false;
#pragma unroll
      for (int j = 0; j < 8; ++j) over |= sv[j] > st[r].thr;
      const bool moved = __any(over);
      if (moved) {
        float mx = sv[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) mx = fmaxf(mx, sv[j]);
        mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
        mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
        const float m_new = fmaxf(st[r].m_ref, mx * a.scale_log2);
        const float alpha = __builtin_amdgcn_exp2f(st[r].m_ref - (m_new == -INFINITY ? 0.f : m_new));  // -inf: 0
        st[r].l_run *= alpha;
        if (g == 0) alx[gi][c] = alpha;
        st[r].m_ref = m_new;
        st[r].thr = m_new == -INFINITY ? -INFINITY : (m_new + kLazyLog2) / a.scale_log2;
      }
      if (lane == 0) rflag[gi] = moved ? 1 : 0;
      const float m_use = st[r].m_ref == -INFINITY ? 0.f : st[r].m_ref;
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[j], a.scale_log2, -m_use));
        st[r].l_run += p[j];
      }
      u32x4_t pop;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        pop[q] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{p[2 * q], p[2 * q + 1]}), bf16x2_t));
      pex[gi][lane] = pop;
    }
    lds_barrier();
    // 3. O_sl += P V_sl for this wave's groups (rescaled first when the group's reference max moved)
    {
      u32x4_t pop[kPwSub];
#pragma unroll
      for (int u = 0; u < kPwSub; ++u) {
        const int gi = m + M * u;
        if (!sees(gi, key0)) continue;
        if (rflag[gi]) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float al = alx[gi][4 * g + i];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[u][e][i] *= al;
          }
        }
        pop[u] = pex[gi][lane];
      }
      // V operands by transpose reads from this wave's slice of the rows: within 16 lanes, lane 4r + q points at key r,
      // dimensions 4q .. + 3, and lane c receives dimension c of the four keys.
      const int rr = c >> 2, q4 = c & 3;
      const lds_char* vls = (const lds_char*)vl[t & 1];  // vl lives in LDS
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int off = (8 * g + rr) * kRowB + 256 * sl + (16 * e + 4 * q4) * 2;
        const v4i16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vls + off));
        const v4i16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vls + off + 4 * kRowB));
        u32x4_t bop;
        bop[0] = (uint32_t)(uint16_t)lo[0] | ((uint32_t)(uint16_t)lo[1] << 16);
        bop[1] = (uint32_t)(uint16_t)lo[2] | ((uint32_t)(uint16_t)lo[3] << 16);
        bop[2] = (uint32_t)(uint16_t)hi[0] | ((uint32_t)(uint16_t)hi[1] << 16);
        bop[3] = (uint32_t)(uint16_t)hi[2] | ((uint32_t)(uint16_t)hi[3] << 16);
#pragma unroll
        for (int u = 0; u < kPwSub; ++u) {
          if (!sees(m + M * u, key0)) continue;
          o[u][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, pop[u]),
                                                            __builtin_bit_cast(bf16x8_t, bop), o[u][e], 0, 0, 0);
        }
      }
    }
    if (t + 1 < nt) {
      put(vl[(t + 1) & 1]);  // read last by tile t - 1's P V, before this tile's first barrier
      if (t + 2 < nt) fetch(t + 2, kbase);
    }
  }

  // ---- probability sums from the softmax owners, then each group's 16 output rows of this wave's slice
#pragma unroll
  for (int r = 0; r < OWN; ++r) {
    const int gi = w + kPwWaves * r;
    if (gi >= NG) continue;
    float l_tot = st[r].l_run + __shfl_xor(st[r].l_run, 16, kWave);
    l_tot += __shfl_xor(l_tot, 32, kWave);
    if (g == 0) lsum[gi][c] = l_tot;
  }
  lds_barrier();
#pragma unroll
  for (int u = 0; u < kPwSub; ++u) {
    const int gi = m + M * u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int qq = qb + 16 * gi + 4 * g + i;
      if (qq >= a.width) continue;
      const float li = lsum[gi][4 * g + i];
      const float div = li > 0.f ? li : 1.f;
      uint16_t* orow = a.out + ((int64_t)(b * a.width + qq) * a.H + h) * D + 128 * sl;
#pragma unroll
      for (int e = 0; e < 8; ++e) orow[16 * e + c] = (uint16_t)pack_bf16x2(o[u][e][i] / div, 0.f);
    }
  }
}

// Head dim 512: one workgroup of 8 waves per 64 queries, two kinds of waves side by side on each SIMD.  Waves 0..3
// ("scores") compute S^T = K Q^T, the softmax and P; waves 4..7 ("values") compute O^T += V^T P^T one 64-key tile
// behind, so the softmax of a tile runs beside the matrix work of the one before, and a wave holds either Q (32 queries
// x 512 dimensions, 128 registers) or O (64 queries x 128 dimensions, 128 registers), never both.  Both products are
// v_mfma_f32_32x32x16_bf16.  One barrier per tile.
//
//  * Score wave w: queries 32 (w & 1) .. + 31, keys 32 (w >> 1) .. + 31 of the tile, all 512 dimensions.  Lane (x =
//    lane % 32, g = lane / 32) gets query x's scores of keys 8 (i / 4) + 4g + i % 4, i < 16, and writes them as
//    probabilities to LDS, 8 at a time: exactly the lane's B operand of O^T += V^T P^T.
//  * Value wave w: dimensions 128w .. + 127 of all 64 queries.  V comes straight from memory into registers (each
//    wave reads its own quarter of every row: nothing to share through LDS) in 16-byte loads, a whole tile ahead; a lane
//    swap and a byte permute per operand dword transpose it.  Rows past the context read 0 (buffer bounds).  These
//    waves also bring the next tile's K rows to LDS (global_load_lds, one 1 KB row each, rows 1040 bytes apart so
//    that the 32 rows of an operand read start on different banks).
//  * Softmax reference: a query's reference is the maximum of the first tile, and moves only when a score exceeds it
//    by 2^kWsGuard (probabilities are relative, so fp32 and bf16 lose nothing; only their range is used).  Then, and
//    on the first tile, the tile's two key halves exchange their maxima, P is written again and O is rescaled, between
//    two more barriers (uniform over the workgroup: a flag every wave reads after the tile's barrier).
//
// What bounds a tile (64 queries x 64 keys): 2048 clocks of matrix work per SIMD, 2048 of the CU's vector memory path
// (128 KB of K and V at 64 bytes a clock), 1860 of LDS; as a value wave issues its loads and its products in one order, a
// tile takes ~3000 (1.3 us) where one context leaves CUs idle, and ~5200 (2.5 us, 39% of it matrix work) with every CU
// reading its XCD's L2.  The kernel this replaced added the partial scores of four 128-dimension slices through LDS, with
// three barriers per 32 keys of 96 queries (5500 clocks for 1536 of matrix work).  Measured, 8 heads: 8 contexts x 2048
// 521 -> 357 us (770 TFLOP/s; in chains 329, see ws_group); one context of 1433, where the longest block is the launch,
// 110 -> 38 us.  Tried: 8-byte V loads of the operand's own rows, 390 / 45 us (the memory path takes a load instruction
// per 64 lanes, not only its bytes); the loads spread between the products, 390-430 us (the tile's rows arrive later and
// its products compete with the scores'); K rows brought by the score waves, 404 us; wave priorities, no change.
constexpr int kWsD = 512, kWsQ = 64, kWsK = 64;
constexpr int kWsRow = kWsD * 2 + 16;  // LDS bytes per K row
constexpr int kWsAhead = 4;
constexpr float kWsGuard = 16.0f;

__device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                 0, 0);
}

// A wave-uniform pointer in scalar registers.
__device__ __forceinline__ const char* scalar_pointer(const void* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<const char*>((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)u) |
                                       (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32);
}

// Chains: a workgroup fills a CU's LDS, so with more blocks than CUs each block's start (first K tile and Q, 6-7 us)
// and end (2-3 us) stood between the tiles of two blocks.  In a chain the next block's first tile is the tile after the
// last: its K and V are on the way and its scores run beside the last values of the block before.  XCD x's blocks, those
// of units (head, context) x, x + 8, .., are listed group after group of ``group`` units, within a group the longest
// blocks first, and dealt to the XCD's kWsPerXcd workgroups there and back, so that long and short blocks even out.
constexpr int kWsPerXcd = 32;  // workgroups at a time: one per CU

// The longest chain of an XCD's workgroups, in tiles (and one for each block), with ``group`` units listed together: the
// deal of prefill_attn_ws_kernel's ``place``, block after block.
inline int ws_longest(int nqb, int units8, int group) {
  int tiles[kWsPerXcd] = {}, c = 0, step = 1;
  for (int g0 = 0; g0 < units8; g0 += group) {
    const int members = std::min(group, units8 - g0);
    for (int t = nqb; t > 0; --t) {
      for (int m = 0; m < members; ++m) {
        tiles[c] += t + 1;
        c += step;
        if (c == kWsPerXcd || c < 0) {  // there and back: the end's workgroup takes two in a row
          step = -step;
          c += step;
        }
      }
    }
  }
  return *std::max_element(tiles, tiles + kWsPerXcd);
}

// The units in a group, 0 for no chains: what is predicted to end first, in tiles.
//  * No chains: an even share of the XCD's tiles and two for each block's start and end, and nqb / 4 for what the last
//    blocks leave idle.
//  * Groups of up to 8 units, or one of all: the longest chain of the deal (whether groups end with a round decides: at
//    8 x 1433 two units at a time take 201 us, all 193, no chains 199, at 8 x 1536 199, 209 and 228), 0.1% longer for each
//    block of a group past 128, whose K and V the XCD's L2 no longer holds (16 x 1024, even chains all: 214 us with 2
//    units, 225 with 8, 253 with 16), and 2% for a unit alone (8 x 2048 336, with 2 330).
// Below two rounds nothing evens out (2 contexts x 1433, 1.4 rounds: 49.5 us in chains, 47.9 without), nor with one unit,
// whose longest block is the launch (1 x 4100: 152, 146).
// Measured at 103 shapes, 8 heads, 2 to 16 contexts x 330 to 3000, every group size, repeated on one state: the choice is
// within 1% of the best one on the mean, 14% at most (16 x 640, 126 us against 111).  us, 8 contexts x width, without
// chains / in the chosen groups: 500 42 / 37, 1984 317 (none chosen; 343 with all 8), 2048 360 / 330, 2049 369 / 354, 2300
// 432 / 398, 2560 507 / 488, 3000 640 (none); 5 x 1024 84 / 74; 12 x 500 78 / 64; 16 x 1536 443 / 391.  The choice takes
// the host ~2 ns for each block of each candidate.
inline int ws_group(int nqb, int units8) {
  if ((int64_t)nqb * units8 < 2 * kWsPerXcd || units8 < 2) return 0;
  const float n = (float)nqb;
  float least = (float)units8 * n * ((n + 1.f) * 0.5f + 2.f) / kWsPerXcd + 0.25f * n;
  int pick = 0;
  for (int i = 1; i <= std::min(units8, 9); ++i) {
    const int group = i == 9 ? units8 : i;
    const float spilled = (float)std::max((int64_t)group * nqb - 128, (int64_t)0);
    const float tiles =
        (float)ws_longest(nqb, units8, group) * (1.f + 0.001f * spilled) * (group == 1 ? 1.02f : 1.f);
    if (tiles < least) {
      least = tiles;
      pick = group;
    }
  }
  return pick;
}

// Packed prompts in chains: the blocks of an XCD's heads (the same for each head) in a list, sequence by sequence, those with
// the most work and their longest blocks first, heads beside each other.  32 blocks at a time are dealt to its workgroups, the
// longest to the one with the fewest tiles so far.  Every workgroup does that for itself from the lengths, in ~3 us of a
// launch.
// Measured, us, blocks one by one and in chains: 8 heads x 512, 8 prompts of 750-2400 218 / 195, of 300-700 59 / 52, 32
// of 100-800 169 / 133, 64 of 20-600 229 / 171, 8 of 3000-6000 1338 / 1346.  At head dim 128, where only the next
// block's first K tile is brought beside a block's output: 32 heads, 4 of 2048 201 / 169, 64 of 20-600 258 / 216, 16 of
// up to 500 behind up to 900 keys 106 / 91; 32 over 8 heads, 32 of 100-800 137 / 120, 16 of up to 500 behind up to 900
// 81 / 81, 8 of 3000-6000 1167 / 1200; at head dim 256, 16 over 2 heads, 32 of 100-800 144 / 121, 64 of 20-600 203 /
// 156.  Dealt there and back instead, groups of sequences each longest first (head dim 512): 8 of 750-2400 223, of
// 3000-6000 1445.
constexpr int kPfRounds = 128;
constexpr int kPfListBytes = kPfRounds * kWsPerXcd * 8;

struct PfChain {
  PfSequence seqs[kWave];  // by rank
  int list[kPfRounds];     // the chain: sequence << 24 | query block << 12 | of the XCD's blocks of heads; -1 behind the last
  uint32_t redo[4][kPfRounds / 32];  // [value wave]: rounds with outputs that are not finite
};

// Blocks of ``queries``, ``heads`` blocks of heads.  ``scratch``: kPfListBytes.  Queries of blocks that see no key are zeroed.
template <int D>
__device__ __forceinline__ void pf_chain(const PrefillArgs& a, int queries, int heads, PfChain& c, char* scratch) {
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  {
    const PfSequence one = pf_sequence(a, min(lane, a.sequences - 1));
    const int rank = pf_rank(one, a.sequences);
    if (w == 0 && lane < a.sequences) c.seqs[rank] = one;
    if (tid < 4 * (kPfRounds / 32)) c.redo[tid % 4][tid / 4] = 0;
  }
  lds_barrier();
  // A lane's sequence, and its blocks: ``seen`` that see a key, of which ``upto`` come up to its end.
  const PfSequence mine = c.seqs[min(lane, a.sequences - 1)];
  const int nq = min(mine.nq, a.width), before = mine.nk - mine.nq;
  const int blocks = lane < a.sequences ? (nq + queries - 1) / queries : 0;
  const int blind = before >= 0 || blocks == 0 ? 0 : nq + before <= 0 ? blocks : min(blocks - 1, -before / queries);
  const int seen = blocks - blind, upto = wave_scan(seen);
  const int members = heads / 8, listed = __builtin_amdgcn_readlane(upto, kWave - 1) * members;
  // Rounds of 32 blocks by their time, each wave some.  (A tile of one 64-query group takes ~0.9 us, of four, at head dim 128,
  // ~1.6; a start and end what half a tile takes.)
  u32x2_t(*sorted)[kWsPerXcd] = reinterpret_cast<u32x2_t(*)[kWsPerXcd]>(scratch);
  auto of = [&](int from, int v) { return __builtin_amdgcn_ds_bpermute(from * 4, v); };
  for (int round = w; round < kPfRounds && round * kWsPerXcd < listed; round += 8) {
    const int p = round * kWsPerXcd + (lane & 31), i = p / members;
    int s = 0;
    for (int t = 0; t < a.sequences - 1; ++t) s += __builtin_amdgcn_readlane(upto, t) <= i ? 1 : 0;
    const int j = of(s, blocks) - 1 - (i - (of(s, upto) - of(s, seen)));
    const int end = min(queries * (j + 1), of(s, nq)), groups = (end - queries * j + 63) / 64 * a.together;
    const uint32_t tiles = (uint32_t)(end + of(s, before) + 63) / 64;
    const uint32_t cost = p < listed ? tiles * (3 + groups) + 2 : 0;
    int rank = 0;
#pragma unroll 4
    for (int t = 0; t < kWsPerXcd; ++t) {
      const uint32_t other = __builtin_amdgcn_readlane(cost, t);
      rank += other > cost || (other == cost && t < (lane & 31)) ? 1 : 0;
    }
    if (lane < kWsPerXcd)
      sorted[round][rank] = u32x2_t{cost, p < listed ? (uint32_t)(s << 24 | j << 12 | (p - i * members)) : ~0u};
  }
  // Blocks that see no key at all.
  for (uint64_t with = __ballot(blind > 0); with; with &= with - 1) {
    const int s = __builtin_ctzll(with), n = __builtin_amdgcn_readlane(blind, s);
    const int64_t q0 = pf_readlane64(mine.q0, s), end = q0 + __builtin_amdgcn_readlane(nq, s);
    for (int64_t i = blockIdx.x; i < (int64_t)n * a.H; i += gridDim.x) {
      const int64_t at = q0 + i / a.H * queries;
      pf_zeros<D>(a, at, at + queries < end ? at + queries : end, (int)(i % a.H));
    }
  }
  lds_barrier();
  if (w == 0) {
    uint32_t load = 0;  // of the XCD's workgroup lane % 32
    for (int round = 0; round < kPfRounds; ++round) {
      if (round * kWsPerXcd >= listed) {
        if (lane == 0) c.list[round] = -1;
        break;
      }
      int rank = 0;
#pragma unroll 4
      for (int t = 0; t < kWsPerXcd; ++t) {
        const uint32_t other = __builtin_amdgcn_readlane(load, t);
        rank += other < load || (other == load && t < (lane & 31)) ? 1 : 0;
      }
      const u32x2_t its = sorted[round][rank];
      load += its[0];
      if (lane == (int)blockIdx.x / 8) c.list[round] = (int)its[1];
    }
  }
  lds_barrier();
}

// The block of a round of the chain: sequence (by rank), query block, block of heads; false past its end.
struct PfListed {
  int s, j, h;
};
__device__ __forceinline__ bool pf_listed(const PfChain& c, int round, int heads, PfListed& at) {
  const int e = round < kPfRounds ? __builtin_amdgcn_readfirstlane(c.list[round]) : -1;
  if (e < 0) return false;
  at = PfListed{e >> 24, e >> 12 & 0xfff, (int)blockIdx.x % 8 * (heads / 8) + (e & 0xfff)};
  return true;
}
__device__ __forceinline__ PfSequence pf_of(const PfChain& c, int s) {
  const PfSequence& q = c.seqs[s];
  return PfSequence{pf_readlane64(q.q0, 0), pf_readlane64(q.k0, 0), __builtin_amdgcn_readfirstlane(q.nq),
                    __builtin_amdgcn_readfirstlane(q.nk)};
}

// A query block of a workgroup at head dim 512, its chain's ``round``-th.
struct WsBlock {
  int round, qb, h, b;
};
struct WsTile {  // key tile t of a block, the last its ``last``
  WsBlock blk;
  int t, last, nk;
  const char *kbase, *vbase;
};

template <bool kChain, bool kPacked>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void prefill_attn_ws_kernel(PrefillArgs a) {
  constexpr int D = kWsD;
  __shared__ __attribute__((aligned(16))) char kls[2][kWsK * kWsRow];
  __shared__ u32x4_t ps[2][2][4][64];  // [tile parity][query half][16-key step][lane]
  __shared__ float mxs[2][kWsQ];       // a tile's maxima by key half, when the reference moves
  __shared__ float als[kWsQ];          // then: the factors O is rescaled by
  __shared__ float lsum[2][2][2][kWsQ];  // [parity of the block in the chain]: probability sums by key half, lane half
  __shared__ int moved[4];             // by tile % 4: a score passed the guard
  constexpr bool kListed = kChain && kPacked;
  static_assert(kPfListBytes <= sizeof(kls), "");
  __shared__ char chain_at[kListed ? sizeof(PfChain) : 1] __attribute__((aligned(16)));
  PfChain& chain = *reinterpret_cast<PfChain*>(chain_at);
  const int nqb = (a.width + kWsQ - 1) / kWsQ;
  const int tid = threadIdx.x, lane = tid & 63, x = lane & 31, g = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (tid < 4) moved[tid] = 0;
  // The workgroup's block of a round, from its XCD's list; false past its end.
  auto place = [&](WsBlock& blk, int round) {
    if constexpr (kListed) {
      PfListed at;
      if (!pf_listed(chain, round, a.H, at)) return false;
      blk = WsBlock{round, at.j * kWsQ, at.h, at.s};
      return true;
    }
    const int c = (int)blockIdx.x / 8;
    const int p = round * kWsPerXcd + (round & 1 ? kWsPerXcd - 1 - c : c);
    if (p >= a.units8 * nqb) return false;
    const int full = a.group * nqb, g0 = p / full * a.group, r = p % full, members = min(a.group, a.units8 - g0);
    const int unit = (g0 + r % members) * 8 + (int)blockIdx.x % 8;
    blk = WsBlock{round, (nqb - 1 - r / members) * kWsQ, unit % a.H, unit / a.H};
    return true;
  };
  WsBlock only;  // packed: the one block of the workgroup, and its span
  PfSpan only_span;
  PfPacked one = {};
  if constexpr (kListed) {
    pf_chain<D>(a, kWsQ, a.H, chain, &kls[0][0]);
    if (chain.list[0] < 0) return;
  } else if constexpr (kPacked) {
    one = pf_packed_block(a, nqb, kWsQ, a.H, (int)gridDim.z / a.parts);
    only = WsBlock{0, (nqb - 1 - one.j) * kWsQ, one.h, 0};
    only_span = pf_packed_span(a, one.h, one.s);
    if (only.qb >= only_span.nq) return;
    const int end = min(only.qb + kWsQ, only_span.nq);
    int keys = end + only_span.before;
    if (!pf_part(a, one, only_span, keys)) return;
    if (keys <= 0) return pf_zeros<D>(a, only_span.q0 + only.qb, only_span.q0 + end, only.h);
  }
  auto first = [&]() {
    WsBlock blk;
    if constexpr (kChain) {
      place(blk, 0);
    } else if constexpr (kPacked) {
      blk = only;
    } else {
      const PfBlock one = pf_block(nqb, a.H, (int)gridDim.z);
      blk = WsBlock{0, (nqb - 1 - one.j) * kWsQ, one.h, one.b};  // the longest blocks first
    }
    return blk;
  };
  auto next = [&](WsBlock& blk) {  // false (and blk as it was): that was the last
    if constexpr (kChain) return place(blk, blk.round + 1);
    return false;
  };
  auto span = [&](const WsBlock& blk) {
    if constexpr (kListed) {
      return pf_packed_span(a, blk.h, pf_of(chain, blk.b));
    }
    if constexpr (kPacked) return only_span;
    return pf_span<D>(a, blk.h, blk.b);
  };
  // The block's last tile: the one of its last query's last key, or of the part's.
  auto last_tile = [&](const WsBlock& blk, const PfSpan& sp) {
    return kPacked ? (min(min(blk.qb + kWsQ, sp.nq) + sp.before, sp.nk) - 1) / kWsK : blk.qb / kWsK;
  };

  if (w < 4) {  // ------------------------------------------------------------------------------ scores
    const int qh = w & 1, kh = w >> 1;
    // K operands in a ring kWsAhead steps ahead of the products: an LDS read takes a few products' time to arrive.
    u32x4_t kf[kWsAhead];
    auto k_at = [&](int t, int s) {
      return *reinterpret_cast<const u32x4_t*>(&kls[t & 1][(32 * kh + x) * kWsRow + g * 16 + s * 32]);
    };
    WsBlock blk = first();
    int t = 0;  // counted over the workgroup's blocks, as is all LDS
    for (int odd = 0;; odd ^= 1) {
      const PfSpan sp = span(blk);
      const int qb = blk.qb, query = qb + 32 * qh + x, t_first = t;
      const int t_last = t + last_tile(blk, sp);  // the last tile holds the diagonal
      u32x4_t q[D / 16];  // q[query][16s + 8g .. + 7] (past the end the last query's: its results are not stored)
      {
        const uint16_t* qrow = a.q + ((sp.q0 + min(query, sp.nq - 1)) * a.H + blk.h) * D + g * 8;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) q[s] = *reinterpret_cast<const u32x4_t*>(qrow + s * 16);
      }
      float m_ref = -INFINITY, thr = -INFINITY, l_run = 0.f;
      if (t == 0) {
        lds_barrier();  // the first K tile
#pragma unroll
        for (int s = 0; s < kWsAhead; ++s) kf[s] = k_at(0, s);
      }
      for (; t <= t_last; ++t) {
        f32x16_t s0, s1;
#pragma unroll
        for (int i = 0; i < 16; ++i) s0[i] = s1[i] = 0.f;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          if (s & 1) s1 = mfma32(kf[s % kWsAhead], q[s], s1);
          else s0 = mfma32(kf[s % kWsAhead], q[s], s0);
          if (s + kWsAhead < D / 16) {
            kf[s % kWsAhead] = k_at(t, s + kWsAhead);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // one product, one LDS read
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          }
        }
        float sv[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) sv[i] = s0[i] + s1[i];
        const int whole = kPacked ? qb + sp.before - (t - t_first) * kWsK : 0;  // of the tile's keys, seen by every query
        if (kPacked ? whole < kWsK - 1 : t == t_last) {
          const int rel = whole + 32 * qh + x - (32 * kh + 4 * g);  // keys 8 (i / 4) + i % 4 <= rel are seen
#pragma unroll
          for (int i = 0; i < 16; ++i) sv[i] = 8 * (i >> 2) + (i & 3) <= rel ? sv[i] : -INFINITY;
        }
        bool over = false;
#pragma unroll
        for (int i = 0; i < 16; ++i) over |= sv[i] > thr;
        if (__any(over) && lane == 0) moved[t & 3] = 1;
        float lt = 0.f;
        // Probabilities as the value waves' operand: bf16, what the matrix instruction takes, each rounded once (2^-8 of itself
        // at most); their sum is of the unrounded ones, in fp32.
        auto put_p = [&](float m) {
          lt = 0.f;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            u32x4_t pop;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[8 * s + 2 * e], a.scale_log2, -m));
              const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[8 * s + 2 * e + 1], a.scale_log2, -m));
              lt += p0 + p1;
              pop[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{p0, p1}), bf16x2_t));
            }
            ps[t & 1][qh][2 * kh + s][lane] = pop;
          }
        };
        put_p(m_ref == -INFINITY ? 0.f : m_ref);
        lds_barrier();
        const int again = moved[t & 3];  // uniform over the workgroup
#pragma unroll
        for (int s = 0; s < kWsAhead; ++s) kf[s] = k_at(t + 1, s);  // (past the last tile: unused)
        if (w == 0 && lane == 0) moved[(t + 2) & 3] = 0;
        if (again) {
          float mx = sv[0];
#pragma unroll
          for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sv[i]);
          mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
          if (g == 0) mxs[kh][32 * qh + x] = mx;
          lds_barrier();
          const float m_new = fmaxf(m_ref, fmaxf(mxs[0][32 * qh + x], mxs[1][32 * qh + x]) * a.scale_log2);
          const float alpha = __builtin_amdgcn_exp2f(m_ref - (m_new == -INFINITY ? 0.f : m_new));  // m_ref = -inf: 0
          if (kh == 0 && g == 0) als[32 * qh + x] = alpha;
          l_run *= alpha;
          m_ref = m_new;
          thr = m_new == -INFINITY ? -INFINITY : (m_new + kWsGuard) / a.scale_log2;
          put_p(m_ref == -INFINITY ? 0.f : m_ref);
          lds_barrier();
        }
        l_run += lt;
      }
      lsum[odd][kh][g][32 * qh + x] = l_run;
      if (kPacked && !kChain && pf_in_parts(one)) pf_leave_ml(a, one, w, g, x, m_ref, l_run);
      if (!next(blk)) break;
    }
    lds_barrier();
    return;
  }

  // ---------------------------------------------------------------------------------------------- values
  const int vw = w - 4;
  // [query half][e]: row r is dimension 128 vw + 8 (r % 16) + 4 (r / 16) + e, column x query x of the half
  f32x16_t o[2][4];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[u][e][i] = 0.f;
  // K rows 16 vw .. + 15 of tile t to LDS, one row (64 lanes x 16 bytes) per load; rows past the context read its last
  // key (finite: masked).
  auto bring_k = [&](const WsTile& c, int n) {  // as tile n of the workgroup
    const uint32_t row_bytes = kPacked ? (uint32_t)a.k_pos * 2 : D * 2;
    const int t0 = kPacked ? c.t * kWsK : 0;  // packed rows may be far apart: their offsets within the tile
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(c.kbase + (int64_t)t0 * row_bytes), 0, -1, 0x00020000);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int key = min(c.t * kWsK + 16 * vw + r, (kPacked ? c.nk : a.width) - 1) - t0;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          kr, (__attribute__((address_space(3))) void*)&kls[n & 1][(16 * vw + r) * kWsRow], 16, lane * 16,
          (int)((uint32_t)key * row_bytes), 0,
          0);
    }
  };
  // V of 16-key step s of tile t: lane (c = x % 16, u = x / 16, g) loads keys 16s + 8u + 4g + j, dimensions 128 vw + 8c
  // .. + 7, j < 4.  A buffer resource per step, its size what is left of the context's rows: scalar work only, and rows
  // past the end read 0.
  const uint32_t v_bytes = kPacked ? (uint32_t)a.v_pos * 2 : D * 2;
  const uint32_t vlane = (uint32_t)(8 * (x >> 4) + 4 * g) * v_bytes + (uint32_t)(128 * vw + 8 * (x & 15)) * 2;
  const uint32_t vbytes = (uint32_t)a.width * (D * 2);
  u32x4_t v[4][4];
  auto load_v = [&](const WsTile& c, int s) {
    const char* from;
    uint32_t room;  // bytes from there that are the context's
    if constexpr (kPacked) {
      const int at = c.t * kWsK + 16 * s, rows = min(c.nk - at, 16);
      from = c.vbase + (int64_t)at * v_bytes;
      room = rows > 0 ? (uint32_t)(rows - 1) * v_bytes + D * 2 : 0;
    } else {
      const uint32_t off = (uint32_t)(c.t * kWsK + 16 * s) * (D * 2);
      uint32_t used = min(off, vbytes);
      asm("" : "+s"(used));  // kept scalar (the saturating subtraction it would become is a vector instruction)
      from = c.vbase + off;
      room = vbytes - used;
    }
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(from), 0, room, 0x00020000);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[s][j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(vr, vlane + j * v_bytes, 0, 0));
  };
  u32x4_t p[2][2];  // steps s, s + 1 of tile t
  auto read_p = [&](int t, int s) {
#pragma unroll
    for (int u = 0; u < 2; ++u) p[u][s & 1] = ps[t & 1][u][s][lane];
  };
  // O^T += V^T P^T for the workgroup's tile t; ``ahead``: the next tile's V loads as its registers fall free.  Step
  // s + 1's operands are built beside step s's products; the scheduler keeps each step's loads behind the permutes that read
  // their registers.
  auto attend_v = [&](int t, const WsTile* ahead) {
    u32x4_t vop[2][4];
    auto operands = [&](int s) {
      // The lanes of a pair (u = 0, 1) hold 8 dimensions of 4 keys each; swapped, 4 dimensions (8c + 4u ..) of 8 keys:
      // lo[j] of key 16s + 4g + j, hi[j] of key 16s + 8 + 4g + j.
      u32x2_t lo[4], hi[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const auto r = __builtin_amdgcn_permlane16_swap(v[s][j][d], v[s][j][2 + d], false, false);
          lo[j][d] = r[0];
          hi[j][d] = r[1];
        }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t sel = (e & 1) ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int q2 = 0; q2 < 2; ++q2) {
          vop[s & 1][e][q2] = __builtin_amdgcn_perm(lo[2 * q2 + 1][e >> 1], lo[2 * q2][e >> 1], sel);
          vop[s & 1][e][2 + q2] = __builtin_amdgcn_perm(hi[2 * q2 + 1][e >> 1], hi[2 * q2][e >> 1], sel);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(vop[s & 1][e]));  // built here, not where first used
    };
    operands(0);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      __builtin_amdgcn_sched_barrier(0);
      if (ahead) load_v(*ahead, s);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int u = 0; u < 2; ++u) o[u][e] = mfma32(vop[s & 1][e], p[u][s & 1], o[u][e]);
      if (s < 2) read_p(t, s + 2);
      if (s < 3) operands(s + 1);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // After tile t's barrier: its probabilities, and O rescaled when the reference moved on it (O holds the tiles
  // before it).
  auto take_p = [&](int t) {
    const int again = moved[t & 3];
    read_p(t, 0);
    read_p(t, 1);
    if (!again) return;
    lds_barrier();
    lds_barrier();
    read_p(t, 0);
    read_p(t, 1);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float al = als[32 * u + x];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[u][e][i] *= al;
    }
  };
  auto output = [&](const WsBlock& blk, int odd) {  // O of a finished block; then O is 0 again
    const PfSpan sp = span(blk);
    bool again = false;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int query = blk.qb + 32 * u + x;
      const float l = (lsum[odd][0][0][32 * u + x] + lsum[odd][0][1][32 * u + x]) +
                      (lsum[odd][1][0][32 * u + x] + lsum[odd][1][1][32 * u + x]);
      const float inv = l > 0.f ? 1.f / l : 1.f;
      uint16_t* orow = a.out + ((sp.q0 + query) * a.H + blk.h) * D + 128 * vw + 32 * g;
      auto pair = [&](float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{lo * inv, hi * inv}), bf16x2_t));
      };
      if (query < sp.nq) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // dimensions 64r + 32g + 8i + 4k + e, k = 0, 1
            u32x4_t out;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int at = 4 * (r + 2 * k) + i;
              out[2 * k] = pair(o[u][0][at], o[u][1][at]);
              out[2 * k + 1] = pair(o[u][2][at], o[u][3][at]);
            }
            *reinterpret_cast<u32x4_t*>(orow + 64 * r + 8 * i) = out;
            if constexpr (kPacked) {
#pragma unroll
              for (int k = 0; k < 4; ++k) again |= pf_nonfinite(out[k]);
            }
          }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[u][e][i] = 0.f;
    }
    if (kPacked && __any(again)) {
      if constexpr (kListed) chain.redo[vw][blk.round >> 5] |= 1u << (blk.round & 31);
      else pf_again<D>(a, sp, blk.h, blk.qb, 4, 128 * vw);
    }
  };
  auto open = [&](WsTile& c) {  // the block's first tile
    const PfSpan sp = span(c.blk);
    c.kbase = scalar_pointer(sp.k);
    c.vbase = scalar_pointer(sp.v);
    c.nk = sp.nk;
    c.last = last_tile(c.blk, sp);
    c.t = 0;
  };
  auto advance = [&](WsTile& c) {  // false (and c as it was): no more tiles
    if (c.t < c.last) {
      ++c.t;
      return true;
    }
    if (!next(c.blk)) return false;
    open(c);
    return true;
  };
  WsTile at, ahead;  // the tiles whose V and whose K come next
  at.blk = first();
  open(at);
  bring_k(at, 0);
  bool more;
  if constexpr (kPacked) {
    // All of the start's loads at once, then waits for the first K tile (32 loads behind it) and the second (16).
    __builtin_amdgcn_sched_barrier(0);
    ahead = at;
    more = advance(ahead);
    bring_k(ahead, 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < 4; ++s) load_v(at, s);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x8f70);  // vmcnt(32)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_s_waitcnt(0x4f70);  // vmcnt(16)
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  } else {
    landed_barrier();
    ahead = at;
    more = advance(ahead);
    bring_k(ahead, 1);
#pragma unroll
    for (int s = 0; s < 4; ++s) load_v(at, s);
    landed_barrier();
  }
  take_p(0);
  int n = 1, odd = 0;
  while (more) {  // tile n's scores, tile n - 1's values
    const WsBlock was = at.blk;
    at = ahead;
    more = advance(ahead);
    bring_k(ahead, n + 1);  // unconditional (past the last tile: that tile again, not used): no wait joins a branch
    attend_v(n - 1, &at);
    // vmcnt(16): tile n + 1's K rows are in LDS, tile n's 16 V loads, issued after them, stay in flight (lds_barrier
    // would wait for those too).  This wave's LDS reads of the tile are in registers by now.
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x4f70);
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    if (kChain && at.t == 0) {
      output(was, odd);
      odd ^= 1;
    }
    take_p(n);
    ++n;
  }
  attend_v(n - 1, nullptr);
  lds_barrier();
  if (kPacked && !kChain && pf_in_parts(one)) return pf_leave_o(a, one, vw, lane, only_span.nq - only.qb, o);
  output(at.blk, odd);
  if constexpr (kListed) {
    WsBlock blk = first();
    do {
      if (chain.redo[vw][blk.round >> 5] >> (blk.round & 31) & 1) pf_again<D>(a, span(blk), blk.h, blk.qb, 4, 128 * vw);
    } while (next(blk));
  }
}

// Head dim 128: 256 queries per workgroup, four pairs of a score wave and a value wave (see prefill_attn_ws_kernel), each
// pair its own 64 queries against the same 64-key tiles.  Score wave p of step t multiplies tile t (K from LDS, Q in
// registers) beside the softmax of tile t - 1, so its matrix and vector work overlap within the wave; value wave p
// accumulates tile t - 2.  A pair keeps its own softmax reference (a lane's two queries see every key of the tile
// through lanes x and x + 32), so a moved reference costs no barrier: the factors wait in LDS for the value wave.
// K and V rows go to LDS by direct loads (score waves bring V, value waves K: neither reads what it brings, so its
// loads are waited for at the step's barrier alone, landed_barrier), 1 KB = 4 rows each, 16-byte chunks permuted within
// a row so that the operand reads spread over the banks: chunk c of key r at position c ^ (r % 16) in K, c ^ 4 (r % 4)
// in V.
//
// What bounds a tile (a pair's 64 queries x 64 keys): 2048 clocks of matrix work on its SIMD beside ~1900 of the score
// wave's vector work (64 exponentials per lane at a quarter rate), one barrier per tile.  The kernel this replaced ran
// both in one wave, one after the other, on 16 x 16 products with 192 queries per workgroup.  Measured, 32 heads, before
// and after: 4 contexts x 1777 203 -> 147 us (705 TFLOP/s), 8 x 2048 405 -> 362 us (760), one of 1433 64 -> 42 us, 8 of
// 130 16 -> 13 us.  Tried: fmaxf in place of max3, 157 / 387 us; K operands 3 steps ahead (3 registers spilled) with
// the products and the vector work interleaved by sched_group_barrier, 151 / 378 us; wave priorities, no change.
constexpr int kPairQ = 256, kPairK = 64;

// Without the copy of each operand that fmaxf makes to quiet a signalling NaN (a product has none).  The compiler does
// not see an instruction that reads a, b, c here: a caller with values of the matrix unit waits for them first.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// kChain (packed): a workgroup runs a list of blocks, see pf_chain.
template <bool kPacked, bool kChain>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void prefill_attn_pairs_kernel(
    PrefillArgs a) {
  constexpr int D = 128;
  __shared__ __attribute__((aligned(16))) char kls[2][kPairK * D * 2];
  __shared__ __attribute__((aligned(16))) char vls[2][kPairK * D * 2];
  __shared__ u32x4_t ps[4][2][2][4][64];  // [pair][tile parity][query half][16-key step][lane]
  __shared__ float als[4][4][64];         // [pair][tile % 4]: O's factors, when the reference moved
  __shared__ int moved[4][4];
  __shared__ float lsum[4][2][64];        // [pair][lane half]
  static_assert(kPfListBytes <= sizeof(kls), "");
  __shared__ char chain_at[kChain ? sizeof(PfChain) : 1] __attribute__((aligned(16)));
  PfChain& chain = *reinterpret_cast<PfChain*>(chain_at);
  // The pairs' 64 queries: of one head one after another, or (packed) of 2 or 4 heads that read the same keys.
  const int together = kPacked ? a.together : 1, queries = kPacked ? a.block : kPairQ;
  const int nqb = (a.width + queries - 1) / queries;
  const int tid = threadIdx.x, lane = tid & 63, x = lane & 31, g = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), pr = w & 3;
  PfPacked one = {};
  PfSpan sp;
  int qb, h, keys;  // the block's first query, the pair's head, what the block's last query sees (packed: of the part's)
  // The chain's block of ``round``; false past its end.
  auto enter = [&](int round) {
    PfListed at;
    if (!pf_listed(chain, round, a.H / together, at)) return false;
    qb = at.j * queries;
    h = at.h * together + pr % together;
    sp = pf_packed_span(a, h, pf_of(chain, at.s));
    keys = min(qb + queries, sp.nq) + sp.before;
    return true;
  };
  if constexpr (kChain) {
    pf_chain<D>(a, queries, a.H / together, chain, &kls[0][0]);
    if (!enter(0)) return;
  } else if constexpr (kPacked) {
    one = pf_packed_block(a, nqb, queries, a.H / together, (int)gridDim.z / a.parts);
    qb = (nqb - 1 - one.j) * queries;  // the longest blocks first
    h = one.h * together + pr % together;
    sp = pf_packed_span(a, h, one.s);
    keys = min(qb + queries, sp.nq) + sp.before;
    if (qb >= sp.nq) return;
    if (!pf_part(a, one, sp, keys)) return;
    if (keys <= 0) {
      for (int i = 0; i < together; ++i)
        pf_zeros<D>(a, sp.q0 + qb, sp.q0 + min(qb + queries, sp.nq), one.h * together + i);
      return;
    }
  } else {
    const PfBlock blk = pf_block(nqb, a.H, (int)gridDim.z);
    qb = (nqb - 1 - blk.j) * queries;
    h = blk.h;
    sp = pf_span<D>(a, h, blk.b);
    keys = min(qb + queries, sp.nq) + sp.before;
  }
  const char *kbase, *vbase;
  int nt, qp, dq, whole;  // tiles; the pair's first query, its last tile, and the last key that all its queries see
  auto derive = [&]() {
    kbase = scalar_pointer(sp.k);
    vbase = scalar_pointer(sp.v);
    nt = (keys + kPairK - 1) / kPairK;
    qp = qb + 64 * (kPacked ? pr / together : pr);
    if (kPacked && qp >= qb + queries) qp = sp.nq;  // a block of fewer pairs
    // The pair's last tile holds its diagonal (-1: no queries, or they see no key).
    const int lastk = kPacked ? min(min(qp + 64, sp.nq) + sp.before, keys) - 1 : qp;
    dq = qp < sp.nq && lastk >= 0 ? lastk / kPairK : -1;
    whole = qp + sp.before;
  };
  derive();

  // Rows 16 pr .. + 15 of tile t to LDS; rows past the context read its last key (finite: masked).  ``swap``: the chunk
  // permutation of key row r of a 16-row group.
  auto bring = [&](const char* base, uint32_t row_bytes, char* dst, int t, auto swap) {
    // Packed rows may be far apart: a resource per tile, its rows' offsets within it.
    const int t0 = kPacked ? t * kPairK : 0;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(base + (int64_t)t0 * row_bytes), 0, -1, 0x00020000);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = 4 * j + (lane >> 4);
      const int key = min(t * kPairK + 16 * pr + r, sp.nk - 1) - t0;
      const uint32_t from = (uint32_t)key * row_bytes + (uint32_t)((lane & 15) ^ swap(r)) * 16;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void*)(dst + (16 * pr + 4 * j) * (D * 2)), 16, from, 0, 0, 0);
    }
  };

  if (w < 4) {  // ------------------------------------------------------------------------------ scores
    auto bring_v = [&](int t) { bring(vbase, sp.v_bytes, vls[t & 1], t, [](int r) { return 4 * (r & 3); }); };
    for (int round = 0;; ++round) {
      u32x4_t q[2][D / 16];  // q[query][16s + 8g .. + 7], query qp + 32u + x
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint16_t* qrow =
            a.q + ((sp.q0 + min(qp + 32 * u + x, sp.nq - 1)) * a.H + h) * D + g * 8;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) q[u][s] = *reinterpret_cast<const u32x4_t*>(qrow + s * 16);
      }
      float m_ref[2] = {-INFINITY, -INFINITY}, thr[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
      const int klane = x * (D * 2) + ((g ^ (x & 15)) * 16);
      auto k_at = [&](int t, int m, int s) {
        return *reinterpret_cast<const u32x4_t*>(&kls[t & 1][32 * m * (D * 2) + (klane ^ (32 * s))]);
      };
      typedef f32x16_t Scores[2][2];  // [key half m][query half u]
      f32x16_t zero;
#pragma unroll
      for (int i = 0; i < 16; ++i) zero[i] = 0.f;
      // One 16-key step's probabilities of query half u: keys 16 (2m + hf) .., as the value wave's operand, in bf16 as
      // prefill_attn_ws_kernel's.
      auto put_p = [&](const Scores& sc, int t, int m, int hf, int u, float mu) {
        u32x4_t pop;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[m][u][8 * hf + 2 * e], a.scale_log2, -mu));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[m][u][8 * hf + 2 * e + 1], a.scale_log2, -mu));
          l_run[u] += p0 + p1;
          pop[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{p0, p1}), bf16x2_t));
        }
        ps[pr][t & 1][u][2 * m + hf][lane] = pop;
      };
      // The reference of tile t's scores (masked on the pair's last tile).
      auto refer = [&](Scores& sc, int t) {
        // max3's operands come from the matrix unit: every product has written its result after 24 wait states.
        asm volatile("s_nop 15\n\ts_nop 7" : "+v"(sc[0][0]), "+v"(sc[0][1]), "+v"(sc[1][0]), "+v"(sc[1][1]));
        if (kPacked ? t * kPairK + kPairK - 1 > whole : t == dq) {
          const int off = kPacked ? whole - t * kPairK : 0;
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const int rel = off + 32 * u + x - (32 * m + 4 * g);  // keys 8 (i / 4) + i % 4 <= rel are seen
#pragma unroll
              for (int i = 0; i < 16; ++i) sc[m][u][i] = 8 * (i >> 2) + (i & 3) <= rel ? sc[m][u][i] : -INFINITY;
            }
        }
        float mx[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          mx[u] = max3(sc[0][u][0], sc[1][u][0], sc[0][u][1]);
          mx[u] = max3(mx[u], sc[1][u][1], sc[1][u][1]);
#pragma unroll
          for (int i = 2; i < 16; ++i) mx[u] = max3(mx[u], sc[0][u][i], sc[1][u][i]);
        }
        const bool move = __any(mx[0] > thr[0] || mx[1] > thr[1]);
        if (lane == 0) moved[pr][t & 3] = move ? 1 : 0;
        if (move) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float top = fmaxf(mx[u], __shfl_xor(mx[u], 32, kWave));
            const float m_new = fmaxf(m_ref[u], top * a.scale_log2);
            const float alpha = __builtin_amdgcn_exp2f(m_ref[u] - (m_new == -INFINITY ? 0.f : m_new));  // m_ref = -inf: 0
            if (g == 0) als[pr][t & 3][32 * u + x] = alpha;
            l_run[u] *= alpha;
            m_ref[u] = m_new;
            thr[u] = m_new == -INFINITY ? -INFINITY : (m_new + kWsGuard) / a.scale_log2;
          }
        }
      };
      // Step t: tile t's products into ``to``, the softmax of tile t - 1's scores ``from`` beside them.
      auto step = [&](const Scores& from, Scores& to, int t, bool soft) {
        u32x4_t kf[2] = {k_at(t, 0, 0), k_at(t, 1, 0)};
        const float m0 = m_ref[0] == -INFINITY ? 0.f : m_ref[0], m1 = m_ref[1] == -INFINITY ? 0.f : m_ref[1];
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int u = 0; u < 2; ++u) to[m][u] = mfma32(kf[m], q[u][s], s == 0 ? zero : to[m][u]);
          if (s + 1 < D / 16) {
#pragma unroll
            for (int m = 0; m < 2; ++m) kf[m] = k_at(t, m, s + 1);
          }
          if (soft) put_p(from, t - 1, s >> 2, (s >> 1) & 1, s & 1, s & 1 ? m1 : m0);
        }
        refer(to, t);
      };
      auto finish = [&](const Scores& from, int t) {  // the pair's last tile
        const float m0 = m_ref[0] == -INFINITY ? 0.f : m_ref[0], m1 = m_ref[1] == -INFINITY ? 0.f : m_ref[1];
#pragma unroll
        for (int s = 0; s < 8; ++s) put_p(from, t, s >> 2, (s >> 1) & 1, s & 1, s & 1 ? m1 : m0);
#pragma unroll
        for (int u = 0; u < 2; ++u) lsum[pr][g][32 * u + x] = l_run[u];
      };
      Scores sa, sb;
      lds_barrier();  // the first K tile (these waves have brought nothing yet)
      if (dq >= 0) step(sb, sa, 0, false);
      lds_barrier();
      int t = 1;
      for (; t + 1 <= dq; t += 2) {
        bring_v(t - 1);
        step(sa, sb, t, true);
        landed_barrier();
        bring_v(t);
        step(sb, sa, t + 1, true);
        landed_barrier();
      }
      if (t <= dq) {  // one more, then its scores are in sb
        bring_v(t - 1);
        step(sa, sb, t, true);
        landed_barrier();
        bring_v(t);
        finish(sb, t);
        landed_barrier();
        t += 2;
      } else if (dq >= 0) {
        bring_v(t - 1);
        finish(sa, t - 1);
        landed_barrier();
        t += 1;
      }
      for (; t <= nt + 1; ++t) {
        if (t <= nt) bring_v(t - 1);
        landed_barrier();
      }
      if (kPacked && pf_in_parts(one)) {
#pragma unroll
        for (int u = 0; u < 2; ++u) pf_leave_ml(a, one, pr, g, 32 * u + x, m_ref[u], l_run[u]);
      }
      if (!kChain || !enter(round + 1)) return;
      derive();
    }
  }

  // ---------------------------------------------------------------------------------------------- values
  auto bring_k = [&](int t) { bring(kbase, sp.k_bytes, kls[t & 1], t, [](int r) { return r; }); };
  f32x16_t o[2][4];  // [query half][e]: row 16k + 4q + i is dimension 32e + 8q + 4k + i, column x query x of the half
  auto clear = [&]() {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[u][e][i] = 0.f;
  };
  clear();
  // V operands by transpose reads: within 16 lanes (k = lane / 16 % 2), lane 4r + q points at key 4g + r, dimensions
  // 32e + 8q + 4k .., and lane 4q + i receives dimension 32e + 8q + 4k + i of the four keys.
  const int r = (lane & 15) >> 2, q4 = lane & 3, k2 = (lane >> 4) & 1;
  int vlane[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) vlane[e] = (4 * g + r) * (D * 2) + (e ^ r) * 64 + q4 * 16 + k2 * 8;
  auto attend_v = [&](int t) {
    u32x4_t p[2][4];
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int u = 0; u < 2; ++u) p[u][s] = ps[pr][t & 1][u][s][lane];
    if (moved[pr][t & 3]) {  // wave-uniform
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float al = als[pr][t & 3][32 * u + x];
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[u][e][i] *= al;
      }
    }
    const lds_char* vt = (const lds_char*)vls[t & 1];
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const v4i16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vt + vlane[e] + s * 16 * D * 2));
        const v4i16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vt + vlane[e] + (s * 16 + 8) * D * 2));
        const u32x2_t l2 = __builtin_bit_cast(u32x2_t, lo), h2 = __builtin_bit_cast(u32x2_t, hi);
        const u32x4_t vop = {l2[0], l2[1], h2[0], h2[1]};
#pragma unroll
        for (int u = 0; u < 2; ++u) o[u][e] = mfma32(vop, p[u][s], o[u][e]);
      }
  };
  // O of a block's queries from ``first``; whether some is not finite.
  auto output = [&](const PfSpan& s, int head, int first, int d) {
    bool again = false;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int query = first + 32 * u + x;
      if (query >= s.nq) continue;
      const float l = kPacked && d < 0 ? 0.f : lsum[pr][0][32 * u + x] + lsum[pr][1][32 * u + x];
      const float inv = l > 0.f ? 1.f / l : 1.f;
      uint16_t* orow = a.out + ((s.q0 + query) * a.H + head) * D + 8 * g;
      auto pair = [&](float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{lo * inv, hi * inv}), bf16x2_t));
      };
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {  // dimensions 32e + 16 rb + 8g .. + 7
          u32x4_t out;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int at = 4 * (rb + 2 * k);
            out[2 * k] = pair(o[u][e][at], o[u][e][at + 1]);
            out[2 * k + 1] = pair(o[u][e][at + 2], o[u][e][at + 3]);
          }
          *reinterpret_cast<u32x4_t*>(orow + 32 * e + 16 * rb) = out;
          if constexpr (kPacked) {
#pragma unroll
            for (int i = 0; i < 4; ++i) again |= pf_nonfinite(out[i]);
          }
        }
    }
    return again;
  };
  bring_k(0);
  landed_barrier();
  for (int round = 0;; ++round) {
    for (int t = 0; t <= nt + 1; ++t) {
      if (t + 1 < nt) bring_k(t + 1);
      if (t >= 2 && t - 2 <= dq) attend_v(t - 2);
      landed_barrier();
    }
    if constexpr (kChain) {
      // The next block's first K tile on its way (the score waves are past their last one) beside this block's output.
      const PfSpan was = sp;
      const int head = h, first = qp, d = dq;
      const bool more = enter(round + 1);
      if (more) {
        derive();
        bring_k(0);
      }
      if (__any(output(was, head, first, d))) chain.redo[pr][round >> 5] |= 1u << (round & 31);
      if (!more) break;
      clear();
      landed_barrier();
    } else {
      if (kPacked && pf_in_parts(one)) return pf_leave_o(a, one, pr, lane, sp.nq - qp, o);
      if (__any(output(sp, h, qp, dq)) && kPacked) pf_again<D>(a, sp, h, qp, 4, 0);
      return;
    }
  }
  for (int round = 0; enter(round); ++round) {
    derive();
    if (chain.redo[pr][round >> 5] >> (round & 31) & 1) pf_again<D>(a, sp, h, qp, 4, 0);
  }
}

// Packed prompts at head dim 256: 128 queries and 64-key tiles per workgroup of 8 waves, in two groups of 64 queries, of one
// head or (grouped heads) of two that read the same keys.  Score wave w (0..3) has 32 queries, all 256 dimensions in
// registers, and as in prefill_attn_pairs_kernel multiplies tile t beside the softmax of tile t - 1 with a reference of its
// own; value wave w has 128 dimensions of a group's O and as in prefill_attn_ws_kernel takes V straight from memory a tile
// ahead, two tiles behind the scores.  K goes to LDS by direct loads, two rows each, 16-byte chunk c of row r at position
// c ^ (r % 16).  One barrier per tile.
// What bounds a tile is what bounds prefill_attn_ws_kernel's: as many products for 3/4 of its bytes.  Measured, 16 heads
// over 2: 8 prompts of 750-2400 178 us (772 TFLOP/s; block by block 184), 16 of up to 500 behind up to 900 keys 79 us; the form of
// prefill_attn_wide_kernel (192 queries, partial scores added through LDS) 346 and 135 us.
constexpr int kPmQ = 128, kPmK = 64, kPmD = 256;

template <bool kChain>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void packed_attn_mid_kernel(PrefillArgs a) {
  constexpr int D = kPmD;
  __shared__ __attribute__((aligned(16))) char kls[2][kPmK * D * 2];
  __shared__ u32x4_t ps[2][4][4][64];  // [tile parity][score wave][16-key step][lane]
  __shared__ float als[4][4][32];      // [score wave][tile % 4]: O's factors, when the reference moved
  __shared__ int moved[4][4];
  __shared__ float lsum[4][2][32];     // [score wave][lane half]
  static_assert(kPfListBytes <= sizeof(kls), "");
  __shared__ char chain_at[kChain ? sizeof(PfChain) : 1] __attribute__((aligned(16)));
  PfChain& chain = *reinterpret_cast<PfChain*>(chain_at);
  const int together = a.together, queries = a.block;
  const int tid = threadIdx.x, lane = tid & 63, x = lane & 31, g = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), group = (w & 3) >> 1;
  PfPacked blk = {};
  PfSpan sp;
  int qb, h, keys;  // the block's first query, the group's head, what the block's last query sees of the part's keys
  // The chain's block of ``round``; false past its end.
  auto enter = [&](int round) {
    PfListed at;
    if (!pf_listed(chain, round, a.H / together, at)) return false;
    qb = at.j * queries;
    h = at.h * together + group % together;
    sp = pf_packed_span(a, h, pf_of(chain, at.s));
    keys = min(qb + queries, sp.nq) + sp.before;
    return true;
  };
  if constexpr (kChain) {
    pf_chain<D>(a, queries, a.H / together, chain, &kls[0][0]);
    if (!enter(0)) return;
  } else {
    const int nqb = (a.width + queries - 1) / queries;
    blk = pf_packed_block(a, nqb, queries, a.H / together, (int)gridDim.z / a.parts);
    qb = (nqb - 1 - blk.j) * queries;  // the longest blocks first
    h = blk.h * together + group % together;
    sp = pf_packed_span(a, h, blk.s);
    keys = min(qb + queries, sp.nq) + sp.before;
    if (qb >= sp.nq) return;
    if (!pf_part(a, blk, sp, keys)) return;
    if (keys <= 0) {
      for (int i = 0; i < together; ++i)
        pf_zeros<D>(a, sp.q0 + qb, sp.q0 + min(qb + queries, sp.nq), blk.h * together + i);
      return;
    }
  }
  int nt, qp, dq;  // tiles; the group's first query and its last tile (-1: no queries, or they see no key)
  const char *kbase, *vbase;
  auto derive = [&]() {
    kbase = scalar_pointer(sp.k);
    vbase = scalar_pointer(sp.v);
    nt = (keys + kPmK - 1) / kPmK;
    qp = qb + 64 * (group / together);
    if (qp >= qb + queries) qp = sp.nq;  // a block of one group
    const int lastk = min(min(qp + 64, sp.nq) + sp.before, keys) - 1;
    dq = qp < sp.nq && lastk >= 0 ? lastk / kPmK : -1;
  };
  derive();

  if (w < 4) {  // ------------------------------------------------------------------------------ scores
    for (int round = 0;; ++round) {
      const int query = qp + 32 * (w & 1) + x, whole = qp + 32 * (w & 1) + sp.before;  // all 32 see keys [0, whole]
      u32x4_t q[D / 16];  // q[query][16s + 8g .. + 7]
      {
        const uint16_t* qrow = a.q + ((sp.q0 + min(query, sp.nq - 1)) * a.H + h) * D + g * 8;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) q[s] = *reinterpret_cast<const u32x4_t*>(qrow + s * 16);
      }
      float m_ref = -INFINITY, thr = -INFINITY, l_run = 0.f;
      const int klane = x * (D * 2) + ((g ^ (x & 15)) * 16);
      auto k_at = [&](int t, int m, int s) {
        return *reinterpret_cast<const u32x4_t*>(&kls[t & 1][32 * m * (D * 2) + (klane ^ (32 * s))]);
      };
      typedef f32x16_t Scores[2];  // [key half m]
      f32x16_t zero;
#pragma unroll
      for (int i = 0; i < 16; ++i) zero[i] = 0.f;
      // One 16-key step's probabilities: keys 16 (2m + hf) .., as the value wave's operand, in bf16 as
      // prefill_attn_ws_kernel's.
      auto put_p = [&](const Scores& sc, int t, int m, int hf, float mu) {
        u32x4_t pop;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[m][8 * hf + 2 * e], a.scale_log2, -mu));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[m][8 * hf + 2 * e + 1], a.scale_log2, -mu));
          l_run += p0 + p1;
          pop[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{p0, p1}), bf16x2_t));
        }
        ps[t & 1][w][2 * m + hf][lane] = pop;
      };
      // The reference of tile t's scores (masked where not every query sees every key).
      auto refer = [&](Scores& sc, int t) {
        // max3's operands come from the matrix unit: every product has written its result after 24 wait states.
        asm volatile("s_nop 15\n\ts_nop 7" : "+v"(sc[0]), "+v"(sc[1]));
        if (t * kPmK + kPmK - 1 > whole) {
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const int rel = whole - t * kPmK + x - (32 * m + 4 * g);  // keys 8 (i / 4) + i % 4 <= rel are seen
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[m][i] = 8 * (i >> 2) + (i & 3) <= rel ? sc[m][i] : -INFINITY;
          }
        }
        float mx = max3(sc[0][0], sc[1][0], sc[0][1]);
        mx = max3(mx, sc[1][1], sc[1][1]);
#pragma unroll
        for (int i = 2; i < 16; ++i) mx = max3(mx, sc[0][i], sc[1][i]);
        const bool move = __any(mx > thr);
        if (lane == 0) moved[w][t & 3] = move ? 1 : 0;
        if (move) {
          const float top = fmaxf(mx, __shfl_xor(mx, 32, kWave));
          const float m_new = fmaxf(m_ref, top * a.scale_log2);
          const float alpha = __builtin_amdgcn_exp2f(m_ref - (m_new == -INFINITY ? 0.f : m_new));  // m_ref = -inf: 0
          if (g == 0) als[w][t & 3][x] = alpha;
          l_run *= alpha;
          m_ref = m_new;
          thr = m_new == -INFINITY ? -INFINITY : (m_new + kWsGuard) / a.scale_log2;
        }
      };
      // Step t: tile t's products into ``to``, the softmax of tile t - 1's scores ``from`` beside them.
      auto step = [&](const Scores& from, Scores& to, int t, bool soft) {
        u32x4_t kf[2] = {k_at(t, 0, 0), k_at(t, 1, 0)};
        const float mu = m_ref == -INFINITY ? 0.f : m_ref;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
#pragma unroll
          for (int m = 0; m < 2; ++m) to[m] = mfma32(kf[m], q[s], s == 0 ? zero : to[m]);
          if (s + 1 < D / 16) {
#pragma unroll
            for (int m = 0; m < 2; ++m) kf[m] = k_at(t, m, s + 1);
          }
          if (soft && (s & 3) == 3) put_p(from, t - 1, s >> 3, (s >> 2) & 1, mu);
        }
        refer(to, t);
      };
      auto finish = [&](const Scores& from, int t) {  // the group's last tile
        const float mu = m_ref == -INFINITY ? 0.f : m_ref;
#pragma unroll
        for (int s = 0; s < 4; ++s) put_p(from, t, s >> 1, s & 1, mu);
        lsum[w][g][x] = l_run;
      };
      Scores sa, sb;
      lds_barrier();  // the first K tile
      if (dq >= 0) step(sb, sa, 0, false);
      lds_barrier();
      int t = 1;
      for (; t + 1 <= dq; t += 2) {
        step(sa, sb, t, true);
        lds_barrier();
        step(sb, sa, t + 1, true);
        lds_barrier();
      }
      if (t <= dq) {  // one more, then its scores are in sb
        step(sa, sb, t, true);
        lds_barrier();
        finish(sb, t);
        lds_barrier();
        t += 2;
      } else if (dq >= 0) {
        finish(sa, t - 1);
        lds_barrier();
        t += 1;
      }
      for (; t <= nt + 1; ++t) lds_barrier();
      if (!kChain && pf_in_parts(blk)) pf_leave_ml(a, blk, w, g, x, m_ref, l_run);
      if (!kChain || !enter(round + 1)) return;
      derive();
    }
  }

  // ---------------------------------------------------------------------------------------------- values
  const int vw = w - 4, slice = 128 * (vw & 1);
  f32x16_t o[2][4];  // as prefill_attn_ws_kernel's, of queries qp + 32u + x and dimensions slice ..
  auto clear = [&]() {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[u][e][i] = 0.f;
  };
  clear();
  // K rows 16 vw .. + 15 of tile t to LDS (past the last tile: that tile again, not used); rows past the sequence read its
  // last key (finite or masked).
  auto bring_k = [&](int t) {
    const int at = min(t, nt - 1), t0 = at * kPmK;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(kbase + (int64_t)t0 * sp.k_bytes), 0, -1, 0x00020000);
#pragma unroll
    for (int r2 = 0; r2 < 8; ++r2) {
      const int r = 16 * vw + 2 * r2 + g;
      const int key = min(t0 + r, sp.nk - 1) - t0;
      const uint32_t from = (uint32_t)key * sp.k_bytes + (uint32_t)(x ^ (r & 15)) * 16;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          kr, (__attribute__((address_space(3))) void*)&kls[t & 1][(16 * vw + 2 * r2) * (D * 2)], 16, from, 0, 0, 0);
    }
  };
  const uint32_t v_bytes = (uint32_t)a.v_pos * 2;
  const uint32_t vlane = (uint32_t)(8 * (x >> 4) + 4 * g) * v_bytes + (uint32_t)(slice + 8 * (x & 15)) * 2;
  u32x4_t v[4][4];
  auto load_v = [&](int t, int s) {  // 16-key step s of tile t; rows past the sequence read 0
    const int at = t * kPmK + 16 * s, rows = min(sp.nk - at, 16);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(vbase + (int64_t)at * sp.v_bytes), 0, rows > 0 ? (uint32_t)(rows - 1) * sp.v_bytes + D * 2 : 0,
        0x00020000);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[s][j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(vr, vlane + j * v_bytes, 0, 0));
  };
  // O^T += V^T P^T for tile t, and the loads of tile ``ahead`` as its registers fall free.
  auto attend_v = [&](int t, int ahead) {
    u32x4_t p[2][2], vop[2][4];
    auto read_p = [&](int s) {
#pragma unroll
      for (int u = 0; u < 2; ++u) p[u][s & 1] = ps[t & 1][2 * group + u][s][lane];
    };
    read_p(0);
    read_p(1);
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (moved[2 * group + u][t & 3]) {  // wave-uniform
        const float al = als[2 * group + u][t & 3][x];
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[u][e][i] *= al;
      }
    auto operands = [&](int s) {  // as prefill_attn_ws_kernel's
      u32x2_t lo[4], hi[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          const auto r = __builtin_amdgcn_permlane16_swap(v[s][j][d], v[s][j][2 + d], false, false);
          lo[j][d] = r[0];
          hi[j][d] = r[1];
        }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t sel = (e & 1) ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int q2 = 0; q2 < 2; ++q2) {
          vop[s & 1][e][q2] = __builtin_amdgcn_perm(lo[2 * q2 + 1][e >> 1], lo[2 * q2][e >> 1], sel);
          vop[s & 1][e][2 + q2] = __builtin_amdgcn_perm(hi[2 * q2 + 1][e >> 1], hi[2 * q2][e >> 1], sel);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(vop[s & 1][e]));  // built here, not where first used
    };
    operands(0);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      __builtin_amdgcn_sched_barrier(0);
      load_v(ahead, s);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int u = 0; u < 2; ++u) o[u][e] = mfma32(vop[s & 1][e], p[u][s & 1], o[u][e]);
      if (s < 2) read_p(s + 2);
      if (s < 3) operands(s + 1);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // A step's end: its K tile is in LDS, the 16 V loads issued after it may be on their way.
  auto k_landed = [&]() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x4f70);  // vmcnt(16)
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  };
  // O of a block's queries from ``first``; whether some is not finite.
  auto output = [&](const PfSpan& s, int head, int first, int d) {
    bool again = false;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int query = first + 32 * u + x;
      if (query >= s.nq) continue;
      const float l = d < 0 ? 0.f : lsum[2 * group + u][0][x] + lsum[2 * group + u][1][x];
      const float inv = l > 0.f ? 1.f / l : 1.f;
      uint16_t* orow = a.out + ((s.q0 + query) * a.H + head) * D + slice + 32 * g;
      auto pair = [&](float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{lo * inv, hi * inv}), bf16x2_t));
      };
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // dimensions 64r + 32g + 8i + 4k + e, k = 0, 1
          u32x4_t out;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int at = 4 * (r + 2 * k) + i;
            out[2 * k] = pair(o[u][0][at], o[u][1][at]);
            out[2 * k + 1] = pair(o[u][2][at], o[u][3][at]);
          }
          *reinterpret_cast<u32x4_t*>(orow + 64 * r + 8 * i) = out;
#pragma unroll
          for (int k = 0; k < 4; ++k) again |= pf_nonfinite(out[k]);
        }
    }
    return again;
  };
  bring_k(0);
  landed_barrier();
  for (int round = 0;; ++round) {
    bring_k(1);
    landed_barrier();  // step 0
    int t = 1;
    if (dq >= 0) {
      bring_k(2);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < 4; ++s) load_v(0, s);
      k_landed();  // step 1
      for (t = 2; t <= dq + 2; ++t) {
        bring_k(t + 1);
        __builtin_amdgcn_sched_barrier(0);
        attend_v(t - 2, min(t - 1, dq));
        k_landed();
      }
    }
    for (; t <= nt + 1; ++t) {
      bring_k(t + 1);
      landed_barrier();
    }
    if constexpr (kChain) {
      // As prefill_attn_pairs_kernel's.
      const PfSpan was = sp;
      const int head = h, first = qp, d = dq;
      const bool more = enter(round + 1);
      if (more) {
        derive();
        bring_k(0);
      }
      if (__any(output(was, head, first, d))) chain.redo[vw][round >> 5] |= 1u << (round & 31);
      if (!more) break;
      clear();
      landed_barrier();
    } else {
      if (pf_in_parts(blk)) return pf_leave_o(a, blk, vw, lane, sp.nq - qp, o);
      if (__any(output(sp, h, qp, dq))) pf_again<D>(a, sp, h, qp, 4, slice);
      return;
    }
  }
  for (int round = 0; enter(round); ++round) {
    derive();
    if (chain.redo[vw][round >> 5] >> (round & 31) & 1) pf_again<D>(a, sp, h, qp, 4, slice);
  }
}

// The parts of blocks joined: out = sum_p w_p O_p / sum_p w_p l_p, w_p = exp(m_p - max m).  One workgroup for a quarter
// (query half u, rows r of O) of a block's four value waves, each lane what it held of O there.
template <int D>
__global__ __launch_bounds__(256) void packed_attn_join_kernel(PrefillArgs a) {
  const int together = a.together, queries = D == 512 ? kWsQ : a.block;
  const int nqb = (a.width + queries - 1) / queries, j = (int)blockIdx.x >> 2, u = blockIdx.x >> 1 & 1, r = blockIdx.x & 1;
  const int hb = blockIdx.y, lane = threadIdx.x & 63, x = lane & 31, g = lane >> 5;
  const int vw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int share = 1;
  const PfSequence seq = pf_ranked(a, (int)gridDim.z, blockIdx.z, queries, gridDim.y, share);
  const int qb = (nqb - 1 - j) * queries;
  const int group = D == 128 ? vw : D == 256 ? vw >> 1 : 0, h = hb * together + group % together;
  if (64 * (group / together) >= queries) return;  // no queries
  const PfSpan sp = pf_packed_span(a, h, seq);
  const int keys = min(qb + queries, sp.nq) + sp.before;
  if (qb >= sp.nq || keys <= 0) return;
  const int parts = pf_parts(a, keys, share);
  if (parts == 1) return;
  const int64_t slot = ((int64_t)((int)blockIdx.z * (int)gridDim.y + hb) * nqb + j) * a.parts;
  const int slice = D == 128 ? 0 : D == 256 ? 128 * (vw & 1) : 128 * vw;
  const int first = qb + 64 * (group / together) + 32 * u, query = first + x;
  // The score waves of the queries, two (by key half) at head dim 512, and the queries' place there.
  const int sw = D == 128 ? vw : D == 256 ? 2 * group + u : u, at = D == 128 ? 32 * u + x : x;
  auto ml = [&](int p, int w, int half) {
    return *reinterpret_cast<const f32x2_t*>(a.part_ml + (slot + p) * kPartMl + ((w * 2 + half) * 64 + at) * 2);
  };
  float m = -INFINITY;
#pragma unroll 4
  for (int p = 0; p < parts; ++p) m = fmaxf(m, ml(p, sw, 0)[0]);
  f32x4_t o[4][2];
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e][0] = o[e][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  if (first >= sp.nq) return;
#pragma unroll 1  // (by 4 the launch of 16 parts takes 84 us in place of 57)
  for (int p = 0; p < parts && query < sp.nq; ++p) {
    const float* from = a.part_o + (slot + p) * kPartO + (vw * 4 + u * 2 + r) * (8 * 256) + lane * 4;
    const f32x2_t one = ml(p, sw, 0);
    float lp = one[1] + ml(p, sw, 1)[1];
    if constexpr (D == 512) lp += ml(p, sw + 2, 0)[1] + ml(p, sw + 2, 1)[1];
    const float f = one[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(one[0] - m);
    l += f * lp;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int k = 0; k < 2; ++k) o[e][k] += f * *reinterpret_cast<const f32x4_t*>(from + (e * 2 + k) * 256);
  }
  const float inv = l > 0.f ? 1.f / l : 1.f;
  auto pair = [&](float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{lo * inv, hi * inv}), bf16x2_t));
  };
  bool again = false;
  if (query < sp.nq) {
    uint16_t* orow = a.out + ((sp.q0 + query) * a.H + h) * D + slice + (D == 128 ? 16 * r + 8 * g : 64 * r + 32 * g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4_t out;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        out[2 * k] = D == 128 ? pair(o[i][k][0], o[i][k][1]) : pair(o[0][k][i], o[1][k][i]);
        out[2 * k + 1] = D == 128 ? pair(o[i][k][2], o[i][k][3]) : pair(o[2][k][i], o[3][k][i]);
      }
      *reinterpret_cast<u32x4_t*>(orow + (D == 128 ? 32 : 8) * i) = out;
#pragma unroll
      for (int k = 0; k < 4; ++k) again |= pf_nonfinite(out[k]);
    }
  }
  if (__any(again)) pf_again<D>(a, sp, h, first, 2, slice, D == 128 ? 0x3333u << (2 * r) : 0xffu << (8 * r));
}

// Parts of a block at most, for a launch of ``blocks`` that see up to ``keys`` keys: 1 where every CU has a block.  (Their
// workgroups are launched before it is known how many there are.  Up to 4 x 256 of them cost 2 x 600 behind 3000 10 us where
// there were none, 2 x 256 4 us; three prompts of 60-200 behind 1000, with none, take 37 us in place of 34.)
inline int packed_parts(int64_t blocks, int sequences, int64_t keys, int64_t longest) {
  const int64_t tiles = (keys + 63) / 64;
  if (blocks >= kPartCus || sequences > kWave || tiles < kPartBlock) return 1;
  if (tiles < kPartLong && 3 * blocks > kPartCus) return 1;  // not four times an even part
  // No earlier keys: a block's mean is half the longest.
  if (keys <= longest && (tiles < kPartLong || 3 * blocks >= 2 * kPartCus)) return 1;
  return (int)std::min({kPartCus / blocks + 1, tiles / kPartLeast, (int64_t)kPartMost});
}

// Queries of a head in a block, ``rows`` or fewer: fewer to a block take less time, if every CU still has one block at most.
// Measured at head dim 128, us, blocks of 256 and fewer, 32 heads: one prompt of 200 14.5 / 12.0, four of 60-200 15.9 / 14.2; 8
// heads, one of 1433 41.8 / 38.4; past one block for a CU, 32 heads, one of 1433 43 / 59.
inline int packed_block(int rows, int64_t longest, int64_t units) {
  while (rows > 64 && (longest + rows / 2 - 1) / (rows / 2) * units <= kPartCus) rows /= 2;
  return rows;
}

// Whether a launch runs its blocks in chains: where an XCD has two (head dims 128 and 256: three; 10 of 260-300, 32 heads,
// 2.5 for each, take 48 us in place of 45.5) or more for each of its workgroups (no more than their lists hold, and sequences
// that one wave's lanes hold), and the same ``heads`` blocks of heads for every sequence.  64 sequences of 20-600 and, block
// by block, 65, us: 8 heads x 512 200 / 239, 16 over 2 x 256 182 / 196, 32 over 8 x 128 181 / 188, 32 x 128 255 / 242.
inline bool packed_chains(int64_t nqb, int heads, int sequences, int head_dim) {
  const int64_t each = nqb * sequences * (heads / 8);  // blocks of an XCD, at most
  return heads % 8 == 0 && sequences <= kWave && each >= (head_dim == 512 ? 2 : 3) * kWsPerXcd &&
         each <= kPfRounds * kWsPerXcd;
}

// How a call is launched: heads of a kv head and queries of each in a block, blocks in all, in chains, in parts.
struct PackedPlan {
  int together, rows, parts;
  bool chains;
  int64_t units, blocks;  // units: blocks of heads x sequences
};
inline PackedPlan packed_plan(int head_dim, int heads, int kv_heads, int sequences, int64_t longest, int64_t keys) {
  const int group = heads / kv_heads;
  PackedPlan p;
  p.together = 1;
  if (head_dim == 128) p.together = group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
  if (head_dim == 256) p.together = group % 2 == 0 ? 2 : 1;
  p.rows = (head_dim == 128 ? kPairQ : head_dim == 256 ? kPmQ : kWsQ) / p.together;
  p.units = (int64_t)heads / p.together * sequences;
  auto count = [&] { return p.blocks = (longest + p.rows - 1) / p.rows * p.units; };
  p.chains = packed_chains(count() / p.units, heads / p.together, sequences, head_dim);
  p.parts = 1;
  if (p.chains) return p;
  if ((keys + 63) / 64 >= kPartLong) p.parts = packed_parts(p.blocks, sequences, keys, longest);
  if (p.parts > 1) return p;
  p.rows = packed_block(p.rows, longest, p.units);
  p.parts = packed_parts(count(), sequences, keys, longest);
  return p;
}

// Head dim 128 in blocks of 192 queries, for the launches of small_blocks: one workgroup of 4 waves, two workgroups per
// CU.  The block's 32-key tiles go through LDS once for all of its waves (double-buffered: tile t + 1's global loads are
// in flight during tile t's math).  Each wave holds kPfSub groups of 16 queries: per tile it reads the K fragments and,
// by LDS transpose reads, the V operands once, then runs S^T = K Q^T, the lazy softmax (causal limit as the key limit,
// skipped on tiles the whole group sees) and O += P V for every group that sees the tile.  What bounds it is that its
// products and its softmax share one wave: a tile takes ~1.7 times as long as in the pairs kernel, but a CU holds two.
constexpr int kPfWaves = 4;
constexpr int kPfSub = 3;  // 16-query groups per wave (3: 255 VGPRs, two waves per SIMD; measured fastest of 1-4)
constexpr int kPfQueries = 16 * kPfSub * kPfWaves;
constexpr int kPfRow = 128 * 2 + 16;  // LDS bytes per key row: 256 B of data, padded against bank conflicts
constexpr int kPfStage = 32;          // keys per LDS stage (one barrier each), a multiple of the 32-key MFMA tile
constexpr int kPfThreads = 64 * kPfWaves;
constexpr int kPfChunks = kPfStage * 16 / kPfThreads;  // 16-byte chunks of K (and of V) per thread per stage
static_assert(kPfChunks * kPfThreads == kPfStage * 16, "a stage is whole chunks per thread");

// Whether a launch at head dim 128 takes blocks of 192 queries, two per CU, rather than the pairs kernel's 256, one per
// CU: where the pairs kernel needs more than one round of its 256 workgroups and
//  * both sizes give the same number of blocks per unit, so that this one has half the rounds, and the 192 are at most 5/6
//    full on the mean (past that its time grows with the queries, the pairs kernel's does not);
//  * or, with one block more per unit at two or four blocks of 256, the pairs kernel's last round is nearly empty and this
//    kernel takes fewer rounds (with three, the blocks of that round are the short ones, and it costs little).
// Pairs kernel / this one, us: 160 units (5 contexts x 32 heads) x 257 27.3 / 22.7, x 300 27.4 / 24.8, x 385 33.5 / 30.6, x 384
// 30.0 / 32.2 (full: pairs); 256 x 257 29.0 / 24.2; 320 x 129 22.0 / 18.8; 130 x 512 40.7 / 32.9, 192 x 512 42.2 / 48.3
// (as many rounds: pairs); 96 x 800 50.8 / 47.0, 96 x 640 35.4 / 41.5 (three blocks: pairs).
inline bool small_blocks(int width, int64_t units) {
  constexpr int kCus = 256;
  const int n = (width + kPairQ - 1) / kPairQ, small = (width + kPfQueries - 1) / kPfQueries;
  const int64_t blocks = n * units, rounds = (blocks + kCus - 1) / kCus;
  if (rounds < 2) return false;
  if (n == small) return width <= kPfQueries * 5 / 6 * n;
  const int64_t small_rounds = (small * units + 2 * kCus - 1) / (2 * kCus), last = blocks % kCus;
  if (small != n + 1 || (n != 2 && n != 4) || last == 0 || small_rounds >= rounds) return false;
  return last <= 96 || (2 * small_rounds <= rounds && last <= 128);
}

// The softmax step of one 16-query group for one tile: mask (key0 + j >= lim), lazy reference max, this lane's
// 8 probabilities packed as the P operand.  (The same arithmetic as attend().)
template <int NB>
__device__ __forceinline__ u32x4_t softmax_tile(float (&sv)[8], float c_scale, SoftmaxState& st, f32x4_t (&o)[NB],
                                                int g, int key0, int lim, bool whole) {
  bool over = false;
  if (!whole) {  // whole (wave-uniform): every query of the group sees every key of the tile
#pragma unroll
    for (int j = 0; j < 8; ++j) sv[j] = key0 + j < lim ? sv[j] : -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) over |= sv[j] > st.thr;
  if (__any(over)) {
    float mx = sv[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) mx = fmaxf(mx, sv[j]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
    mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
    const float m_new = fmaxf(st.m_ref, mx * c_scale);
    rescale<NB>(st.m_ref, m_new == -INFINITY ? 0.f : m_new, st.l_run, o, g);
    st.m_ref = m_new;
    st.thr = m_new == -INFINITY ? -INFINITY : (m_new + kLazyLog2) / c_scale;
  }
  const float m_use = st.m_ref == -INFINITY ? 0.f : st.m_ref;
  float p[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[j], c_scale, -m_use));
    st.l_run += p[j];
  }
  u32x4_t pop;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    pop[w] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{p[2 * w], p[2 * w + 1]}), bf16x2_t));
  return pop;
}

__global__ __launch_bounds__(64 * kPfWaves) __attribute__((amdgpu_waves_per_eu(2, 2))) void prefill_attn_kernel(
    PrefillArgs a) {
  constexpr int D = 128, KS = D / 32;
  __shared__ __attribute__((aligned(16))) char lds[2][2][kPfStage * kPfRow];  // [buffer][K, V][key rows]
  const int nqb = (a.width + kPfQueries - 1) / kPfQueries;
  const PfBlock blk = pf_block(nqb, a.H, (int)gridDim.z);
  const int qb = (nqb - 1 - blk.j) * kPfQueries;  // the longest blocks first
  const int h = blk.h, b = blk.b;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t slot = clamp64(a.slots[b], 0, a.cache_rows - 1);
  const uint16_t* kbase = a.k + slot * a.s_row + h * a.s_head;
  const uint16_t* vbase = a.v + slot * a.s_row + h * a.s_head;
  const int kend = min(qb + kPfQueries, a.width);  // keys the block's last query sees
  const int nt = (kend + kPfStage - 1) / kPfStage;

  // Global -> LDS: thread tid moves 16-byte chunks tid, tid + kPfThreads, ... of the stage's K and of its V (kPfStage rows x
  // 256 B each).  Rows past the context read its last key (finite: masked by the causal limit, never NaN).
  u32x4_t stage[2 * kPfChunks];
  auto fetch = [&](int t) {
#pragma unroll
    for (int e = 0; e < kPfChunks; ++e) {
      const int ci = tid + e * kPfThreads, r = ci >> 4, col = ci & 15;
      const int key = min(t * kPfStage + r, a.width - 1);
      stage[e] = *reinterpret_cast<const u32x4_t*>(kbase + (int64_t)key * D + col * 8);
      stage[kPfChunks + e] = *reinterpret_cast<const u32x4_t*>(vbase + (int64_t)key * D + col * 8);
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int e = 0; e < kPfChunks; ++e) {
      const int ci = tid + e * kPfThreads, r = ci >> 4, col = ci & 15;
      *reinterpret_cast<u32x4_t*>(&lds[buf][0][r * kPfRow + col * 16]) = stage[e];
      *reinterpret_cast<u32x4_t*>(&lds[buf][1][r * kPfRow + col * 16]) = stage[kPfChunks + e];
    }
  };

  // The wave's groups: queries q0[u] + c, u < kPfSub (group u of wave w: block rows 16 (w + kPfWaves u)).
  int q0[kPfSub];
  u32x4_t qop[kPfSub][KS];  // B operand of S^T = K Q^T: lane (c, g) holds q[q0 + c][32s + 8g .. +7] (0 past the end)
  SoftmaxState st[kPfSub];
  f32x4_t o[kPfSub][D / 16];
#pragma unroll
  for (int u = 0; u < kPfSub; ++u) {
    q0[u] = qb + 16 * (w + kPfWaves * u);
    const bool live = q0[u] + c < a.width;
    const uint16_t* qrow = a.q + ((int64_t)(b * a.width + (live ? q0[u] + c : 0)) * a.H + h) * D + g * 8;
#pragma unroll
    for (int s2 = 0; s2 < KS; ++s2)
      qop[u][s2] = live ? *reinterpret_cast<const u32x4_t*>(qrow + s2 * 32) : u32x4_t{0u, 0u, 0u, 0u};
    st[u] = SoftmaxState{-INFINITY, -INFINITY, 0.f};
#pragma unroll
    for (int nb = 0; nb < D / 16; ++nb) o[u][nb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  fetch(0);
  put(0);
  __syncthreads();
  for (int t = 0; t < nt; ++t) {
    fetch(t + 1 < nt ? t + 1 : t);  // unconditional: the last iteration re-reads its own tile (cache hit)
    // The stage's 32-key MFMA tiles in turn.
#pragma unroll
    for (int sub = 0; sub < kPfStage / 32; ++sub) {
    const int key0 = t * kPfStage + sub * 32;
    // Groups that see the tile (wave-uniform): a live group whose last query reaches the tile's first key.
    bool act[kPfSub];
    bool any = false;
#pragma unroll
    for (int u = 0; u < kPfSub; ++u) {
      act[u] = q0[u] < a.width && key0 <= q0[u] + 15;
      any |= act[u];
    }
    if (any) {
      const char* kl = lds[t & 1][0] + sub * 32 * kPfRow;
      const char* vl = lds[t & 1][1] + sub * 32 * kPfRow;
      u32x4_t pop[kPfSub];
      {
        u32x4_t kf[2][KS];
#pragma unroll
        for (int mb = 0; mb < 2; ++mb) {
          const int rk = 8 * (c >> 2) + 4 * mb + (c & 3);
#pragma unroll
          for (int s2 = 0; s2 < KS; ++s2) kf[mb][s2] = *reinterpret_cast<const u32x4_t*>(kl + rk * kPfRow + g * 16 + s2 * 64);
        }
#pragma unroll
        for (int u = 0; u < kPfSub; ++u) {
          if (!act[u]) continue;
          f32x4_t sacc[2];
#pragma unroll
          for (int mb = 0; mb < 2; ++mb) {
            sacc[mb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s2 = 0; s2 < KS; ++s2)
              sacc[mb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kf[mb][s2]),
                                                                 __builtin_bit_cast(bf16x8_t, qop[u][s2]), sacc[mb],
                                                                 0, 0, 0);
          }
          float sv[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) sv[j] = sacc[j >> 2][j & 3];
          pop[u] = softmax_tile<D / 16>(sv, a.scale_log2, st[u], o[u], g, key0 + 8 * g, q0[u] + c + 1,
                                        key0 + 31 <= q0[u]);
        }
      }
      {
        // V operands by transpose reads: in lane group g (keys 8g .. 8g + 7) lane 4r + q points at key
        // 8g + 4h + r, dimensions 16e + 4q .. 16e + 4q + 3 (h = 0, 1), and ds_read_b64_tr_b16 hands lane c the
        // four keys' dimension 16e + c: block e's B operand, output column c = dimension 16e + c.
        const int rr = c >> 2, q4 = c & 3;
        const lds_char* vls = (const lds_char*)vl;  // vl points into LDS
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int off = (8 * g + rr) * kPfRow + (16 * e + 4 * q4) * 2;
          const v4i16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vls + off));
          const v4i16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vls + off + 4 * kPfRow));
          u32x4_t bop;
          bop[0] = (uint32_t)(uint16_t)lo[0] | ((uint32_t)(uint16_t)lo[1] << 16);
          bop[1] = (uint32_t)(uint16_t)lo[2] | ((uint32_t)(uint16_t)lo[3] << 16);
          bop[2] = (uint32_t)(uint16_t)hi[0] | ((uint32_t)(uint16_t)hi[1] << 16);
          bop[3] = (uint32_t)(uint16_t)hi[2] | ((uint32_t)(uint16_t)hi[3] << 16);
#pragma unroll
          for (int u = 0; u < kPfSub; ++u) {
            if (!act[u]) continue;
            o[u][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, pop[u]),
                                                              __builtin_bit_cast(bf16x8_t, bop), o[u][e], 0, 0, 0);
          }
        }
      }
    }
    }
    put((t + 1) & 1);
    __syncthreads();
  }

  // ---- each group's 16 output rows: O / l, rounded to bf16
#pragma unroll
  for (int u = 0; u < kPfSub; ++u) {
    float l_tot = st[u].l_run + __shfl_xor(st[u].l_run, 16, kWave);
    l_tot += __shfl_xor(l_tot, 32, kWave);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float li = __shfl(l_tot, 4 * g + i, kWave);
      const int qq = q0[u] + 4 * g + i;
      if (qq >= a.width) continue;
      const float div = li > 0.f ? li : 1.f;
      uint16_t* orow = a.out + ((int64_t)(b * a.width + qq) * a.H + h) * D;
#pragma unroll
      for (int e = 0; e < 8; ++e) orow[16 * e + c] = (uint16_t)pack_bf16x2(o[u][e][i] / div, 0.f);  // dim 16e + c
    }
  }
}

}  // namespace omni

extern "C" int omni_prefill_attention(const void* q, const void* k_cache, const void* v_cache, int64_t stride_row,
                                      int64_t stride_head, int64_t stride_pos, int64_t cache_len,
                                      int64_t cache_rows, const int64_t* slots, int32_t contexts, int32_t width,
                                      int32_t heads, int32_t head_dim, float scale, void* out, int32_t dtype,
                                      void* stream) {
  if (contexts < 0 || width < 0 || heads <= 0 || cache_rows <= 0) return OMNI_ERR_INVALID;
  if (dtype != OMNI_BF16) return OMNI_ERR_DTYPE;
  if ((head_dim != 128 && head_dim != 256 && head_dim != 512) || stride_pos != head_dim) return OMNI_ERR_SHAPE;
  if (!(scale > 0.f) || width > cache_len) return OMNI_ERR_INVALID;
  if (contexts == 0 || width == 0) return OMNI_OK;
  if (!q || !k_cache || !v_cache || !slots || !out) return OMNI_ERR_INVALID;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15u) return OMNI_ERR_INVALID;
  if ((stride_row | stride_head) % 8 != 0) return OMNI_ERR_INVALID;
  if ((int64_t)contexts * width * heads >= (int64_t{1} << 31) / head_dim) return OMNI_ERR_INVALID;
  omni::PrefillArgs a;
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k_cache;
  a.v = (const uint16_t*)v_cache;
  a.slots = slots;
  a.s_row = stride_row;
  a.s_head = stride_head;
  a.cache_rows = cache_rows;
  a.width = width;
  a.H = heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = (uint16_t*)out;
  hipStream_t s = (hipStream_t)stream;
  if (head_dim == 128) {
    if (omni::small_blocks(width, (int64_t)heads * contexts)) {
      dim3 grid((width + omni::kPfQueries - 1) / omni::kPfQueries, heads, contexts);
      omni::prefill_attn_kernel<<<grid, omni::kPfThreads, 0, s>>>(a);
    } else {
      dim3 grid((width + omni::kPairQ - 1) / omni::kPairQ, heads, contexts);
      omni::prefill_attn_pairs_kernel<false, false><<<grid, 512, 0, s>>>(a);
    }
  } else if (head_dim == 512) {
    const int nqb = (width + omni::kWsQ - 1) / omni::kWsQ, units = heads * contexts;
    dim3 grid(nqb, heads, contexts);
    a.units8 = units / 8;
    a.group = units % 8 == 0 ? omni::ws_group(nqb, a.units8) : 0;
    if (a.group) {
      omni::prefill_attn_ws_kernel<true, false><<<8 * omni::kWsPerXcd, 512, 0, s>>>(a);
    } else {
      omni::prefill_attn_ws_kernel<false, false><<<grid, 512, 0, s>>>(a);
    }
  } else {
    const int qw = 16 * omni::kPwSub * (omni::kPwWaves / 2);  // queries per workgroup
    dim3 grid((width + qw - 1) / qw, heads, contexts);
    omni::prefill_attn_wide_kernel<<<grid, 64 * omni::kPwWaves, 0, s>>>(a);
  }
  return omni_launch_status();
}

extern "C" size_t omni_packed_attention_workspace(int32_t sequences, int64_t keys, int32_t longest, int32_t heads,
                                                  int32_t kv_heads, int32_t head_dim) {
  if (sequences <= 0 || keys <= 0 || longest <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return 0;
  if (head_dim != 128 && head_dim != 256 && head_dim != 512) return 0;
  const omni::PackedPlan p = omni::packed_plan(head_dim, heads, kv_heads, sequences, longest, keys);
  return p.parts == 1 ? 0 : (size_t)(p.blocks * p.parts * (omni::kPartO + omni::kPartMl) * 4);
}

extern "C" int omni_packed_attention(const void* q, const void* k, const void* v, int64_t k_stride_pos,
                                     int64_t k_stride_head, int64_t v_stride_pos, int64_t v_stride_head,
                                     const int64_t* starts, const int64_t* k_starts, int32_t sequences,
                                     int64_t queries, int64_t keys, int32_t longest, int32_t heads, int32_t kv_heads,
                                     int32_t head_dim, float scale, void* out, void* workspace, size_t workspace_bytes,
                                     int32_t dtype, void* stream) {
  if (dtype != OMNI_BF16) return OMNI_ERR_DTYPE;
  if (sequences < 0 || queries < 0 || keys < 0 || longest < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads)
    return OMNI_ERR_INVALID;
  if (head_dim != 128 && head_dim != 256 && head_dim != 512) return OMNI_ERR_SHAPE;
  if (!(scale > 0.f) || scale == INFINITY) return OMNI_ERR_INVALID;
  if (sequences == 0 || queries == 0 || longest == 0) return OMNI_OK;
  if (!q || !starts || !k_starts || !out || (keys > 0 && (!k || !v))) return OMNI_ERR_INVALID;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k | (uintptr_t)v) & 15u) return OMNI_ERR_INVALID;
  if ((k_stride_pos | k_stride_head | v_stride_pos | v_stride_head) & 7) return OMNI_ERR_INVALID;
  if (k_stride_pos < 0 || k_stride_head < 0 || v_stride_pos < 0 || v_stride_head < 0) return OMNI_ERR_INVALID;
  if (sequences > 65535 || heads > 65535) return OMNI_ERR_SHAPE;
  // A tile's 64 rows are addressed by 32-bit byte offsets; a sequence's keys are counted in 31 bits.
  if (k_stride_pos >= (1 << 24) || v_stride_pos >= (1 << 24) || keys > 0x7fffff00LL || queries > 0x7fffff00LL)
    return OMNI_ERR_SHAPE;
  omni::PrefillArgs a;
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.slots = nullptr;
  a.s_row = a.s_head = a.cache_rows = 0;
  a.width = longest;
  a.H = heads;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = (uint16_t*)out;
  a.units8 = a.group = 0;
  a.starts = starts;
  a.k_starts = k_starts;
  a.queries = queries;
  a.keys = keys;
  a.k_pos = k_stride_pos;
  a.k_head = k_stride_head;
  a.v_pos = v_stride_pos;
  a.v_head = v_stride_head;
  a.heads_per_kv = heads / kv_heads;
  const int64_t seen = k_starts == starts ? std::min<int64_t>(keys, longest) : keys;  // by one sequence, at most
  const omni::PackedPlan p = omni::packed_plan(head_dim, heads, kv_heads, sequences, longest, seen);
  dim3 grid(p.blocks / p.units, heads / p.together, sequences);
  // The blocks are counted in 31 bits, a launch's threads along x, 512 to a block, in 32.
  if (grid.x >= (1u << 23) || p.blocks > 0x7fffffffLL) return OMNI_ERR_SHAPE;
  a.together = p.together;
  a.block = p.rows;
  a.parts = p.parts;
  a.sequences = sequences;
  const bool chains = p.chains;
  if (a.parts > 1) {
    if (!workspace || ((uintptr_t)workspace & 255u) ||
        workspace_bytes < omni_packed_attention_workspace(sequences, seen, longest, heads, kv_heads, head_dim))
      return OMNI_ERR_WORKSPACE;
    a.part_o = (float*)workspace;
    a.part_ml = a.part_o + p.blocks * a.parts * omni::kPartO;
  }
  const dim3 join(grid.x * 4, grid.y, grid.z);
  grid.z *= a.parts;
  const hipStream_t s = (hipStream_t)stream;
  if (head_dim == 128) {
    if (chains) omni::prefill_attn_pairs_kernel<true, true><<<8 * omni::kWsPerXcd, 512, 0, s>>>(a);
    else omni::prefill_attn_pairs_kernel<true, false><<<grid, 512, 0, s>>>(a);
    if (a.parts > 1) omni::packed_attn_join_kernel<128><<<join, 256, 0, s>>>(a);
  } else if (head_dim == 256) {
    if (chains) omni::packed_attn_mid_kernel<true><<<8 * omni::kWsPerXcd, 512, 0, s>>>(a);
    else omni::packed_attn_mid_kernel<false><<<grid, 512, 0, s>>>(a);
    if (a.parts > 1) omni::packed_attn_join_kernel<256><<<join, 256, 0, s>>>(a);
  } else {
    if (chains) omni::prefill_attn_ws_kernel<true, true><<<8 * omni::kWsPerXcd, 512, 0, s>>>(a);
    else omni::prefill_attn_ws_kernel<false, true><<<grid, 512, 0, s>>>(a);
    if (a.parts > 1) omni::packed_attn_join_kernel<512><<<join, 256, 0, s>>>(a);
  }
  return omni_launch_status();
}
