// Decode attention of rows that share the first pages of a paged cache: the keys
// that a group of rows shares are read, and multiplied, once for all of its rows.
//   out[n, h] = sum_j softmax_j(q[n, h] . K[n, j] * scale) V[n, j]
// splits at the prefix: with m the running maximum, l = sum_j 2^(s_j - m) and o =
// sum_j 2^(s_j - m) V_j over the prefix and over the row's own keys, in log2 units,
//   out = (o_p 2^(m_p - m) + o_r 2^(m_r - m)) / (l_p 2^(m_p - m) + l_r 2^(m_r - m)).
//
// Two launches: the rows' own keys (paged_tile.h, kState) and the prefixes beside each
// other, then the merge.  A prefix's rows are the query heads of a kv head of all its
// requests, 128 to a tile; a piece of work is a tile and a range of keys, dealt so that
// every work-group has one (the lengths are known to the GPU only: each work-group
// counts the pieces for itself).  A wave takes 32 rows and walks 64 keys a step as dense
// attention does (attn_dense.hip): K and V tiles go to a ring of three LDS slots, S^T =
// K Q^T and O^T += V^T P^T on 32x32x16 matrix instructions, weights from the scores'
// registers, rounded once to 16 bits (each weight by half a step at most, the same in the
// sum of the values and in the weights' own sum, which puts an output off by about as
// much as its own rounding: in bf16 2.3e-3 of the outputs' norm, against 1.7e-3 with two
// parts a weight as for the own keys, which take 198 us where one takes 156, 33 for 31 in
// the cases below).  fp16's small weights go in apart, by products of their own in the steps
// that have any (131072 keys behind a sink 20 nats above them: 250 us for 185).  Only whole
// 64-key tiles of a prefix are walked here, without masks; what is left of it comes with the
// row's own keys.
//
// us, bf16, D 128: 64 rows of 28 query and 4 kv heads that share 131072 keys: 156 for
// 120 GFLOP (770 TFLOP/s; the rows' tiles hold 8/7 of that): 30 at any length (launches,
// counting, 33 MB of states written and read again), then steps at 1000 TFLOP/s and more,
// where the matrix cores' power is the bound, as in dense attention.  Every row for
// itself: 2466.  40 rows of 32 query and 8 kv heads in six groups of 8192 keys: 31 for
// 96 MB (15 at a large read's 6.3 TB/s), where every row for itself takes 67: at 27 rows a kv
// head one wave of four computes.
// Tried, and no faster: rings of four and six slots; two to eight K and V fragments read
// ahead; three work-groups a CU; the keys of a step between two waves where a tile has 64
// rows at most (a half step takes 0.8 of a whole one: 162 -> 184 with twice the steps a
// piece); ranges that begin their walks at different steps.
#include "dense_tile.h"
#include "lanes.h"
#include "paged_ops.h"
#include "paged_tile.h"

namespace va {

namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr int kRows = 128;       // rows of a tile
constexpr int kMostGroups = 512;  // of the prefixes: two a CU
constexpr int kIdKeys = 1024;    // keys whose page ids lie in LDS, for pages of any size

// Where a state lies: that of the first piece with its row, (request, query head); those
// of the others in slots of `stride` rows.
struct SharedArgs {
  PagedArgs a;
  FastDiv by_g;
  float2* first_ml;   // (N * Hq)
  float* first;       // (N * Hq, D)
  float2* more_ml;    // (groups slots)
  float* more;
  int4* record;       // (N * Hq): pieces of the row behind its first, their slots' first, its row
  int32_t groups, stride;  // stride: rows of a tile that there can be
  uint32_t least;          // steps of a piece, at least
};

__device__ inline uint32_t plus(uint32_t a, uint32_t b) {
  const uint32_t s = a + b;
  return s < a ? 0xffffffffu : s;
}

// Rows and shared keys of the group that begins at row n: `tiles` tiles of rows for
// each kv head, `steps` steps of each.
struct Group {
  int32_t first, rows;
  uint32_t tiles, steps;
};
__device__ inline Group group_at(const PagedArgs& a, int64_t n) {
  Group g{int32_t(n), 0, 0, 0};
  if (n >= a.N) return g;
  const int64_t rows = a.group_rows[n] < a.N - n ? a.group_rows[n] : a.N - n;
  if (rows <= 0) return g;
  g.rows = int32_t(rows);
  g.steps = uint32_t(shared_keys(a.prefix_lens[n], a.M * a.page) / kPrefixTile);
  g.tiles = g.steps ? uint32_t((rows * a.G + kRows - 1) / kRows) : 0;
  return g;
}
__device__ inline uint32_t uniform(uint32_t x) {
  return uint32_t(__builtin_amdgcn_readfirstlane(int(x)));
}

// A piece: some steps of a tile of rows of a kv head.  Every work-group counts them
// for itself.  The pieces of a group are numbered by kv head, then range of keys, then
// tile, so that work-groups of neighbouring numbers, which run on one XCD at a time,
// read the same keys from its L2 (in the order of tiles, then ranges, 131072 keys of
// 448 rows of 4 kv heads came from the fabric four times, at the most that it gives).
struct Sum { uint32_t pieces, more; };  // `more`: those that are not the first of their rows
struct PiecesLds {
  uint2 sum[kWaves];
  Sum before[kThreads], mine[kThreads];
  Group found;
  Sum at;
};
struct Pieces {
  uint32_t length, count;  // steps of a piece, at most; all pieces
};
__device__ inline Sum pieces_of(const PagedArgs& a, const Group& g, uint32_t length) {
  const uint32_t segments = uint32_t(a.Hk) * g.tiles;
  if (!segments) return Sum{0, 0};
  const uint32_t ranges = (g.steps - 1) / length + 1;
  const uint64_t n = uint64_t(segments) * ranges;
  const uint32_t all = n < 0xffffffffu ? uint32_t(n) : 0xffffffffu;
  return Sum{all, all - segments};
}
// Sums over the work-group of two values, and over the threads before.
__device__ inline uint2 block_sum(uint2 x, uint2* part, uint2* before) {
  const int lane = threadIdx.x % 64, w = threadIdx.x / 64;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t u = __shfl_up(x.x, d), v = __shfl_up(x.y, d);
    if (lane >= d) x = make_uint2(plus(x.x, u), plus(x.y, v));
  }
  __syncthreads();  // the sums before have been read
  if (lane == 63) part[w] = x;
  const uint32_t u = __shfl_up(x.x, 1), v = __shfl_up(x.y, 1);
  __syncthreads();
  uint2 b = lane ? make_uint2(u, v) : make_uint2(0, 0), total = make_uint2(0, 0);
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) b = make_uint2(plus(b.x, part[i].x), plus(b.y, part[i].y));
    total = make_uint2(plus(total.x, part[i].x), plus(total.y, part[i].y));
  }
  *before = b;
  return make_uint2(uniform(total.x), uniform(total.y));
}
__device__ inline int32_t run_of(const PagedArgs& a) {
  return (int32_t(a.N) + kThreads - 1) / kThreads;
}
// Steps of a piece: a work-group one piece, where there are fewer segments than work-groups.
__device__ inline uint32_t piece_length(uint32_t steps, uint32_t segments, uint32_t groups,
                                        uint32_t least) {
  const uint32_t spare = segments < groups / 2 ? groups - segments : groups / 2;
  const uint32_t n = steps / (spare ? spare : 1) + 1;
  return n < least ? least : n;
}
__device__ inline uint2 steps_of(const PagedArgs& a, const Group& g) {  // and segments
  const uint64_t segments = uint64_t(a.Hk) * g.tiles, steps = segments * g.steps;
  return make_uint2(steps < 0xffffffffu ? uint32_t(steps) : 0xffffffffu, uint32_t(segments));
}
// Up to 64 rows are a lane each, in every wave by itself.
__device__ inline uint2 wave_sum(uint2 x) {
  const int lane = threadIdx.x % 64;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t u = __shfl_up(x.x, d), v = __shfl_up(x.y, d);
    if (lane >= d) x = make_uint2(plus(x.x, u), plus(x.y, v));
  }
  return x;
}
__device__ inline uint32_t lane_of(uint32_t x, int lane) {
  return uint32_t(__builtin_amdgcn_readlane(int(x), lane));
}
struct LanePieces {
  Group g;
  Sum before, mine;
};
__device__ inline Pieces count_in_lanes(const PagedArgs& a, uint32_t groups, uint32_t least,
                                        LanePieces* to) {
  to->g = group_at(a, threadIdx.x % 64);
  const uint2 all = wave_sum(steps_of(a, to->g));
  Pieces p;
  p.length = piece_length(lane_of(all.x, 63), lane_of(all.y, 63), groups, least);
  to->mine = pieces_of(a, to->g, p.length);
  const uint2 sum = wave_sum(make_uint2(to->mine.pieces, to->mine.more));
  p.count = lane_of(sum.x, 63);
  const uint32_t u = __shfl_up(sum.x, 1), v = __shfl_up(sum.y, 1);
  to->before = threadIdx.x % 64 ? Sum{u, v} : Sum{0, 0};
  return p;
}
__device__ inline Group find_in_lanes(const LanePieces& l, uint32_t piece, Sum* before) {
  const uint64_t here =
      __ballot(piece >= l.before.pieces && piece - l.before.pieces < l.mine.pieces);
  const int at = here ? __builtin_ctzll(here) : 0;  // (piece is below the sum)
  *before = Sum{lane_of(l.before.pieces, at), lane_of(l.before.more, at)};
  return Group{at, int32_t(lane_of(uint32_t(l.g.rows), at)), lane_of(l.g.tiles, at),
               lane_of(l.g.steps, at)};
}

__device__ inline Pieces count_pieces(const PagedArgs& a, uint32_t groups, uint32_t least,
                                      PiecesLds& lds) {
  const int32_t N = int32_t(a.N), per = run_of(a), lo = int32_t(threadIdx.x) * per;
  uint2 mine = make_uint2(0, 0), before;
  for (int32_t i = lo; i < lo + per && i < N; ++i) {
    const uint2 n = steps_of(a, group_at(a, i));
    mine = make_uint2(plus(mine.x, n.x), plus(mine.y, n.y));
  }
  const uint2 all = block_sum(mine, lds.sum, &before);
  Pieces p;
  p.length = piece_length(all.x, all.y, groups, least);
  mine = make_uint2(0, 0);
  for (int32_t i = lo; i < lo + per && i < N; ++i) {
    const Sum s = pieces_of(a, group_at(a, i), p.length);
    mine = make_uint2(plus(mine.x, s.pieces), plus(mine.y, s.more));
  }
  p.count = block_sum(mine, lds.sum, &before).x;
  lds.before[threadIdx.x] = Sum{before.x, before.y};
  lds.mine[threadIdx.x] = Sum{mine.x, mine.y};
  return p;
}
// The group of a piece, and the pieces before the group.
__device__ inline Group find_piece(const PagedArgs& a, uint32_t piece, uint32_t length,
                                   PiecesLds& lds, Sum* before) {
  __syncthreads();  // the one found before has been read
  const int32_t per = run_of(a), lo = int32_t(threadIdx.x) * per;
  Sum at = lds.before[threadIdx.x];
  if (piece >= at.pieces && piece - at.pieces < lds.mine[threadIdx.x].pieces) {
    for (int32_t i = lo; i < lo + per && i < a.N; ++i) {
      const Group g = group_at(a, i);
      const Sum n = pieces_of(a, g, length);
      if (piece - at.pieces < n.pieces) {
        lds.found = g;
        lds.at = at;
        break;
      }
      at = Sum{plus(at.pieces, n.pieces), plus(at.more, n.more)};
    }
  }
  __syncthreads();
  *before = Sum{uniform(lds.at.pieces), uniform(lds.at.more)};
  const Group g = lds.found;  // in scalar registers
  return Group{int32_t(uniform(uint32_t(g.first))), int32_t(uniform(uint32_t(g.rows))),
               uniform(g.tiles), uniform(g.steps)};
}

// The same by a wave alone.
__device__ inline Group find_in_wave(const PagedArgs& a, uint32_t piece, uint32_t length,
                                     const PiecesLds& lds, Sum* before) {
  int32_t at = 0;
  for (int32_t i = threadIdx.x % 64; i < kThreads; i += 64) {
    const Sum b = lds.before[i];
    const uint64_t here =
        __ballot(piece >= b.pieces && piece - b.pieces < lds.mine[i].pieces);
    if (here) at = i / 64 * 64 + __builtin_ctzll(here);
  }
  const int32_t lo = __builtin_amdgcn_readfirstlane(at) * run_of(a);
  Group g = group_at(a, lo);
  *before = lds.before[__builtin_amdgcn_readfirstlane(at)];
  for (int32_t i = lo;;) {
    const Sum n = pieces_of(a, g, length);
    if (piece - before->pieces < n.pieces || ++i >= lo + run_of(a)) return g;
    *before = Sum{plus(before->pieces, n.pieces), plus(before->more, n.more)};
    g = group_at(a, i);
  }
}

// One of them: a range of the 64-key tiles [t0, t0 + count) of a tile of rows.
struct Piece {
  uint32_t hk, tile, range, ranges, t0, count;
  uint32_t slots;  // the first of the segment's further pieces
  uint32_t rows;   // from this tile on
};
__device__ __forceinline__ Piece piece_at(const PagedArgs& a, const Group& grp, const Sum& before,
                                          uint32_t piece, uint32_t length) {
  Piece p;
  p.ranges = (grp.steps - 1) / length + 1;
  const uint32_t at = piece - before.pieces;
  p.hk = at / (p.ranges * grp.tiles);
  const uint32_t in_head = at - p.hk * p.ranges * grp.tiles;
  p.range = in_head / grp.tiles;
  p.tile = in_head - p.range * grp.tiles;
  p.t0 = p.range * length;
  p.count = grp.steps - p.t0 < length ? grp.steps - p.t0 : length;
  p.slots = before.more + (p.hk * grp.tiles + p.tile) * (p.ranges - 1);
  p.rows = uint32_t(grp.rows) * uint32_t(a.G) - p.tile * kRows;
  return p;
}
// The row of place `place` of the tile (those behind the last are the last): request and head.
struct RowOf {
  int64_t request, head;
};
__device__ __forceinline__ RowOf row_of(const SharedArgs& x, const Group& grp, const Piece& p,
                                        uint32_t place) {
  const uint32_t row = p.tile * kRows + (place < p.rows ? place : p.rows - 1);
  const uint32_t in = x.by_g.div(row);
  return RowOf{grp.first + int64_t(in), p.hk * x.a.G + int64_t(row - in * uint32_t(x.a.G))};
}
// Where the state of a row over a piece lies: the row's own place for its first piece, the
// place in a slot for the others; -1 for neither.
__device__ __forceinline__ int64_t state_at(const SharedArgs& x, const Piece& p, uint32_t place,
                                            const RowOf& row) {
  if (place >= p.rows) return -1;
  if (p.range == 0) return row.request * x.a.Hk * x.a.G + row.head;
  const uint32_t slot = p.slots + p.range - 1;
  return slot < uint32_t(x.groups) ? int64_t(slot) * x.stride + place : -1;
}

// 16 bytes a lane from `base` (uniform) + `offset` into LDS from base + kOffset on, as
// copy16_row_to_lds_at.
template <uint32_t kOffset>
__device__ inline void copy16_at(uint32_t lds_base, uint64_t base, uint32_t offset) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 sc1"
               :
               : "s"(lds_base), "v"(offset), "s"(base), "n"(kOffset)
               : "memory", "scc");
}
// The same with an address for each lane.
template <uint32_t kOffset>
__device__ inline void copy16_from(uint32_t lds_base, uint64_t address) {
  asm volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off sc1"
               :
               : "s"(lds_base), "v"(address), "n"(kOffset)
               : "memory", "scc");
}

template <typename T> constexpr bool kIsF16 = std::is_same_v<T, f16_t>;
template <typename T> constexpr bool kIsF32 = std::is_same_v<T, float>;

// Leaves the state of a row over a piece: o[i][e], feature 32 i + 8 (e / 4) + 4 hh + e % 4.
// Whether one of its sums is a NaN that the sum of the weights is none of.
template <int D, int NB>
__device__ __forceinline__ bool leave_state(const SharedArgs& x, const Piece& p, bool active,
                                            uint32_t place, const RowOf& row, float m, float l,
                                            const f32x16_t (&o)[NB]) {
  const int hh = threadIdx.x % 64 / 32;
  const int64_t to = active ? state_at(x, p, place, row) : -1;
  if (to < 0) return false;
  float* out = (p.range == 0 ? x.first : x.more) + to * D;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 y = make_float4(o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]);
      *reinterpret_cast<float4*>(out + 32 * i + 8 * g + 4 * hh) = y;
      sum += (y.x + y.y) + (y.z + y.w);
    }
  if (hh == 0) {
    (p.range == 0 ? x.first_ml : x.more_ml)[to] = make_float2(m, l);
    if (p.range == 0)
      x.record[row.request * x.a.Hk * x.a.G + row.head] =
          make_int4(int(p.ranges) - 1, int(p.slots), int(place), 0);
  }
  return sum != sum && l == l;
}

// Values that are not finite meet weights of 0 (or too small for their type) and make NaN
// of a row's sum; with any weight, however small, they would make it what they are, whatever
// the others are, and with none (a score of -infinity) NaN.  So the sums that are NaN, and no
// others, are made anew from those values alone: behind the work-group's pieces, once more
// through them, so that the walk over the keys has the registers.  A wave for 32 rows of a
// piece looks the values of its keys through, 1 KB a load, and takes those with such a value
// one by one.  us, 64 rows of 28 and 4 heads of 128, 131072 keys, one value a NaN: 560 (183
// without; 22900 where each row and query head went through its keys in the merge).
template <typename T, int D>
__device__ __forceinline__ void repair_piece(const SharedArgs& x, const Group& grp,
                                             const Piece& p) {
  constexpr int kPart = 16 / int(sizeof(T)), kLanes = D / kPart, kKeys = 64 / kLanes, U = 4;
  const PagedArgs& a = x.a;
  int thread = threadIdx.x;
  asm volatile("" : "+v"(thread));  // what follows from it is formed here, not kept
  const int lane = thread % 64, hh = lane / 32;
  const uint32_t place = thread / 64 * 32 + lane % 32;
  const RowOf mine = row_of(x, grp, p, place);
  const int64_t at = state_at(x, p, place, mine);
  float* sums = (p.range == 0 ? x.first : x.more) + at * D;
  const T* q = static_cast<const T*>(a.q) + mine.request * a.qn + mine.head * a.qh;
  const T* kbase = static_cast<const T*>(a.k) + p.hk * a.kh;
  const T* vbase = static_cast<const T*>(a.v) + p.hk * a.vh;
  const int32_t* table = a.table + grp.first * a.table_stride;
  auto finite = [](float v) { return __builtin_fabsf(v) < __builtin_inff(); };
  auto key_row = [&](uint32_t key, const T* base, int64_t sp, int64_t sn) {
    const uint32_t page = a.by_page.div(key);
    const int32_t id = table[page];
    return base + (is_page(id, a.num_pages) ? id : 0) * sp +
           int64_t(key - page * uint32_t(a.page)) * sn;
  };
  // Bit 4 (f / 8) + f % 4 of `nan`: feature f of the lane's half (f % 8 / 4 == hh).
  uint64_t nan = 0;
  if (at >= 0) {
    const float l = (p.range == 0 ? x.first_ml : x.more_ml)[at].y;
#pragma unroll 1
    for (int i = 0; i < D / 2 && l == l; ++i) {
      float& sum = sums[8 * (i / 4) + 4 * hh + i % 4];
      if (sum == sum) continue;
      nan |= uint64_t(1) << i;
      sum = 0.f;
    }
  }
  if (!__any(nan != 0)) return;
  struct alignas(16) Part { T x[kPart]; };
  const uint32_t end = (p.t0 + p.count) * kPrefixTile;
  for (uint32_t k0 = p.t0 * kPrefixTile; k0 < end; k0 += U * kKeys) {
    Part v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t key = k0 + u * kKeys + lane / kLanes;
      v[u] = reinterpret_cast<const Part*>(
          key_row(key < end ? key : end - 1, vbase, a.vp, a.vn))[lane % kLanes];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      bool odd = false;
#pragma unroll
      for (int e = 0; e < kPart; ++e) odd |= !finite(to_f32(v[u].x[e]));
      uint64_t found = __ballot(odd && k0 + u * kKeys + lane / kLanes < end);
      while (found) {
        const int in = __builtin_ctzll(found) / kLanes;  // of the load's keys
        found &= ~(((uint64_t(1) << kLanes) - 1) << (in * kLanes));
        const uint32_t key = k0 + u * kKeys + in;
        const T *k = key_row(key, kbase, a.kp, a.kn), *value = key_row(key, vbase, a.vp, a.vn);
        float s = 0.f;
#pragma unroll 4
        for (int d = hh * (D / 2); d < (hh + 1) * (D / 2); ++d) s += to_f32(q[d]) * to_f32(k[d]);
        const bool none = sum_halves(s) * a.scale_log2 == -__builtin_inff();
#pragma unroll 1
        for (int i = 0; i < D / 2; ++i) {
          const int f = 8 * (i / 4) + 4 * hh + i % 4;
          const float y = to_f32(value[f]);
          if (!finite(y) && (nan >> i & 1)) sums[f] += none ? __builtin_nanf("") : y;
        }
      }
    }
  }
}

// kWhole: pages of a multiple of 16 tokens, so that the 16 keys that a wave copies of
// a tile lie in one.
template <typename T, int D, bool kWhole> struct PrefixLds {
  __attribute__((aligned(1024))) unsigned char tiles[3 * DenseTile<T, D>::kTileBytes];
  PiecesLds pieces;
  int bad[kWaves];
  int32_t ids[kWhole ? 1 : kIdKeys + 2];
};
template <typename T, int D, bool kWhole>
__device__ __forceinline__ void prefix_tile(const SharedArgs& x, PrefixLds<T, D, kWhole>& shared,
                                            uint32_t block) {
  using S = DenseTile<T, D>;
  using M = typename S::M;
  using vec = typename S::vec;
  constexpr int H = S::kCopies, NCH = S::kChunks, RPC = S::kRowsPerCopy;
  constexpr uint32_t TB = uint32_t(S::kTileBytes);
  constexpr int NQK = S::NQK, NB = S::NB, NPV = S::NPV;
  // fp16's normal numbers begin at 2^-14: weights 2^7 times larger are held, 2^15 at most.
  constexpr float kBias = kIsF16<T> ? 7.f : 0.f, kSmallest = -14.f;
  unsigned char* smem = shared.tiles;
  PiecesLds& lds = shared.pieces;
  auto& sbad = shared.bad;
  auto& sid = shared.ids;
  const PagedArgs& a = x.a;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
  const int l32 = lane % 32, hh = lane / 32;
  const uint32_t page = uint32_t(a.page);

  const bool few = a.N <= 64;
  LanePieces lanes;
  const Pieces all = few ? count_in_lanes(a, uint32_t(x.groups), x.least, &lanes)
                         : count_pieces(a, uint32_t(x.groups), x.least, lds);
  // Neighbouring pieces to one XCD.
  const uint32_t eighth = uint32_t(x.groups) / 8;
  const uint32_t number = block < 8 * eighth ? block % 8 * eighth + block / 8 : block;

  // ---- copies: copy c of this wave fills tile rows [(wave*H + c)*RPC, +RPC), the lane
  // row crow + c*RPC, of which it fetches chunk p ^ chunk_swizzle(row).
  const uint32_t crow = uint32_t(wave * H * RPC + lane / NCH);
  const uint32_t c0off = uint32_t(16 * ((lane % NCH) ^ chunk_swizzle<D>(int(crow))));
  constexpr uint32_t kXorStep = D == 128 ? 16 : 32;
  static_assert(H * RPC == 16, "a wave copies 16 keys of a tile");
  const uint32_t lds_copy_base =
      uint32_t(__builtin_amdgcn_readfirstlane(int(lds_addr(smem) + uint32_t(wave * H * 1024))));
  const uint32_t kn2 = uint32_t(a.kn) * 2, vn2 = uint32_t(a.vn) * 2;
  const uint32_t krow = uint32_t(lane / NCH) * kn2, vrow = uint32_t(lane / NCH) * vn2;

  const typename S::Offsets offset(lane);

  bool nan = false;
  for (uint32_t piece = number; piece < all.count; piece += uint32_t(x.groups)) {
    Sum before;
    if (few && piece != number) __syncthreads();  // the piece before is done with its flags
    const Group grp = few ? find_in_lanes(lanes, piece, &before)
                          : find_piece(a, piece, all.length, lds, &before);
    const Piece pc = piece_at(a, grp, before, piece, all.length);
    const uint32_t hk = pc.hk, t0 = pc.t0, count = pc.count, rows = pc.rows;
    const bool active = uint32_t(32 * wave) < rows;  // uniform
    auto place_of = [&]() {  // of the lane
      uint32_t l = uint32_t(l32);
      asm volatile("" : "+v"(l));  // formed where it is used
      return uint32_t(32 * wave) + l;
    };
    const int32_t* table = a.table + int64_t(grp.first) * a.table_stride;
    const T* kbase = static_cast<const T*>(a.k) + int64_t(hk) * a.kh;
    const T* vbase = static_cast<const T*>(a.v) + int64_t(hk) * a.vh;
    bool bad = false;

    vec qreg[NQK];
    {
      const RowOf row = row_of(x, grp, pc, place_of());
      const T* qp = static_cast<const T*>(a.q) + row.request * a.qn + row.head * a.qh;
#pragma unroll
      for (int s = 0; s < NQK; ++s)
        qreg[s] = __builtin_bit_cast(vec, *reinterpret_cast<const uint4*>(qp + 16 * s + 8 * hh));
    }
#pragma unroll
    for (int s = 0; s < NQK; ++s) asm volatile("" ::"v"(qreg[s]));  // landed before the copies

    // Page ids are read as scalars, ahead of the copies that use them (a vector load would
    // make the compiler wait for all copies in flight).
    typedef const __attribute__((address_space(4))) int32_t* scalar_ptr;
    const scalar_ptr ids = (scalar_ptr)(uintptr_t)table;
    struct Next { int32_t id; uint32_t in; };
    struct At { uint64_t k, v; };  // addresses of the wave's first key
    auto find = [&](uint32_t t) {  // of tile t, at most the last one
      const uint32_t last = t0 + count - 1;
      const uint32_t key = (t < last ? t : last) * kTileKeys + uint32_t(16 * wave);
      const uint32_t p = a.by_page.div(key);
      return Next{ids[p], key - p * page};
    };
    auto check = [&](Next n) {
      if (uint32_t(n.id) >= uint32_t(a.num_pages)) {
        bad = true;
        n.id = 0;
      }
      return At{reinterpret_cast<uint64_t>(kbase + n.id * a.kp) + n.in * kn2,
                reinterpret_cast<uint64_t>(vbase + n.id * a.vp) + n.in * vn2};
    };
    // Pages of any size: the ids of kIdKeys keys in LDS.
    uint32_t id_first = 0;
    auto fill_ids = [&](uint32_t t) {
      if constexpr (!kWhole) {
        const uint32_t from = t * kTileKeys, to = (t0 + count) * kTileKeys;
        const uint32_t stop = to - from < kIdKeys ? to : from + kIdKeys;
        id_first = a.by_page.div(from);
        const uint32_t n = a.by_page.div(stop - 1) - id_first + 1;
        for (uint32_t i = tid; i < n; i += kThreads) {
          int32_t id = table[id_first + i];
          if (id < 0 || id >= a.num_pages) {
            bad = true;
            id = 0;
          }
          sid[i] = id;
        }
        __syncthreads();
      }
    };
    auto copy = [&](auto base_tag, auto c_tag, uint64_t at, const T* from, int64_t sp,
                    uint32_t row_bytes, uint32_t row_at, uint32_t t) {
      constexpr int c = decltype(c_tag)::value;
      uint32_t ch = c0off;
      asm volatile("" : "+v"(ch));  // formed at each copy
      if constexpr (kWhole) {
        copy16_at<decltype(base_tag)::value + c * 1024u>(
            lds_copy_base, at + uint32_t(c * RPC) * row_bytes, row_at + (ch ^ (c * kXorStep)));
      } else {
        const uint32_t last = t0 + count - 1;
        const uint32_t key = (t < last ? t : last) * kTileKeys + crow + uint32_t(c * RPC);
        const uint32_t p = a.by_page.div(key);
        const uint64_t row = reinterpret_cast<uint64_t>(from + sid[p - id_first] * sp) +
                             (key - p * page) * row_bytes;
        copy16_from<decltype(base_tag)::value + c * 1024u>(lds_copy_base,
                                                           row + (ch ^ (c * kXorStep)));
      }
    };
    auto copy_k = [&](auto base_tag, auto c_tag, const At& at, uint32_t t) {
      copy(base_tag, c_tag, at.k, kbase, a.kp, kn2, krow, t);
    };
    auto copy_v = [&](auto base_tag, auto c_tag, const At& at, uint32_t t) {
      copy(base_tag, c_tag, at.v, vbase, a.vp, vn2, vrow, t);
    };

    f32x16_t o[NB];
    float mneg, lsum;
    {
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
      mneg = __builtin_inff();  // -(running maximum), less kBias
      bool far = false;         // for some row, 2^16 or more in size
      lsum = 0.f;
      fill_ids(t0);
      At now{};
      Next next{};
      if constexpr (kWhole) now = check(find(t0)), next = find(t0 + 1);
      static_for<H>([&](auto c) { copy_k(lds_off<0>{}, c, now, t0); });
      static_for<H>([&](auto c) { copy_v(lds_off<TB>{}, c, now, t0); });
      // Waves without rows copy, and meet the others at the barriers.
      auto step = [&](uint32_t t, auto r_tag, auto active_tag) {
        constexpr int r = decltype(r_tag)::value;
        constexpr uint32_t k_this = uint32_t((2 * r) % 3) * TB;
        constexpr uint32_t v_this = uint32_t((2 * r + 1) % 3) * TB;
        constexpr uint32_t k_next = uint32_t((2 * r + 2) % 3) * TB;
        constexpr uint32_t v_next = k_this;
        if constexpr (!kWhole)
          if (t > t0 && (t + 1 - t0) % (kIdKeys / kTileKeys) == 0 && t + 1 < t0 + count) {
            __syncthreads();
            fill_ids(t + 1);
          }
        if constexpr (kWhole) now = check(next);
        auto kcopies = [&](auto c) { copy_k(lds_off<k_next>{}, c, now, t + 1); };
        auto vcopies = [&](auto c) { copy_v(lds_off<v_next>{}, c, now, t + 1); };
        vm_lds_barrier_keep<H>();  // K(t) landed; every wave is done with V(t-1)
        if constexpr (!decltype(active_tag)::value) {
          static_for<H>(kcopies);
          if constexpr (kWhole) next = find(t + 2);
          vm_lds_barrier_keep<H>();
          static_for<H>(vcopies);
          return;
        } else {
        f32x16_t sc[2];
        S::scores(smem + k_this, offset.k, qreg, sc, kcopies);
        if constexpr (kWhole) next = find(t + 2);  // here by the next barrier
        constexpr bool kApart = kIsF16<T>;
        float tmax = 0.f, tmin = 0.f;
        static_for<2>([&](auto half) {
          constexpr int hf = decltype(half)::value;
          if constexpr (hf == 1) settle(sc[1]);
          float u0 = max3_plain(sc[hf][0], sc[hf][1], sc[hf][2]), u1 = sc[hf][3];
#pragma unroll
          for (int e = 4; e < 16; e += 4) {
            u0 = max3_plain(u0, sc[hf][e], sc[hf][e + 1]);
            u1 = max3_plain(u1, sc[hf][e + 2], sc[hf][e + 3]);
          }
          tmax = hf == 0 ? max_plain(u0, u1) : max3_plain(tmax, u0, u1);
          if constexpr (kApart) {
            float u2 = min3_plain(sc[hf][0], sc[hf][1], sc[hf][2]), u3 = sc[hf][3];
#pragma unroll
            for (int e = 4; e < 16; e += 4) {
              u2 = min3_plain(u2, sc[hf][e], sc[hf][e + 1]);
              u3 = min3_plain(u3, sc[hf][e + 2], sc[hf][e + 3]);
            }
            tmin = hf == 0 ? min3_plain(u2, u3, u3) : min3_plain(tmin, u2, u3);
          }
        });
        // The maximum moves when a score's weight would exceed 2 to the slack.
        const float lead = tmax * a.scale_log2 + mneg;
        const bool first = mneg == __builtin_inff();
        if (__builtin_amdgcn_ballot_w64(first ? tmax > -__builtin_inff()
                                              : lead > kRescaleSlack + kBias)) {
          tmax = max_halves(tmax);
          const float top = tmax * a.scale_log2;
          float to = kBias - top;  // of this tile
          if (!(to < mneg)) to = mneg;
          const float alpha = to == mneg ? 1.f : __builtin_amdgcn_exp2f(to - mneg);
#pragma unroll
          for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[i][e] *= alpha;
          lsum *= alpha;
          mneg = to;
          far = __any(__builtin_fabsf(mneg) > 0x1p16f && mneg != __builtin_inff());
        }
        const float bias = mneg == __builtin_inff() ? 0.f : mneg;  // no score yet: weights of 0
        // Scores are scaled and rounded as the maximum is where its steps are large: a fused
        // multiplication's exact product would lie tens of powers of two beside it from 2^27
        // on, or -2^27 down: weights of 0, or beyond the type.  Below 2^16 the two are within
        // 2^-8 of each other.
        //
        // fp16 weights below its normal numbers go in apart, 2^24 times larger, where a step has
        // any: they keep their bits down to 2^-45 of the maximum's.
        vec bfrag[4], blow[kApart ? 4 : 1];
        bool small = false;
        auto weights = [&](auto exponent) {
          if constexpr (kApart) small = __any(exponent(tmin) < kSmallest);
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            __builtin_amdgcn_sched_barrier(0);
            float pr[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              pr[e] = __builtin_amdgcn_exp2f(exponent(sc[f / 2][8 * (f % 2) + e]));
            bfrag[f] = M::pack(pr);
          }
          if constexpr (kApart) {
            if (!small) return;
#pragma unroll
            for (int f = 0; f < 4; ++f) {
              float high[8], low[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                float s = sc[f / 2][8 * (f % 2) + e];
                asm volatile("" : "+v"(s));  // computed again, not kept
                const float x = exponent(s), w = __builtin_amdgcn_exp2f(x);
                high[e] = x < kSmallest ? 0.f : w;
                low[e] = x < kSmallest ? w * 0x1p24f : 0.f;
              }
              bfrag[f] = M::pack(high);
              blow[f] = M::pack(low);
              asm volatile("" : "+v"(bfrag[f]), "+v"(blow[f]));  // rounded here, not later
            }
          }
        };
        if (far)
          weights([&](float s) { return s * a.scale_log2 + bias; });
        else
          weights([&](float s) { return __builtin_fmaf(s, a.scale_log2, bias); });
        vm_lds_barrier_keep<H>();  // V(t) landed; every wave is done with K(t)
        uint32_t v0 = offset.v[0], v1 = offset.v[1];
        asm volatile("" : "+v"(v0), "+v"(v1));
        const unsigned char* vb = smem + v_this;
        if constexpr (kApart) {
          if (small) {
            auto scale = [&](float by) {
#pragma unroll
              for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[i][e] *= by;
              lsum *= by;
            };
            scale(0x1p24f);
#pragma unroll
            for (int f = 0; f < NPV; ++f) {
              __builtin_amdgcn_sched_barrier(0);
              o[f % NB] = M::run(S::vread(vb, v0, v1, f), blow[f / NB], o[f % NB]);
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) lsum = M::add_pair(blow[j / 4], j % 4, lsum);
            scale(0x1p-24f);
          }
        }
        S::values(
            vb, v0, v1, [&](int f, vec v) { o[f % NB] = M::run(v, bfrag[f / NB], o[f % NB]); },
            vcopies,
            [&](int f) {
#pragma unroll
              for (int j = f * 16 / NPV; j < (f + 1) * 16 / NPV; ++j)
                lsum = M::add_pair(bfrag[j / 4], j % 4, lsum);
            });
        }
      };
      auto steps = [&](auto active_tag) {
        const uint32_t stop = t0 + count;
        for (uint32_t t = t0; t < stop; t += 3) {
          step(t, std::integral_constant<int, 0>{}, active_tag);
          if (t + 1 < stop) step(t + 1, std::integral_constant<int, 1>{}, active_tag);
          if (t + 2 < stop) step(t + 2, std::integral_constant<int, 2>{}, active_tag);
        }
      };
      if (active)
        steps(std::true_type{});
      else
        steps(std::false_type{});
      vm_lds_barrier();  // the last copies have landed
    }
    const bool lane_bad = __any(bad);
    if (lane == 0) sbad[wave] = lane_bad;
    lds_barrier();
    float l = sum_halves(lsum);
    if (sbad[0] | sbad[1] | sbad[2] | sbad[3]) l = __builtin_nanf("");
    const uint32_t place = place_of();
    nan |= leave_state<D>(x, pc, active, place, row_of(x, grp, pc, place), -mneg, l, o);
  }
  if (!__any(nan)) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");  // what other lanes have left is read
  for (uint32_t piece = number; piece < all.count; piece += uint32_t(x.groups)) {
    Sum before;
    const Group grp = few ? find_in_lanes(lanes, piece, &before)
                          : find_in_wave(a, piece, all.length, lds, &before);
    repair_piece<T, D>(x, grp, piece_at(a, grp, before, piece, all.length));
  }
}

// The same in fp32.  A wave takes 32 rows and walks 32 keys at a time by itself, rows of K
// and V going from memory to the registers of the lane that multiplies them: S^T = K Q^T
// in D/2 v_mfma_f32_32x32x2_f32 (lane l: key or row l % 32, features from l / 32 * D / 2
// on), O^T += V^T P^T in D/2 more, weights from the scores' registers.  Where a tile has 64
// (32) rows at most, two (four) waves take turns at the same rows' keys.  Bound by the fp32
// matrix cores: 8192 cycles for 32 keys of D 128, beside which loads and exponentials are
// little (64 rows of 28 and 4 heads of 128 over 8192 keys: 137 us for 7.5 GFLOP, of which 45
// at any length; every row for itself 307).
template <int D> struct PrefixLdsF32 {
  PiecesLds pieces;
  float2 ml[kWaves][64];
  float o[3][32 * D];
};
template <int D>
__device__ __forceinline__ void prefix_tile_f32(const SharedArgs& x, PrefixLdsF32<D>& shared,
                                                uint32_t block) {
  constexpr int NB = D / 32, NQ = D / 8, kStep = 32;
  PiecesLds& lds = shared.pieces;
  const PagedArgs& a = x.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int l32 = lane % 32, hh = lane / 32;
  const bool few = a.N <= 64;
  LanePieces lanes;
  const Pieces all = few ? count_in_lanes(a, uint32_t(x.groups), x.least, &lanes)
                         : count_pieces(a, uint32_t(x.groups), x.least, lds);
  // Neighbouring pieces to one XCD.
  const uint32_t eighth = uint32_t(x.groups) / 8;
  const uint32_t number = block < 8 * eighth ? block % 8 * eighth + block / 8 : block;
  bool nan = false;
  for (uint32_t piece = number; piece < all.count; piece += uint32_t(x.groups)) {
    Sum before;
    if (few && piece != number) __syncthreads();  // the piece before is done with the LDS
    const Group grp = few ? find_in_lanes(lanes, piece, &before)
                          : find_piece(a, piece, all.length, lds, &before);
    const Piece pc = piece_at(a, grp, before, piece, all.length);
    const uint32_t hk = pc.hk, t0 = pc.t0, count = pc.count, rows = pc.rows;
    const int blocks = rows > 64 ? 4 : rows > 32 ? 2 : 1, parts = kWaves / blocks;
    const int block_of = wave % blocks, part = wave / blocks;
    const bool active = uint32_t(32 * block_of) < rows;  // uniform
    auto place_of = [&]() {  // of the lane
      uint32_t l = uint32_t(l32);
      asm volatile("" : "+v"(l));  // formed where it is used
      return uint32_t(32 * block_of) + l;
    };
    const int32_t* table = a.table + int64_t(grp.first) * a.table_stride;
    const float* kbase = static_cast<const float*>(a.k) + int64_t(hk) * a.kh + hh * (D / 2);
    const float* vbase = static_cast<const float*>(a.v) + int64_t(hk) * a.vh + l32;

    float m = -__builtin_inff(), l = 0.f;
    f32x16_t o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
    if (active) {
      const RowOf row = row_of(x, grp, pc, place_of());
      const float* qp =
          static_cast<const float*>(a.q) + row.request * a.qn + row.head * a.qh + hh * (D / 2);
      float4 q[NQ];
#pragma unroll
      for (int c = 0; c < NQ; ++c) q[c] = reinterpret_cast<const float4*>(qp)[c];
      const uint32_t end = 2 * (t0 + count), from = 2 * t0 + uint32_t(part);
      bool bad = false;
      // The lane's key of 32-key tile t (the last one for those behind it): its page entry,
      // read ahead, and its place there.
      auto key_of = [&](uint32_t t) { return (t < end ? t : end - 1) * kStep + uint32_t(l32); };
      auto entry = [&](uint32_t t) { return table[a.by_page.div(key_of(t))]; };
      struct Key { int32_t id; uint32_t in; };
      auto key_at = [&](uint32_t t, int32_t id) {
        if (!is_page(id, a.num_pages)) {
          bad = true;
          id = 0;
        }
        const uint32_t key = key_of(t);
        return Key{id, key - a.by_page.div(key) * uint32_t(a.page)};
      };
      float4 k[NQ];
      auto load_k = [&](const Key& at) {
        const float* p = kbase + at.id * a.kp + int64_t(at.in) * a.kn;
#pragma unroll
        for (int c = 0; c < NQ; ++c) k[c] = reinterpret_cast<const float4*>(p)[c];
      };
      Key now = key_at(from, entry(from));
      load_k(now);
      int32_t next_id = entry(from + parts);
      for (uint32_t t = from; t < end; t += parts) {
        // Row 8 (e / 4) + 4 hh + e % 4 of the tile: the key whose weight is the lane's e-th.
        float v[16][NB];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = 8 * (e / 4) + 4 * hh + e % 4;
          const int64_t id = __shfl(now.id, j);
          const float* p = vbase + id * a.vp + int64_t(__shfl(now.in, j)) * a.vn;
#pragma unroll
          for (int i = 0; i < NB; ++i) v[e][i] = p[32 * i];
        }
        f32x16_t sc;
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = 0.f;
#pragma unroll
        for (int c = 0; c < NQ; ++c) {
          sc = __builtin_amdgcn_mfma_f32_32x32x2f32(k[c].x, q[c].x, sc, 0, 0, 0);
          sc = __builtin_amdgcn_mfma_f32_32x32x2f32(k[c].y, q[c].y, sc, 0, 0, 0);
          sc = __builtin_amdgcn_mfma_f32_32x32x2f32(k[c].z, q[c].z, sc, 0, 0, 0);
          sc = __builtin_amdgcn_mfma_f32_32x32x2f32(k[c].w, q[c].w, sc, 0, 0, 0);
        }
        now = key_at(t + parts, next_id);
        load_k(now);
        next_id = entry(t + 2 * parts);
        float top = m;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          sc[e] *= a.scale_log2;
          top = __builtin_fmaxf(top, sc[e]);
        }
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const float base = top == -__builtin_inff() ? 0.f : top;
        if (__any(top != m)) {
          const float alpha = __builtin_amdgcn_exp2f(m - base);
          l *= alpha;
#pragma unroll
          for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
          m = top;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float w = __builtin_amdgcn_exp2f(sc[e] - base);
          l += w;
#pragma unroll
          for (int i = 0; i < NB; ++i)
            o[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[e][i], w, o[i], 0, 0, 0);
        }
      }
      l += __shfl_xor(l, 32);
      if (__any(bad)) l = __builtin_nanf("");
    }
    if (parts > 1) {  // the states of the same rows, in the order of the waves
      if (part > 0) {
        shared.ml[wave][lane] = make_float2(m, l);
        float* to = shared.o[wave - blocks];
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) to[(16 * i + e) * 64 + lane] = o[i][e];
      }
      __syncthreads();
      if (part > 0) continue;
      for (int w = wave + blocks; w < kWaves; w += blocks) {
        const float2 y = shared.ml[w][lane];
        const float top = __builtin_fmaxf(m, y.x), base = top == -__builtin_inff() ? 0.f : top;
        const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(y.x - base);
        const float* from = shared.o[w - blocks];
        l = l * f + y.y * g;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            o[i][e] = o[i][e] * f + from[(16 * i + e) * 64 + lane] * g;
        m = top;
      }
    }
    const uint32_t place = place_of();
    nan |= leave_state<D>(x, pc, active, place, row_of(x, grp, pc, place), m, l, o);
  }
  if (!__any(nan)) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");  // what other lanes have left is read
  for (uint32_t piece = number; piece < all.count; piece += uint32_t(x.groups)) {
    Sum before;
    const Group grp = few ? find_in_lanes(lanes, piece, &before)
                          : find_in_wave(a, piece, all.length, lds, &before);
    repair_piece<float, D>(x, grp, piece_at(a, grp, before, piece, all.length));
  }
}

// The work-groups of the rows' own keys, which are the shorter ones, then those of the
// prefixes, which take their places as they end.  us, 40 rows of 6 prompts / 64 rows of
// 131072 keys: in this order 26.1 / 158, own keys behind 30.1 / 164, own keys in a launch
// of their own 32.1 / 171.
template <typename T, int D, bool kWhole>
__global__ __launch_bounds__(kThreads, kIsF32<T> ? 1 : D == 128 ? 2 : 3) void prefix_kernel(
    SharedArgs x) {
  __shared__ union Lds {
    __device__ Lds() {}
    std::conditional_t<kIsF32<T>, PrefixLdsF32<D>, PrefixLds<T, D, kWhole>> prefix;
    TileLds<T, D, kFormSplit> own;
  } lds;
  const uint32_t own = uint32_t(x.a.groups);
  if (blockIdx.x < own)
    paged_tile<T, D, kWhole, kFormSplit, false, true>(x.a, lds.own, blockIdx.x);
  else if constexpr (kIsF32<T>)
    prefix_tile_f32<D>(x, lds.prefix, blockIdx.x - own);
  else
    prefix_tile<T, D, kWhole>(x, lds.prefix, blockIdx.x - own);
}

// Joins the states of a (request, query head): those of the prefix's shares, then
// those of its own keys, always in this order.
constexpr int kJoinThreads = 128;
template <typename T, int D>
__global__ __launch_bounds__(kJoinThreads) void prefix_merge_kernel(SharedArgs x) {
  constexpr int kW = kJoinThreads / 64;
  constexpr int kLanes = D / 4, kSide = kJoinThreads / kLanes, U = 8;
  constexpr int kMost = 2 * 512 + 2;
  typedef float vec4 __attribute__((ext_vector_type(4)));
  __shared__ float weight[kMost];
  __shared__ vec4 sacc[kJoinThreads];
  __shared__ float top[kW], den[kW];
  const PagedArgs& a = x.a;
  const int64_t row = blockIdx.x;
  const uint32_t Hq = uint32_t(a.Hk * a.G), n = uint32_t(row) / Hq, head = uint32_t(row) - n * Hq;
  T* out = static_cast<T*>(a.out) + n * a.on + head * a.oh;
  const int c = threadIdx.x % kLanes, side = threadIdx.x / kLanes, me = threadIdx.x;
  const uint32_t hk = head / uint32_t(a.G), in = head - hk * uint32_t(a.G);
  const uint32_t tile = in / uint32_t(a.rows), r = in - tile * uint32_t(a.rows);
  // Read together, whatever is needed of them.
  const int32_t len = a.lens[n], prefix = a.prefix_lens[n];
  const int4 record = x.record[row];
  const int2 split = a.split[int64_t(n) * a.per_request + hk * uint32_t(a.tiles) + tile];
  if (len <= 0) {
    if (side == 0)
#pragma unroll
      for (int e = 0; e < 4; ++e) out[4 * c + e] = Round<T>::store(0.f);
    return;
  }
  // The prefix's pieces, and those of the row's own segment.
  int pre = 0, pre_from = 0, place = 0;
  const int32_t shared = shared_keys(prefix, a.M * a.page);
  if (shared > 0) {
    pre_from = record.y >= 0 && record.y < x.groups ? record.y : 0;
    pre = 1 + (record.x < 0 ? 0
                            : record.x < x.groups - pre_from ? record.x : x.groups - pre_from);
    place = record.z >= 0 && record.z < x.stride ? record.z : 0;
  }
  const int own_from = split.x < 0 ? 0 : split.x / 2;
  const int own = 1 + (split.x < 0 ? 0 : split.y - own_from);
  const int64_t slots = 2 * int64_t(a.groups);
  // Part i: `own` of them from i = 0 on, those of the prefix behind.
  const int parts = own + pre;
  auto ml = [&](int i) {
    if (i < own)
      return i == 0 ? a.state_ml[row]
                    : reinterpret_cast<const float2*>(a.part)[2 * (own_from + i) * a.rows + r];
    i -= own;
    return i == 0 ? x.first_ml[row] : x.more_ml[int64_t(pre_from + i - 1) * x.stride + place];
  };
  auto state = [&](int i) {
    const float* p;
    if (i < own) {
      p = i == 0 ? a.state + row * D
                 : a.part + 2 * slots * a.rows + (int64_t(2 * (own_from + i)) * a.rows + r) * D;
    } else {
      i -= own;
      p = i == 0 ? x.first + row * D : x.more + (int64_t(pre_from + i - 1) * x.stride + place) * D;
    }
    return reinterpret_cast<const vec4*>(p)[c];
  };
  vec4 y[U];
  auto load = [&](int from) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      y[i] = state(from + i * kSide < parts ? from + i * kSide : parts - 1);
  };
  load(side);
  float m = -__builtin_inff();
  for (int i = me; i < parts; i += kJoinThreads) {
    const float2 s = ml(i);
    if (!(s.y == 0.f)) m = __builtin_fmaxf(m, s.x);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = __builtin_fmaxf(m, __shfl_xor(m, d));
  if (me % 64 == 0) top[me / 64] = m;
  lds_barrier();
#pragma unroll
  for (int w = 0; w < kW; ++w) m = __builtin_fmaxf(m, top[w]);
  float l = 0.f;
  for (int i = me; i < parts; i += kJoinThreads) {
    const float2 s = ml(i);
    const float f = __builtin_amdgcn_exp2f(s.x - m);
    weight[i] = s.y == 0.f ? -1.f : f;  // -1: no weight at all
    l += s.y == 0.f ? 0.f : f * s.y;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);
  if (me % 64 == 0) den[me / 64] = l;
  lds_barrier();
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kW; ++w) l += den[w];
  vec4 acc = vec4(0.f);
  for (int from = side; from < parts; from += U * kSide) {
    vec4 z[U];
#pragma unroll
    for (int i = 0; i < U; ++i) z[i] = y[i];
    if (from + U * kSide < parts) load(from + U * kSide);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const float f = from + i * kSide < parts ? weight[from + i * kSide] : -1.f;
      if (f > 0.f) acc += f * z[i];
      if (f == 0.f || f != f)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += f != f ? f : weighed(f, z[i][e]);
    }
  }
  sacc[me] = acc;
  lds_barrier();
  if (side != 0) return;
#pragma unroll
  for (int i = 1; i < kSide; ++i) acc += sacc[i * kLanes + c];
  struct alignas(sizeof(T) * 4) Out { T v[4]; } z;
#pragma unroll
  for (int e = 0; e < 4; ++e) z.v[e] = Round<T>::store(acc[e] / l);
  *reinterpret_cast<Out*>(out + 4 * c) = z;
}

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

// Work-groups for the prefixes: no more than there can be steps.
int64_t prefix_groups(const PagedArgs& a) {
  const int64_t tiles = a.N * a.G / kRows + (a.N + 1) / 2;  // groups have two rows at least
  const int64_t steps = a.Hk * tiles * (a.M * a.page / kPrefixTile);
  return steps < 1 ? 1 : steps < kMostGroups ? steps : kMostGroups;
}

template <typename T, int D>
hipError_t launch_prefix(const SharedArgs& x, hipStream_t stream) {
  const dim3 grid{unsigned(x.groups + x.a.groups)}, block{kThreads};
  if (x.a.page % 16 == 0)
    hipLaunchKernelGGL((prefix_kernel<T, D, true>), grid, block, 0, stream, x);
  else
    hipLaunchKernelGGL((prefix_kernel<T, D, false>), grid, block, 0, stream, x);
  return hipGetLastError();
}
template <typename T, int D>
hipError_t launch_join(const SharedArgs& x, hipStream_t stream) {
  // (At most 2^23 rows: fewer than 2^32 threads.)
  hipLaunchKernelGGL((prefix_merge_kernel<T, D>), dim3(unsigned(x.a.N * x.a.Hk * x.a.G)),
                     dim3(kJoinThreads), 0, stream, x);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_both(const SharedArgs& x, hipStream_t stream) {
  const bool wide = x.a.D == 128;
  const hipError_t e = wide ? launch_prefix<T, 128>(x, stream) : launch_prefix<T, 64>(x, stream);
  if (e != hipSuccess) return e;
  return wide ? launch_join<T, 128>(x, stream) : launch_join<T, 64>(x, stream);
}

// Whether the prefix is computed once: rows that the matrix-core form takes, a scale that
// orders scores as the products are ordered, and enough to read if every row did so for
// itself, to the tables' width (the lengths are known to the GPU only).  What the two launches
// here cost at any length grows with the rows (states written and merged), and tables of few
// keys have a form of one launch otherwise.  us, every row for itself / shared, bf16, N rows
// that share all of `keys` (room in MB at two bytes a value):
//   28 + 4 heads of 128     8 x 4096 (67) 18.5 / 23.0, 8 x 6144 (101) 23.8 / 22.8,
//     8 x 8192 (135) 28.9 / 24.2, 2 x 32768 (134) 28.0 / 31.2, 3 x 32768 (201) 38.0 / 31.2,
//     64 x 1024 (136) 24.5 / 27.3, 64 x 1536 (203) 29.6 / 27.6, 200 x 512 (216) 35.7 / 42.1,
//     200 x 1024 (426) 54.2 / 43.3
//   32 + 8 heads of 128     64 x 512 (138) 19.7 / 28.9, 64 x 1024 (273) 33.1 / 29.7,
//     200 x 256 (223) 22.7 / 45.5, 200 x 512 (433) 59.3 / 45.9
//   16 + 16 heads of 64     8 x 1024 (34) 14.2 / 14.7, 8 x 2048 (68) 19.2 / 14.6,
//     64 x 512 (138) 20.3 / 20.7, 64 x 1024 (273) 30.9 / 21.1, 200 x 256 (223) 26.4 / 49.9,
//     200 x 512 (433) 76.9 / 49.7
// fp32, 28 + 4 heads of 128: 8 x 8192 (135) 52 / 56, 4 x 16384 (134) 51 / 62, 8 x 16384 (269)
// 89 / 70, 64 x 2048 (271) 86 / 76; 16 + 16 of 64: 4 x 4096 (67) 28.4 / 27.2, 8 x 2048 (68)
// 28.1 / 23.0.  Of 138 such points the rule is 11% above the better side at one, and below 10
// at the others.
constexpr int64_t kLeastKeys = 512;
bool shares_prefix(int dtype, const PagedArgs& a) {
  const double mib = 1 << 20, rows = double(a.N * a.Hk * a.G);
  const double bytes = 4.0 * double(a.N * a.Hk * a.D) * double(a.M * a.page);
  const bool wide = a.D == 128;
  const double least = dtype == kF32 ? (wide ? 256 : 64) * mib
                       : wide        ? 80 * mib + 40 * 1024 * rows
                                     : 48 * mib + 20 * 1024 * rows;
  return a.N > 1 && bytes >= least && a.M * a.page >= kLeastKeys && a.scale_log2 >= 0.f &&
         a.kn < (int64_t(1) << 26) && a.vn < (int64_t(1) << 26) && paged_tile_form(dtype, a);
}

// The regions of the workspace, behind those of the rows' own keys (`own` bytes).
int64_t lay_out(PagedArgs& a, SharedArgs* x, char* work, int64_t own) {
  const int64_t rows = a.N * a.Hk * a.G, groups = prefix_groups(a);
  const int64_t stride = a.N * a.G < kRows ? a.N * a.G : kRows;
  int64_t at = own;
  auto take = [&](int64_t bytes) {
    char* p = work + at;
    at += round256(bytes);
    return p;
  };
  char* p[7];
  p[0] = take(8 * rows);
  p[1] = take(4 * rows * a.D);
  p[2] = take(8 * rows);
  p[3] = take(4 * rows * a.D);
  p[4] = take(8 * groups * stride);
  p[5] = take(4 * groups * stride * a.D);
  p[6] = take(16 * rows);
  if (x) {
    a.state_ml = reinterpret_cast<float2*>(p[0]);
    a.state = reinterpret_cast<float*>(p[1]);
    x->first_ml = reinterpret_cast<float2*>(p[2]);
    x->first = reinterpret_cast<float*>(p[3]);
    x->more_ml = reinterpret_cast<float2*>(p[4]);
    x->more = reinterpret_cast<float*>(p[5]);
    x->record = reinterpret_cast<int4*>(p[6]);
    x->groups = int32_t(groups);
    x->stride = int32_t(stride);
    x->by_g = FastDiv(uint32_t(a.G));
    x->least = 2;
    x->a = a;
  }
  return at;
}

}  // namespace

int64_t prefix_attn_workspace(int dtype, PagedArgs a) {
  const int64_t plain = paged_attn_workspace(dtype, a);
  if (plain < 0 || (a.D != 64 && a.D != 128)) return plain;
  const int64_t own = paged_states_workspace(dtype, a);
  if (own < 0) return -1;
  const int64_t all = lay_out(a, nullptr, nullptr, own);
  return all > plain ? all : plain;
}

hipError_t launch_prefix_attn(int dtype, PagedArgs a, void* workspace, hipStream_t stream) {
  if (!shares_prefix(dtype, a)) return launch_paged_attn(dtype, a, workspace, stream);
  char* work = static_cast<char*>(workspace);
  const int64_t own = paged_states_workspace(dtype, a);
  if (own < 0) return hipErrorInvalidValue;
  a.part = reinterpret_cast<float*>(work);
  a.split = reinterpret_cast<int2*>(work + own - round256(8 * a.N * a.per_request));
  SharedArgs x{};
  lay_out(a, &x, work, own);
  if (dtype == kF32) return launch_both<float>(x, stream);
  return dtype == kBF16 ? launch_both<bf16_t>(x, stream) : launch_both<f16_t>(x, stream);
}

}  // namespace va
