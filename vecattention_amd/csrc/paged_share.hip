// Pages that several rows of a paged key-value cache hold: the next step's rows
// from this one's (fork), the pages in use moved together (compact), and the
// pages that neighbouring rows begin with (prefix).  Integer work on tables, a
// count for each page and the list of free pages.
//
// shares[p] counts the rows that hold page p beyond the first: 0 for a page of
// one row and for a free one, so that the plan, which takes pages off the free
// list, has nothing to note.  A page whose last row goes has -1, which is how
// the fork finds it.
//
// What bounds them are launches, and reads that wait for one another, not bytes: in us,
// a fork of 512 rows of up to 2092 pages 33 in four launches (7.6 MB, 2 at a copy's rate),
// a compaction of 256 rows 34 in five, prefixes of 256 rows of 8200 pages 9.3 in two.
// Each launch ends where all of a sum has to be there before its first use; those over
// pages have a work-group for 4096 of them, too few to fill the GPU below a million pages
// (scan, count and place take 7 to 9 us for 140,000 to 400,000).  Rows look for their parent,
// or their group, among all rows before them: a fork of 8192 rows of 8 pages 92, of 65536
// 2014; prefixes 141 to 192 and 7629 to 10372.
#include "common.h"
#include "lanes.h"
#include "paged_ops.h"

namespace va {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kChunk = 1024;       // table entries of a work-group
constexpr int kPagesPer = 4096;    // pages of a work-group: 64 words of 64 bits

__device__ inline int64_t head_of(const int32_t* head, int64_t F) {
  const int64_t h = head ? *head : 0;
  return h < 0 ? 0 : h > F ? F : h;
}
// For counts that other work-groups of the same launch change.
__device__ inline int32_t load_agent(const int32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline void add_agent(int32_t* p, int32_t v) {
  __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether any thread of the work-group has `x`.
__device__ inline bool any_of(bool x) { return __syncthreads_or(x) != 0; }

// Sum over a wave.
__device__ inline int32_t wave_total(int32_t x) {
  return __builtin_amdgcn_readlane(wave_inclusive_sum(x), 63);
}
// Exclusive sum over the work-group and the total.  `part`: kT / 64 values of LDS, which may be
// written again after the next barrier.
template <int kT>
__device__ inline int32_t block_exclusive_sum(int32_t x, int32_t* part, int32_t* total) {
  const int lane = threadIdx.x % 64, w = threadIdx.x / 64;
  const int32_t s = wave_inclusive_sum(x);
  if (lane == 63) part[w] = s;
  __syncthreads();
  int32_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kT / 64; ++i) {
    if (i < w) before += part[i];
    all += part[i];
  }
  *total = all;
  return before + s - x;
}

// ---------------------------------------------------------------------------
// Fork.  With s1 = shares - (rows that held p) + (rows that hold it now), the
// steps are: the new tables and s1 (fork_rows, fork_counts); the pages with s1 <
// 0 and the rows that need a page of their own (fork_scan); who gets which page
// (fork_place).  Rows keep a page that they would write to if they alone hold
// it; where rows share it, the first of them keeps it if no row that has it whole
// and no row outside the call holds it too.  All results are sums and ranks, so
// they do not depend on the order of the atomics.
struct ForkWork {
  uint32_t* least;    // (P) first row that would write to a page
  int32_t* writers;   // (P) and their number; both are set where a row writes
  uint8_t* first;     // (R) no row before it has its parent; (N) behind it: rows with children
  int32_t* end;       // (R) page that the row would write to, -1 for none
  int32_t* rank;      // (R) number of the row's copy, -1 for none
  int32_t* row_of;    // (R) row of each copy
  uint64_t* gone;     // (P / 64) pages with s1 < 0
  int32_t* counts;    // of them in each chunk of kPagesPer, then the number of copies
};
__host__ __device__ inline int64_t fork_chunks(int64_t P) {
  return P > 0 ? (P + kPagesPer - 1) / kPagesPer : 1;
}

ForkWork fork_work(void* workspace, int64_t R, int64_t P) {
  const int64_t chunks = fork_chunks(P);
  ForkWork w;
  w.gone = static_cast<uint64_t*>(workspace);
  w.least = reinterpret_cast<uint32_t*>(w.gone + chunks * (kPagesPer / 64));
  w.writers = reinterpret_cast<int32_t*>(w.least + P);
  w.end = w.writers + P;
  w.rank = w.end + R;
  w.row_of = w.rank + R;
  w.counts = w.row_of + R;
  w.first = reinterpret_cast<uint8_t*>(w.counts + chunks + 1);
  return w;
}

// Row r's parent or -1, its length and pages.
struct ForkRow {
  int32_t parent, len;
  uint32_t held, had;  // pages, and its parent's
  __device__ ForkRow(const ForkArgs& a, int64_t r) {
    parent = a.parents[r];
    if (parent < 0 || parent >= a.N) {
      parent = -1;
      len = 0;
      held = had = 0;
      return;
    }
    const int32_t was = a.kv_lens[parent];
    len = was > 0 ? was : 0;
    if (a.keep) {
      const int32_t most = a.keep[r] > 0 ? a.keep[r] : 0;
      len = len < most ? len : most;
    }
    held = held_pages(len, a.page, uint32_t(a.M));
    had = held_pages(was, a.page, uint32_t(a.M));
  }
  // The page that its next token goes into beside its own, or -1.
  __device__ int32_t open(const ForkArgs& a) const {
    const int64_t at = open_page(len, a.page, uint32_t(a.M));
    if (parent < 0 || at < 0) return -1;
    const int32_t id = a.table[parent * a.table_stride + at];
    return is_page(id, a.P) ? id : -1;
  }
};

// Work-groups [0, R * chunks): entries of the new tables; then one for each row of
// before; behind them copies of the shares and of the free list.
__global__ __launch_bounds__(kThreads) void fork_rows_kernel(ForkArgs a, ForkWork w,
                                                             int64_t chunks) {
  int64_t g = blockIdx.x;
  if (g < a.R * chunks) {
    const int64_t r = g / chunks, first = (g - r * chunks) * kChunk;
    const ForkRow row(a, r);
    const int32_t* from = a.table + (row.parent < 0 ? 0 : row.parent) * a.table_stride;
    for (int64_t k = first + threadIdx.x; k < first + kChunk && k < a.M; k += kThreads)
      a.table_out[r * a.M + k] = k < row.held ? from[k] : -1;
    if (first != 0) return;
    bool earlier = false;
    for (int64_t j = threadIdx.x; j < r; j += kThreads) earlier |= a.parents[j] == row.parent;
    earlier = any_of(earlier);
    if (threadIdx.x == 0) {
      w.first[r] = !earlier;
      a.kv_out[r] = row.len;
      const int32_t p = row.open(a);
      w.end[r] = p;
      if (p >= 0) {
        w.least[p] = 0xffffffffu;
        w.writers[p] = 0;
      }
    }
    return;
  }
  g -= a.R * chunks;
  if (g < a.N) {
    bool child = false;
    for (int64_t j = threadIdx.x; j < a.R; j += kThreads) child |= a.parents[j] == int32_t(g);
    child = any_of(child);
    if (threadIdx.x == 0) w.first[a.R + g] = child;
    return;
  }
  g -= a.N;
  const int64_t step = int64_t(gridDim.x - a.R * chunks - a.N) * kThreads;
  for (int64_t i = g * kThreads + threadIdx.x; i < a.P + a.F; i += step) {
    if (i < a.P)
      a.shares_out[i] = a.shares[i];
    else
      a.free_out[i - a.P] = a.free_pages[i - a.P];
  }
}

// What a page's count changes by: a row's first child stands for the row itself
// in the pages that it keeps.  Work-groups [0, R * chunks) are the children's,
// the others those of the rows that have none.
__global__ __launch_bounds__(kThreads) void fork_counts_kernel(ForkArgs a, ForkWork w,
                                                               int64_t chunks) {
  const int64_t g = blockIdx.x, i = g / chunks, first = (g - i * chunks) * kChunk;
  int64_t from, to;
  int32_t parent, change;
  if (i < a.R) {
    const ForkRow row(a, i);
    if (first == 0 && threadIdx.x == 0) {
      const int32_t p = w.end[i];
      if (p >= 0) {
        atomicMin(w.least + p, uint32_t(i));
        add_agent(w.writers + p, 1);
      }
    }
    parent = row.parent;
    if (parent < 0 || first >= row.had) return;
    if (w.first[i])
      from = row.held, to = row.had, change = -1;
    else
      from = 0, to = row.held, change = 1;
  } else {
    parent = int32_t(i - a.R);
    to = held_pages(a.kv_lens[parent], a.page, uint32_t(a.M));
    if (first >= to || w.first[i]) return;
    from = 0, change = -1;
  }
  if (from < first) from = first;
  if (to > first + kChunk) to = first + kChunk;
  for (int64_t k = from + threadIdx.x; k < to; k += kThreads) {
    const int32_t id = a.table[parent * a.table_stride + k];
    if (is_page(id, a.P)) add_agent(a.shares_out + id, change);
  }
}

// The pages that went, 64 to a word, and how many of each chunk; the last
// work-group numbers the rows' copies.
__global__ __launch_bounds__(kThreads) void fork_scan_kernel(ForkArgs a, ForkWork w) {
  __shared__ int32_t part[kWaves];
  const int64_t chunks = gridDim.x - 1, g = blockIdx.x;
  const int lane = threadIdx.x % 64;
  if (g < chunks) {
    int32_t mine = 0;
    for (int64_t p = g * kPagesPer + threadIdx.x; p < (g + 1) * kPagesPer; p += kThreads) {
      const bool gone = p < a.P && a.shares_out[p] < 0;
      const uint64_t word = __ballot(gone);
      if (lane == 0) w.gone[p / 64] = word;
      if (gone) a.shares_out[p] = 0;
      mine += gone;
    }
    int32_t total;
    block_exclusive_sum<kThreads>(mine, part, &total);
    if (threadIdx.x == 0) w.counts[g] = total;
    return;
  }
  int32_t before = 0;
  for (int64_t base = 0; base < a.R; base += kThreads) {
    const int64_t r = base + threadIdx.x;
    bool copies = false;
    if (r < a.R) {
      const int32_t p = w.end[r];
      if (p >= 0) {
        const int32_t s = load_agent(a.shares_out + p);  // below 0, or made 0 by its chunk
        copies = w.least[p] != uint32_t(r) || (s > 0 ? s : 0) + 1 > w.writers[p];
      }
    }
    int32_t total;
    const int32_t at = before + block_exclusive_sum<kThreads>(copies, part, &total);
    if (r < a.R) w.rank[r] = copies ? at : -1;
    if (copies) w.row_of[at] = int32_t(r);
    before += total;
    __syncthreads();  // `part` is written again
  }
  if (threadIdx.x == 0) w.counts[chunks] = before;
}

// Freed page j lies at head - freed + j of the list, copy j takes what is there.
__global__ __launch_bounds__(kThreads) void fork_place_kernel(ForkArgs a, ForkWork w) {
  __shared__ int32_t part[2][kWaves];
  const int64_t chunks = fork_chunks(a.P), g = blockIdx.x;
  const int lane = threadIdx.x % 64;
  const int32_t taken = w.counts[chunks];
  int32_t x = 0, y = 0, freed, before;
  for (int64_t i = threadIdx.x; i < chunks; i += kThreads) {
    x += w.counts[i];
    if (i < g) y += w.counts[i];
  }
  block_exclusive_sum<kThreads>(x, part[0], &freed);
  block_exclusive_sum<kThreads>(y, part[1], &before);
  const int64_t head = head_of(a.free_head, a.F), top = head - freed;
  if (g < chunks) {
    if (w.counts[g] == 0) return;
    // Lane i of every wave: word i, and the freed pages of the words before it.
    const uint64_t mine = w.gone[g * (kPagesPer / 64) + lane];
    const int32_t bits = __builtin_popcountll(mine);
    const int32_t ahead = before + wave_inclusive_sum(bits) - bits;
    for (int i = threadIdx.x / 64; i < kPagesPer / 64; i += kWaves) {
      const uint64_t word =
          uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(mine)), i))) |
          uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(mine >> 32)), i))) << 32;
      const int32_t j = __builtin_amdgcn_readlane(ahead, i) +
                        __builtin_popcountll(word & ((uint64_t(1) << lane) - 1));
      if (!(word >> lane & 1)) continue;
      const int32_t id = int32_t(g * kPagesPer + 64 * i + lane);
      if (j < taken) {
        const int32_t r = w.row_of[j];
        a.copy_dst[r] = id;
        a.table_out[r * a.M + open_page(a.kv_out[r], a.page, uint32_t(a.M))] = id;
      } else if (top + j >= 0) {
        a.free_out[top + j] = id;
      }
    }
    return;
  }
  // Rows: kThreads to a work-group.
  const int64_t r = (g - chunks) * kThreads + threadIdx.x;
  if (r == 0) {
    const int64_t left = top + taken;
    *a.head_out = int32_t(left < 0 ? 0 : left < 0x7fffffff ? left : 0x7fffffff);
  }
  if (r >= a.R) return;
  const int32_t p = w.end[r], j = w.rank[r], len = a.kv_out[r];
  if (p >= 0 && w.least[p] == uint32_t(r)) {
    // The copies' share in the page goes.
    const int32_t copies = w.writers[p] - (j < 0), s = a.shares_out[p] - copies;
    a.shares_out[p] = s > 0 ? s : 0;
  }
  a.copy_src[r] = j < 0 ? -1 : p;
  a.copy_rows[r] = j < 0 ? 0 : int32_t(uint32_t(len) % a.page);
  if (j < 0) {
    a.copy_dst[r] = -1;
  } else if (j >= freed) {
    const int32_t id = free_page(a.free_pages, a.F, top + j);
    a.copy_dst[r] = id;
    a.table_out[r * a.M + open_page(len, a.page, uint32_t(a.M))] = id;
  }
}

// ---------------------------------------------------------------------------
// Compact.  U: the pages in the tables and the free ones, in order; the t in the
// tables shall be the first t of U.  Those behind (movers) go to the free ones
// among the first t (holes), in order.
struct CompactWork {
  uint8_t *used, *open;  // (P) whether a table, or the list, has the page
  uint64_t *used_bits, *open_bits;  // 64 pages to a word; open: and not used
  int2* counts;          // of both in each chunk of kPagesPer
  int32_t* moved;        // (P) number of a page's move, -1 for none
};
CompactWork compact_work(void* workspace, int64_t P) {
  const int64_t chunks = fork_chunks(P), words = chunks * (kPagesPer / 64);
  CompactWork w;
  w.used_bits = static_cast<uint64_t*>(workspace);
  w.open_bits = w.used_bits + words;
  w.counts = reinterpret_cast<int2*>(w.open_bits + words);
  w.moved = reinterpret_cast<int32_t*>(w.counts + chunks);
  w.used = reinterpret_cast<uint8_t*>(w.moved + P);
  w.open = w.used + chunks * kPagesPer;
  return w;
}

__global__ __launch_bounds__(kThreads) void compact_clear_kernel(CompactArgs a, CompactWork w) {
  // Both byte arrays lie behind `moved`, 4-byte aligned.
  const int64_t words = 2 * fork_chunks(a.P) * (kPagesPer / 4), half = a.P / 2;
  const int64_t step = int64_t(gridDim.x) * kThreads;
  for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
       i < words + 2 * half + a.F + a.P; i += step) {
    int64_t k = i;
    if (k < words) {
      reinterpret_cast<uint32_t*>(w.used)[k] = 0;
    } else if ((k -= words) < half) {
      a.copy_src[k] = -1;
    } else if ((k -= half) < half) {
      a.copy_dst[k] = -1;
    } else if ((k -= half) < a.F) {
      a.free_out[k] = a.free_pages[k];
    } else {
      a.shares_out[k - a.F] = a.shares[k - a.F];
    }
  }
}

// Bytes, which every thread may store to: with a bit for each page and atomic ORs this
// took 95 us for 180,000 entries and 280,000 free pages.
__global__ __launch_bounds__(kThreads) void compact_mark_kernel(CompactArgs a, CompactWork w,
                                                                int64_t chunks) {
  const int64_t g = blockIdx.x;
  if (g < a.N * chunks) {
    const int64_t n = g / chunks, first = (g - n * chunks) * kChunk;
    int64_t to = held_pages(a.kv_lens[n], a.page, uint32_t(a.M));
    if (to > first + kChunk) to = first + kChunk;
    for (int64_t k = first + threadIdx.x; k < to; k += kThreads) {
      const int32_t id = a.table[n * a.table_stride + k];
      if (is_page(id, a.P)) w.used[id] = 1;
    }
    return;
  }
  const int64_t step = int64_t(gridDim.x - a.N * chunks) * kThreads;
  for (int64_t i = head_of(a.free_head, a.F) + (g - a.N * chunks) * kThreads + threadIdx.x;
       i < a.F; i += step) {
    const int32_t id = a.free_pages[i];
    if (is_page(id, a.P)) w.open[id] = 1;
  }
}

__global__ __launch_bounds__(kThreads) void compact_count_kernel(CompactWork w) {
  __shared__ int32_t part[2][kWaves];
  const int64_t g = blockIdx.x;
  const int lane = threadIdx.x % 64;
  int32_t used = 0, open = 0;
  for (int64_t p = g * kPagesPer + threadIdx.x; p < (g + 1) * kPagesPer; p += kThreads) {
    const bool u = w.used[p] != 0, o = w.open[p] != 0 && !u;
    const uint64_t x = __ballot(u), y = __ballot(o);
    if (lane == 0) {
      w.used_bits[p / 64] = x;
      w.open_bits[p / 64] = y;
    }
    used += u;
    open += o;
  }
  int32_t tu, to;
  block_exclusive_sum<kThreads>(used, part[0], &tu);
  block_exclusive_sum<kThreads>(open, part[1], &to);
  if (threadIdx.x == 0) w.counts[g] = make_int2(tu, to);
}

// Where every page goes.
__global__ __launch_bounds__(kThreads) void compact_place_kernel(CompactArgs a, CompactWork w) {
  __shared__ int32_t part[4][kWaves];
  __shared__ int2 edge;   // chunk that holds the page of rank t, and U's pages before it
  __shared__ int32_t low; // free pages before that chunk
  __shared__ int32_t shole;
  constexpr int kWords = kPagesPer / 64;
  const int64_t chunks = gridDim.x, g = blockIdx.x;
  const int64_t per = (chunks + kThreads - 1) / kThreads, lo = threadIdx.x * per;
  const int64_t hi = lo + per < chunks ? lo + per : chunks;
  int32_t u = 0, o = 0, ub = 0, ob = 0;
  for (int64_t i = lo; i < hi; ++i) {
    const int2 c = w.counts[i];
    u += c.x;
    o += c.y;
    if (i < g) ub += c.x, ob += c.y;
  }
  int32_t t, free, used0, open0;
  const int32_t u0 = block_exclusive_sum<kThreads>(u, part[0], &t);
  const int32_t o0 = block_exclusive_sum<kThreads>(o, part[1], &free);
  block_exclusive_sum<kThreads>(ub, part[2], &used0);
  block_exclusive_sum<kThreads>(ob, part[3], &open0);
  if (threadIdx.x == 0) {
    edge = make_int2(-1, 0);
    low = 0;
  }
  __syncthreads();
  {
    int32_t x = u0, y = o0;
    for (int64_t i = lo; i < hi; ++i) {
      const int2 c = w.counts[i];
      if (x + y <= t && t < x + y + c.x + c.y) {
        edge = make_int2(int(i), x + y);
        low = y;
      }
      x += c.x;
      y += c.y;
    }
  }
  __syncthreads();
  // Moves: the holes, free pages of rank below t.  A wave counts the chunk that rank t lies in
  // (in none, all free ones are holes: there are none).
  const int lane = threadIdx.x % 64;
  if (threadIdx.x < 64) {
    int32_t holes = free;
    if (edge.x >= 0) {
      const uint64_t x = w.used_bits[edge.x * int64_t(kWords) + lane];
      const uint64_t y = w.open_bits[edge.x * int64_t(kWords) + lane];
      const int32_t n = __builtin_popcountll(x | y);
      const int32_t rank = edge.y + wave_inclusive_sum(n) - n;
      int32_t mine = rank + n <= t ? __builtin_popcountll(y) : 0;
      if (rank < t && t < rank + n) {  // the word with rank t
        uint64_t all = x | y;
        for (int32_t k = rank; k < t; ++k) {
          const uint64_t bit = all & -all;
          mine += (y & bit) != 0;
          all ^= bit;
        }
      }
      holes = low + wave_total(mine);
    }
    if (lane == 0) shole = holes;
  }
  __syncthreads();
  const int32_t moves = shole;
  if (g == 0 && threadIdx.x == 0) {
    *a.num_moves = moves;
    *a.head_out = int32_t(a.F - free);
  }
  // The pages of this chunk, a word of 64 to a wave at a time; lane i: word i.
  const uint64_t mx = w.used_bits[g * kWords + lane], my = w.open_bits[g * kWords + lane];
  const int32_t nx = __builtin_popcountll(mx), ny = __builtin_popcountll(my);
  const int32_t ax = used0 + wave_inclusive_sum(nx) - nx;
  const int32_t ay = open0 + wave_inclusive_sum(ny) - ny;
  auto word_of = [](uint64_t x, int i) {
    return uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(x)), i))) |
           uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(x >> 32)), i))) << 32;
  };
  for (int i = threadIdx.x / 64; i < kWords; i += kWaves) {
    const uint64_t x = word_of(mx, i), y = word_of(my, i), below = (uint64_t(1) << lane) - 1;
    const int32_t ru = __builtin_amdgcn_readlane(ax, i) + __builtin_popcountll(x & below);
    const int32_t ro = __builtin_amdgcn_readlane(ay, i) + __builtin_popcountll(y & below);
    const int64_t p = g * kPagesPer + 64 * i + lane;
    if (p >= a.P) continue;
    const bool is_used = x >> lane & 1, is_open = y >> lane & 1;
    const int32_t rank = ru + ro;
    int32_t move = -1;
    if (is_used && rank >= t) {
      move = ru - (t - moves);
      a.copy_src[move] = int32_t(p);
    }
    if (is_open && rank < t) a.copy_dst[ro] = int32_t(p);
    if ((is_used || is_open) && rank >= t) a.free_out[a.F - free + (rank - t)] = int32_t(p);
    w.moved[p] = move;
  }
}

__global__ __launch_bounds__(kThreads) void compact_tables_kernel(CompactArgs a, CompactWork w,
                                                                  int64_t chunks) {
  const int64_t g = blockIdx.x;
  if (g < a.N * chunks) {
    const int64_t n = g / chunks, first = (g - n * chunks) * kChunk;
    const int64_t held = held_pages(a.kv_lens[n], a.page, uint32_t(a.M));
    for (int64_t k = first + threadIdx.x; k < first + kChunk && k < a.M; k += kThreads) {
      int32_t id = a.table[n * a.table_stride + k];
      if (k < held && is_page(id, a.P)) {
        const int32_t move = w.moved[id];
        if (move >= 0) id = a.copy_dst[move];
      }
      a.table_out[n * a.M + k] = id;
    }
    return;
  }
  const int32_t moves = *a.num_moves;
  const int64_t step = int64_t(gridDim.x - a.N * chunks) * kThreads;
  for (int64_t i = (g - a.N * chunks) * kThreads + threadIdx.x; i < moves; i += step) {
    const int32_t from = a.copy_src[i], to = a.copy_dst[i];
    a.shares_out[to] = a.shares[from];
    a.shares_out[from] = 0;
  }
}

// ---------------------------------------------------------------------------
// Prefix.  Row n goes with the row before it when both hold tokens and have the
// same id (without ids: the same first page).
__device__ inline bool joins(const PrefixArgs& a, int64_t n) {
  if (n == 0 || a.kv_lens[n] <= 0 || a.kv_lens[n - 1] <= 0) return false;
  if (a.ids) return a.ids[n] == a.ids[n - 1];
  const int32_t id = a.M ? a.table[n * a.table_stride] : -1;
  return id >= 0 && id == a.table[(n - 1) * a.table_stride];
}

// A work-group a row: the first row of its group, and the whole pages that the
// two begin with.
__global__ __launch_bounds__(kThreads) void prefix_rows_kernel(PrefixArgs a, int32_t* first,
                                                               int32_t* pages) {
  __shared__ int32_t best[kWaves];
  const int64_t n = blockIdx.x;
  const int lane = threadIdx.x % 64;
  // The last row up to this one that does not join.
  int32_t lead = 0;
  for (int64_t i = threadIdx.x; i <= n; i += kThreads)
    if (!joins(a, i)) lead = int32_t(i);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t other = __shfl_xor(lead, d);
    lead = lead > other ? lead : other;
  }
  if (lane == 0) best[threadIdx.x / 64] = lead;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) lead = lead > best[i] ? lead : best[i];
  const int32_t len = a.kv_lens[n] > 0 ? a.kv_lens[n] : 0;
  int64_t whole = uint32_t(len) / a.page;
  if (whole > a.M) whole = a.M;
  const int32_t *row = a.table + n * a.table_stride, *with = a.table + lead * a.table_stride;
  int64_t same = whole;
  constexpr int kPer = 16;
  for (int64_t k0 = 0; k0 < whole; k0 += kPer * kThreads) {
    int64_t miss = whole;  // the thread's first entry that differs
    int32_t x[kPer], y[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int64_t k = k0 + e * kThreads + threadIdx.x < whole ? k0 + e * kThreads + threadIdx.x
                                                                : whole - 1;
      x[e] = row[k];
      y[e] = with[k];
    }
#pragma unroll
    for (int e = kPer - 1; e >= 0; --e) {
      const int64_t k = k0 + e * kThreads + threadIdx.x;
      if (k < whole && (x[e] < 0 || x[e] != y[e])) miss = k;
    }
    if (any_of(miss < whole)) {
      // The least over the work-group.
      int32_t m = int32_t(miss);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int32_t other = __shfl_xor(m, d);
        m = m < other ? m : other;
      }
      if (lane == 0) best[threadIdx.x / 64] = m;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kWaves; ++i) m = m < best[i] ? m : best[i];
      same = m;
      break;
    }
  }
  if (threadIdx.x == 0) {
    first[n] = lead;
    pages[n] = int32_t(same);
  }
}

// A wave a row: the fewest pages over its group, and the group's rows.
__global__ __launch_bounds__(kThreads) void prefix_groups_kernel(PrefixArgs a,
                                                                 const int32_t* first,
                                                                 const int32_t* pages) {
  const int64_t n = int64_t(blockIdx.x) * kWaves + threadIdx.x / 64;
  const int lane = threadIdx.x % 64;
  if (n >= a.N) return;
  const int32_t lead = first[n];
  int32_t least = 0x7fffffff;
  int64_t rows = 0;
  for (int64_t base = lead; base < a.N; base += 64) {
    const int64_t i = base + lane;
    const bool in = i < a.N && first[i] == lead;
    if (in) least = least < pages[i] ? least : pages[i];
    const uint64_t all = __ballot(in);
    rows += __builtin_popcountll(all);
    if (all != ~uint64_t(0)) break;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t other = __shfl_xor(least, d);
    least = least < other ? least : other;
  }
  if (lane == 0) {
    const int32_t len = rows > 1 ? int32_t(uint32_t(least) * a.page) : 0;
    a.prefix_lens[n] = len;
    a.group_rows[n] = n == lead && len > 0 ? int32_t(rows) : 0;
  }
}

// ---------------------------------------------------------------------------
// The same for small batches and pools in one work-group, with the counts in LDS:
// the launches and the reads that wait for one another are what such a call takes
// (us, 8 rows: fork 14.8 in the general form, 8.2 here; compaction of 12 rows 18.1 and 8.4;
// prefixes of 8 rows 9.4 and 5.9).
constexpr int kSmallThreads = 1024, kSmallWaves = kSmallThreads / 64;
constexpr int kSmallRows = 256;
constexpr int kSmallPages = 8192;       // 32 KB of counts
// Table entries, above which the general forms are as fast.  us, here / general: fork (rows
// before and after), 8 rows of 2048 entries 14.2 / 19, 64 of 256 15.2 / 19, 32 of 1024 24 /
// 20.5; compaction, 16384 entries 17.6 / 21, 32768 32 / 22; prefixes, 16384 entries 7.4 to
// 10.0 / 9.5, 32768 11.5 to 17.6 / 9.5.
constexpr int64_t kSmallForkEntries = 32768, kSmallEntries = 16384;
constexpr int32_t kGone = -(1 << 30);   // the count of a page that no row holds any more

__global__ __launch_bounds__(kSmallThreads) void fork_small_kernel(ForkArgs a, FastDiv by_m) {
  __shared__ int32_t s[kSmallPages];
  __shared__ int32_t parent[kSmallRows], held[kSmallRows], had[kSmallRows], ends[kSmallRows];
  __shared__ int32_t old_held[kSmallRows], freed[kSmallRows];
  __shared__ uint8_t is_first[kSmallRows], kids[kSmallRows], later[kSmallRows];
  __shared__ int32_t part[2][kSmallWaves];
  const int t = threadIdx.x, lane = t % 64, wave = t / 64;
  const int R = int(a.R), N = int(a.N), P = int(a.P), F = int(a.F);
  const uint32_t M = uint32_t(a.M);
  const int64_t head = head_of(a.free_head, a.F);
  for (int p = t; p < P; p += kSmallThreads) s[p] = a.shares[p];
  int32_t len = 0;
  if (t < R) {
    const ForkRow row(a, t);
    parent[t] = row.parent;
    held[t] = int32_t(row.held);
    had[t] = int32_t(row.had);
    ends[t] = row.open(a);
    is_first[t] = 1;
    later[t] = 0;
    len = row.len;
    a.kv_out[t] = len;
  } else if (t >= kSmallRows && t < kSmallRows + N) {
    old_held[t - kSmallRows] = int32_t(held_pages(a.kv_lens[t - kSmallRows], a.page, M));
    kids[t - kSmallRows] = 0;
  }
  __syncthreads();
  // Whether a row before has the same parent, or ends in the same page: four threads a row.
  const int32_t end = t < R ? ends[t] : -1;
  {
    constexpr int kParts = kSmallThreads / kSmallRows;
    const int r = t % kSmallRows, run = (R + kParts - 1) / kParts, j0 = t / kSmallRows * run;
    const int stop = j0 + run < R ? j0 + run : R;
    if (r < R) {
      const int32_t p = parent[r], at = ends[r];
      int same = 0, writes = 0;
#pragma unroll 8
      for (int j = j0; j < stop; ++j) {
        same |= int(j < r) & int(parent[j] == p);
        writes |= int(j < r) & int(ends[j] == at);
      }
      if (same) is_first[r] = 0;
      if (writes) later[r] = 1;
      if (t < R && p >= 0) kids[p] = 1;
    }
  }
  __syncthreads();
  const bool not_least = t < R && later[t] != 0;
  for (uint32_t e = t; e < uint32_t(R) * M; e += kSmallThreads) {
    const uint32_t r = by_m.div(e), k = e - r * M;
    int32_t id = -1;
    const bool in = int32_t(k) < held[r];
    if (in || (is_first[r] && int32_t(k) < had[r])) {
      id = a.table[parent[r] * a.table_stride + k];
      if (is_page(id, P) && !(in && is_first[r])) atomicAdd(&s[id], in ? 1 : -1);
    }
    a.table_out[e] = in ? id : -1;
  }
  for (uint32_t e = t; e < uint32_t(N) * M; e += kSmallThreads) {
    const uint32_t n = by_m.div(e), k = e - n * M;
    if (kids[n] || int32_t(k) >= old_held[n]) continue;
    const int32_t id = a.table[n * a.table_stride + k];
    if (is_page(id, P)) atomicAdd(&s[id], -1);
  }
  __syncthreads();
  // The pages that went: a run of whole words of 64 to a wave.
  const int run = (P + kSmallThreads - 1) / kSmallThreads * 64, from = wave * run;
  int32_t mine = 0;
  for (int p = from + lane; p < from + run; p += 64) {
    const bool gone = p < P && s[p] < 0;
    if (gone) s[p] = kGone;
    mine += __builtin_popcountll(__ballot(gone));
  }
  if (lane == 0) part[0][wave] = mine;
  __syncthreads();
  int32_t before = 0, nf = 0;
#pragma unroll
  for (int i = 0; i < kSmallWaves; ++i) {
    if (i < wave) before += part[0][i];
    nf += part[0][i];
  }
  // Rows that get a page of their own leave the shared one: all but the first, then the first
  // if somebody holds it still.
  bool copies = end >= 0 && not_least;
  if (copies) atomicSub(&s[end], 1);
  __syncthreads();
  if (end >= 0 && !not_least && s[end] > 0) {
    copies = true;
    --s[end];
  }
  const uint64_t word = __ballot(copies);
  if (lane == 0) part[1][wave] = __builtin_popcountll(word);
  __syncthreads();
  int32_t rank = 0, nt = 0;
#pragma unroll
  for (int i = 0; i < kSmallWaves; ++i) {
    if (i < wave) rank += part[1][i];
    nt += part[1][i];
  }
  rank += __builtin_popcountll(word & ((uint64_t(1) << lane) - 1));
  const int64_t top = head - nf;
  for (int p = from + lane; p < from + run; p += 64) {
    const int32_t v = p < P ? s[p] : 0;
    const bool gone = v < kGone / 2;
    const uint64_t all = __ballot(gone);
    const int32_t j = before + __builtin_popcountll(all & ((uint64_t(1) << lane) - 1));
    before += __builtin_popcountll(all);
    if (p < P) a.shares_out[p] = v > 0 ? v : 0;
    if (gone) {
      if (j < nt)
        freed[j] = p;
      else if (top + j >= 0)
        a.free_out[top + j] = p;
    }
  }
  for (int i = t; i < F; i += kSmallThreads)
    if (i < top + nt || i >= head) a.free_out[i] = a.free_pages[i];
  __syncthreads();
  if (t == 0) *a.head_out = int32_t(top + nt < 0 ? 0 : top + nt);
  if (t >= R) return;
  int32_t to = -1;
  if (copies) {
    to = rank < nf ? freed[rank] : free_page(a.free_pages, a.F, top + rank);
    a.table_out[uint32_t(t) * M + uint32_t(open_page(len, a.page, M))] = to;
  }
  a.copy_src[t] = copies ? end : -1;
  a.copy_dst[t] = to;
  a.copy_rows[t] = copies ? int32_t(uint32_t(len) % a.page) : 0;
}

__global__ __launch_bounds__(kSmallThreads) void compact_small_kernel(CompactArgs a,
                                                                      FastDiv by_m) {
  constexpr int kWords = kSmallPages / 32;
  __shared__ uint32_t used[kWords], open[kWords];
  __shared__ int32_t pu[kWords], po[kWords], part[3][kSmallWaves];
  __shared__ int32_t hole[kSmallPages / 2];
  const int t = threadIdx.x;
  const int N = int(a.N), P = int(a.P), F = int(a.F), half = P / 2;
  const uint32_t M = uint32_t(a.M);
  const int64_t head = head_of(a.free_head, a.F);
  for (int i = t; i < kWords; i += kSmallThreads) used[i] = open[i] = 0;
  __syncthreads();
  for (uint32_t e = t; e < uint32_t(N) * M; e += kSmallThreads) {
    const uint32_t n = by_m.div(e), k = e - n * M;
    if (k >= held_pages(a.kv_lens[n], a.page, M)) continue;
    const int32_t id = a.table[n * a.table_stride + k];
    if (is_page(id, P)) atomicOr(&used[id / 32], 1u << (id % 32));
  }
  for (int64_t i = head + t; i < F; i += kSmallThreads) {
    const int32_t id = a.free_pages[i];
    if (is_page(id, P)) atomicOr(&open[id / 32], 1u << (id % 32));
  }
  __syncthreads();
  uint32_t x = 0, y = 0;
  if (t < kWords) {
    x = used[t];
    y = open[t] & ~x;
    open[t] = y;
  }
  const int32_t nx = __builtin_popcount(x), ny = __builtin_popcount(y);
  int32_t total, free, moves;
  const int32_t ux = block_exclusive_sum<kSmallThreads>(nx, part[0], &total);
  const int32_t uy = block_exclusive_sum<kSmallThreads>(ny, part[1], &free);
  int32_t holes = 0;
  if (t < kWords) {
    pu[t] = ux;
    po[t] = uy;
    uint32_t all = x | y;
    const int32_t rank = ux + uy, n = nx + ny;
    if (rank + n <= total) {
      holes = ny;
    } else {
      for (int32_t k = rank; k < total; ++k) {
        const uint32_t bit = all & -all;
        holes += (y & bit) != 0;
        all ^= bit;
      }
    }
  }
  block_exclusive_sum<kSmallThreads>(holes, part[2], &moves);
  auto ranks = [&](int p, int32_t* ru, int32_t* ro) {
    const uint32_t below = (1u << (p % 32)) - 1;
    *ru = pu[p / 32] + __builtin_popcount(used[p / 32] & below);
    *ro = po[p / 32] + __builtin_popcount(open[p / 32] & below);
  };
  auto has = [](const uint32_t* bits, int p) { return (bits[p / 32] >> (p % 32) & 1) != 0; };
  __syncthreads();
  for (int p = t; p < P; p += kSmallThreads) {
    int32_t ru, ro;
    ranks(p, &ru, &ro);
    const bool is_used = has(used, p), is_open = has(open, p);
    if (is_open && ru + ro < total) {
      hole[ro] = p;
      a.copy_dst[ro] = p;
    }
    if ((is_used || is_open) && ru + ro >= total)
      a.free_out[F - free + (ru + ro - total)] = p;
    if (is_used && ru + ro >= total) a.copy_src[ru - (total - moves)] = p;
  }
  for (int i = t; i < F - free; i += kSmallThreads) a.free_out[i] = a.free_pages[i];
  for (int i = moves + t; i < half; i += kSmallThreads) a.copy_src[i] = a.copy_dst[i] = -1;
  if (t == 0) {
    *a.num_moves = moves;
    *a.head_out = F - free;
  }
  __syncthreads();
  // The new number of a page.
  auto place = [&](int p) {
    int32_t ru, ro;
    ranks(p, &ru, &ro);
    return ru + ro >= total ? hole[ru - (total - moves)] : p;
  };
  for (int p = t; p < P; p += kSmallThreads) {
    int32_t ru, ro;
    ranks(p, &ru, &ro);
    if (has(open, p) && ru + ro < total) continue;  // a hole: its new page writes it
    const int32_t v = a.shares[p];
    const bool moved = has(used, p) && ru + ro >= total;
    a.shares_out[p] = moved ? 0 : v;
    if (moved) a.shares_out[hole[ru - (total - moves)]] = v;
  }
  for (uint32_t e = t; e < uint32_t(N) * M; e += kSmallThreads) {
    const uint32_t n = by_m.div(e), k = e - n * M;
    int32_t id = a.table[n * a.table_stride + k];
    if (k < held_pages(a.kv_lens[n], a.page, M) && is_page(id, P)) id = place(id);
    a.table_out[e] = id;
  }
}

// Up to 64 rows: a lane a row for the groups, a wave a row for the pages.
__global__ __launch_bounds__(kSmallThreads) void prefix_small_kernel(PrefixArgs a) {
  __shared__ int32_t pages[64];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, N = int(a.N);
  const uint64_t leads = __ballot(lane < N && !joins(a, lane));
  for (int n = wave; n < N; n += kSmallWaves) {
    const int lead = 63 - __builtin_clzll(leads & (~uint64_t(0) >> (63 - n)));
    const int32_t len = a.kv_lens[n] > 0 ? a.kv_lens[n] : 0;
    int64_t whole = uint32_t(len) / a.page;
    if (whole > a.M) whole = a.M;
    const int32_t *row = a.table + n * a.table_stride, *with = a.table + lead * a.table_stride;
    int64_t same = whole;
    constexpr int kPer = 4;
    for (int64_t k0 = 0; k0 < whole; k0 += 64 * kPer) {
      uint64_t miss[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int64_t k = k0 + 64 * e + lane;
        miss[e] = __ballot(k < whole && (row[k] < 0 || row[k] != with[k]));
      }
      bool found = false;
#pragma unroll
      for (int e = kPer - 1; e >= 0; --e)
        if (miss[e]) same = k0 + 64 * e + __builtin_ctzll(miss[e]), found = true;
      if (found) break;
    }
    if (lane == 0) pages[n] = int32_t(same);
  }
  __syncthreads();
  if (wave != 0 || lane >= N) return;
  const int lead = 63 - __builtin_clzll(leads & (~uint64_t(0) >> (63 - lane)));
  const uint64_t later = lead < 63 ? leads >> (lead + 1) << (lead + 1) : 0;
  const int end = later ? __builtin_ctzll(later) : N, rows = end - lead;
  int32_t least = pages[lead];
  for (int i = lead + 1; i < end; ++i) least = least < pages[i] ? least : pages[i];
  const int32_t len = rows > 1 ? int32_t(uint32_t(least) * a.page) : 0;
  a.prefix_lens[lane] = len;
  a.group_rows[lane] = lane == lead && len > 0 ? rows : 0;
}

unsigned extra_groups(int64_t work) {
  const int64_t g = (work + 4 * kThreads - 1) / (4 * kThreads);
  return unsigned(g < 1 ? 1 : g > 1024 ? 1024 : g);
}

}  // namespace

int64_t fork_workspace_bytes(int64_t R, int64_t P) {
  const int64_t chunks = fork_chunks(P);
  return 8 * chunks * (kPagesPer / 64) + 4 * (2 * P + 3 * R + chunks + 1) + R + kForkMostRows;
}

hipError_t launch_paged_fork(const ForkArgs& a, void* workspace, hipStream_t stream) {
  if (a.N <= kSmallRows && a.R <= kSmallRows && a.P <= kSmallPages &&
      a.F <= 2 * kSmallPages && (a.N + a.R) * a.M <= kSmallForkEntries) {
    hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(kSmallThreads), 0, stream, a,
                       FastDiv(uint32_t(a.M > 0 ? a.M : 1)));
    return hipGetLastError();
  }
  const ForkWork w = fork_work(workspace, a.R, a.P);
  const int64_t per_row = a.M > 0 ? (a.M + kChunk - 1) / kChunk : 1;
  hipLaunchKernelGGL(fork_rows_kernel, dim3(unsigned(a.R * per_row + a.N) + extra_groups(a.P + a.F)),
                     dim3(kThreads), 0, stream, a, w, per_row);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (a.R + a.N > 0) {
    hipLaunchKernelGGL(fork_counts_kernel, dim3(unsigned((a.R + a.N) * per_row)), dim3(kThreads),
                       0, stream, a, w, per_row);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const int64_t chunks = fork_chunks(a.P);
  hipLaunchKernelGGL(fork_scan_kernel, dim3(unsigned(chunks + 1)), dim3(kThreads), 0, stream, a,
                     w);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t rows = a.R > 0 ? (a.R + kThreads - 1) / kThreads : 1;
  hipLaunchKernelGGL(fork_place_kernel, dim3(unsigned(chunks + rows)), dim3(kThreads), 0, stream,
                     a, w);
  return hipGetLastError();
}

int64_t compact_workspace_bytes(int64_t P) {
  const int64_t chunks = fork_chunks(P);
  return 16 * chunks * (kPagesPer / 64) + 8 * chunks + 4 * P + 2 * chunks * kPagesPer;
}

hipError_t launch_paged_compact(const CompactArgs& a, void* workspace, hipStream_t stream) {
  if (a.P <= kSmallPages && a.F <= 2 * kSmallPages && a.N * a.M <= kSmallEntries) {
    hipLaunchKernelGGL(compact_small_kernel, dim3(1), dim3(kSmallThreads), 0, stream, a,
                       FastDiv(uint32_t(a.M > 0 ? a.M : 1)));
    return hipGetLastError();
  }
  const CompactWork w = compact_work(workspace, a.P);
  const int64_t per_row = a.M > 0 ? (a.M + kChunk - 1) / kChunk : 1;
  const int64_t chunks = fork_chunks(a.P);
  hipLaunchKernelGGL(compact_clear_kernel, dim3(extra_groups(3 * a.P + a.F)), dim3(kThreads), 0,
                     stream, a, w);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(compact_mark_kernel, dim3(unsigned(a.N * per_row) + extra_groups(a.F)),
                     dim3(kThreads), 0, stream, a, w, per_row);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(compact_count_kernel, dim3(unsigned(chunks)), dim3(kThreads), 0, stream, w);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(compact_place_kernel, dim3(unsigned(chunks)), dim3(kThreads), 0, stream, a, w);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(compact_tables_kernel, dim3(unsigned(a.N * per_row) + extra_groups(a.P / 2)),
                     dim3(kThreads), 0, stream, a, w, per_row);
  return hipGetLastError();
}

int64_t prefix_workspace_bytes(int64_t N) { return 8 * N; }

hipError_t launch_paged_prefix(const PrefixArgs& a, void* workspace, hipStream_t stream) {
  if (a.N <= 64 && a.N * a.M <= kSmallEntries) {
    hipLaunchKernelGGL(prefix_small_kernel, dim3(1), dim3(kSmallThreads), 0, stream, a);
    return hipGetLastError();
  }
  int32_t* first = static_cast<int32_t*>(workspace);
  int32_t* pages = first + a.N;
  hipLaunchKernelGGL(prefix_rows_kernel, dim3(unsigned(a.N)), dim3(kThreads), 0, stream, a, first,
                     pages);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(prefix_groups_kernel, dim3(unsigned((a.N + kWaves - 1) / kWaves)),
                     dim3(kThreads), 0, stream, a, first, pages);
  return hipGetLastError();
}

}  // namespace va
