// Norms of queries and keys for each head and the position rotation, in one
// pass, and the writes of keys and values to the slots of a paged cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * w            (w given; else y = x)
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin),  f < rot/2
//     on the feature pairs (a, b) = (f, f + rot/2) or, adjacent, (2f, 2f + 1),
//     with the angle position[axis(f)] * inv_freq[f]; features from rot on stay.
//
// Everything is held in fp32 and rounded once, at the store; the angle is a
// product in fp64, reduced to a part of a turn there, since a float holds an
// angle of 10^5 radians to 0.008 only.
#include "common.h"
#include "mfma.h"
#include "paged_ops.h"

#include <initializer_list>
#include <type_traits>

namespace va {

// cos and sin of position * inv_freq, times the scaling.
__device__ inline float2 turn(const RopeArgs& a, int64_t b, int64_t s, int f) {
  int axis = 0;
#pragma unroll
  for (int i = 0; i < kRopeAxes - 1; ++i) axis += i + 1 < a.axes && f >= a.section_end[i];
  const int64_t pos = a.positions[axis * a.pa + b * a.pb + s];
  const double turns = double(pos) * double(a.inv_freq[f]) * 0.15915494309189533577;  // 1 / 2pi
  const float half = float(2.0 * (turns - __builtin_rint(turns)));                    // [-1, 1]
  float sn, cs;
  sincospif(half, &sn, &cs);
  return make_float2(cs * a.scaling, sn * a.scaling);
}

template <typename T> __device__ inline float load_f32(const void* p, int64_t i) {
  return to_f32(static_cast<const T*>(p)[i]);
}
template <typename T> __device__ inline float weight(const RopeArgs& a, const void* w, int f) {
  return a.w_f32 ? static_cast<const float*>(w)[f] : load_f32<T>(w, f);
}

// Rows of a token in order: Hq of q, Hk of k, and Hk of v in the cache form.
// Any head_dim, rotation, stride and alignment: one wave per row, lane l holds
// the features l, l + 64, ..; partners and squares go through LDS.
template <typename T>
__global__ __launch_bounds__(64) void rope_row_kernel(RopeArgs a, int64_t rows_per_token) {
  __shared__ float row[kRopeMaxD];
  const int lane = threadIdx.x;
  const int64_t item = blockIdx.x;
  const int64_t tok = item / rows_per_token, r = item % rows_per_token;
  const int64_t b = tok / a.S, s = tok % a.S;
  int64_t slot = -1;
  if (a.slots) slot = a.slots[tok];
  const bool in_cache = slot >= 0 && slot < a.num_slots;
  const int64_t page = in_cache ? slot / a.page : 0, in = in_cache ? slot % a.page : 0;
  if (r >= a.Hq + a.Hk) {  // a value row: copied
    if (!in_cache) return;
    const int64_t h = r - a.Hq - a.Hk;
    const T* x = static_cast<const T*>(a.v) + h * a.vh + s * a.vs;
    T* y = static_cast<T*>(a.vc) + page * a.vp + in * a.vn + h * a.vch;
    for (int f = lane; f < a.D; f += 64) y[f] = x[f];
    return;
  }
  const bool key = r >= a.Hq;
  const RopeRows& t = key ? a.k : a.q;
  const int64_t h = key ? r - a.Hq : r;
  const void* w = key ? a.kw : a.qw;
  const T* x = static_cast<const T*>(t.x) + b * t.sb + h * t.sh + s * t.ss;
  T* y;
  if (key && a.kc) {
    if (!in_cache) return;
    y = static_cast<T*>(a.kc) + page * a.kp + in * a.kn + h * a.kh;
  } else {
    y = static_cast<T*>(t.y) + b * t.tb + h * t.th + s * t.ts;
  }
  float sum = 0.f;
  for (int f = lane; f < a.D; f += 64) {
    const float v = to_f32(x[f]);
    row[f] = v;
    sum += v * v;
  }
  if (w) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    const float inv = 1.f / __builtin_sqrtf(sum / float(a.D) + a.eps);
    for (int f = lane; f < a.D; f += 64) row[f] = row[f] * inv * weight<T>(a, w, f);
  }
  __syncthreads();
  const int half = a.rot / 2;
  for (int f = lane; f < a.D; f += 64) {
    float out = row[f];
    if (f < a.rot) {
      const bool second = a.adjacent ? (f & 1) : f >= half;
      const int fr = a.adjacent ? f >> 1 : (second ? f - half : f);
      const float other = row[a.adjacent ? f ^ 1 : (second ? f - half : f + half)];
      const float2 cs = turn(a, b, s, fr);
      out = second ? out * cs.x + other * cs.y : out * cs.x - other * cs.y;
    }
    y[f] = Round<T>::store(out);
  }
}

// The form for head_dim 64, 128 and 256 with 16-byte aligned rows.  D / 16 lanes
// take a row, 16 features each in two pieces of 8, so that a piece is whole
// 16-byte accesses and both members of every pair are in one lane (pairs f, f +
// rot/2: pieces 8c and 8c + rot/2; neighbouring pairs: any two pieces).  A
// work-group takes kTokens tokens and all their heads: the angles, which cost as
// much as a few rows, are made once per token, go through LDS, and stay in the
// lanes' registers for all heads of their token, as do the norm weights.
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

template <typename T> struct Piece {  // 8 features as they lie in memory
  u32x4_t w[sizeof(T) / 2];
};
// kPast: past the caches, for data that is not used again soon.
template <bool kPast, typename T> __device__ inline Piece<T> load_piece(const T* p) {
  Piece<T> r;
#pragma unroll
  for (int i = 0; i < int(sizeof(T) / 2); ++i) {
    const u32x4_t* at = reinterpret_cast<const u32x4_t*>(p) + i;
    r.w[i] = kPast ? __builtin_nontemporal_load(at) : *at;
  }
  return r;
}
template <bool kPast, typename T> __device__ inline void store_piece(T* p, const Piece<T>& r) {
#pragma unroll
  for (int i = 0; i < int(sizeof(T) / 2); ++i) {
    u32x4_t* at = reinterpret_cast<u32x4_t*>(p) + i;
    if constexpr (kPast)
      __builtin_nontemporal_store(r.w[i], at);
    else
      *at = r.w[i];
  }
}
__device__ inline void unpack(const Piece<float>& r, float* x) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = bits_to_float(r.w[e / 4][e % 4]);
}
__device__ inline void unpack(const Piece<bf16_t>& r, float* x) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = bits_to_float(r.w[0][e] << 16);
    x[2 * e + 1] = bits_to_float(r.w[0][e] & 0xffff0000u);
  }
}
__device__ inline void unpack(const Piece<f16_t>& r, float* x) {
  const f16x8_t h = __builtin_bit_cast(f16x8_t, r.w[0]);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = float(h[e]);
}
__device__ inline Piece<float> pack(const float* x, float) {
  Piece<float> r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r.w[e / 4][e % 4] = float_to_bits(x[e]);
  return r;
}
template <typename T> __device__ inline Piece<T> pack(const float* x, T) {
  Piece<T> r;
  r.w[0] = __builtin_bit_cast(u32x4_t, Mfma<T>::pack(x));
  return r;
}

// Page and row of a slot; a 64-bit division only where the slot needs one.
struct SlotAt {
  int64_t page, in;
  __device__ SlotAt(int64_t slot, uint32_t size) {
    page = slot >> 32 ? int64_t(uint64_t(slot) / size) : int64_t(uint32_t(slot) / size);
    in = slot - page * size;
  }
};

// Sum over the kLanes lanes of a row (a power of two, 4 to 16), in every lane of
// it: across pairs, across quads' halves, then with the mirrored quad and half of
// a DPP row of 16 lanes, whose lanes hold equal sums by then.
template <int kLanes> __device__ inline float row_sum(float x) {
  auto add = [&x](auto ctrl) {
    x += bits_to_float(uint32_t(__builtin_amdgcn_update_dpp(0, int(float_to_bits(x)),
                                                            decltype(ctrl)::value, 0xf, 0xf, false)));
  };
  add(std::integral_constant<int, 0xb1>{});                                // quad_perm 1,0,3,2
  add(std::integral_constant<int, 0x4e>{});                                // quad_perm 2,3,0,1
  if constexpr (kLanes >= 8) add(std::integral_constant<int, 0x141>{});    // row_half_mirror
  if constexpr (kLanes >= 16) add(std::integral_constant<int, 0x140>{});   // row_mirror
  return x;
}

// The norm weights of a lane's 16 features; ones where there are none.
template <typename T>
__device__ inline void load_weights(const RopeArgs& a, const void* w, int f0, int f1, float* out) {
  if (!w) {
#pragma unroll
    for (int e = 0; e < 16; ++e) out[e] = 1.f;
  } else if (a.w_f32) {
    unpack(load_piece<false>(static_cast<const float*>(w) + f0), out);
    unpack(load_piece<false>(static_cast<const float*>(w) + f1), out + 8);
  } else {
    unpack(load_piece<false>(static_cast<const T*>(w) + f0), out);
    unpack(load_piece<false>(static_cast<const T*>(w) + f1), out + 8);
  }
}

// kCache: keys and values go to their slots, past the caches: the next to read
// them is the next step, after all other layers (8192 tokens 43.4 -> 41.9 us).
// kStream: everything goes past them.  kTokens tokens a work-group; U rows of a
// lane are in flight: the first ones before the angles are made, which take as
// long as they do, and each next one from the moment its place is free.
template <typename T, int D, int kTokens, bool kCache, bool kStream = false>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 4 : 3) void rope_kernel(RopeArgs a) {
  constexpr int kLanes = D / 16, kRows = 256 / kLanes, kHeads = kRows / kTokens;
  constexpr int U = 2;
  static_assert(kHeads >= 1, "a token a row at least");
  __shared__ float2 turns[kTokens][D / 2];
  const int half = a.rot / 2;
  const uint32_t tokens = uint32_t(a.B * a.S), t0 = blockIdx.x * kTokens;
  const int row = threadIdx.x / kLanes, c = threadIdx.x % kLanes;
  const int t = row / kHeads;
  const bool real = t0 + t < tokens;
  const uint32_t tok = real ? t0 + t : tokens - 1;
  const uint32_t b = tok / uint32_t(a.S), s = tok - b * uint32_t(a.S);
  // The lane's pieces and which of them turn.
  int f0 = 8 * c, f1 = 8 * c + D / 2;
  bool turn0 = f0 < a.rot, turn1 = f1 < a.rot;
  if (!a.adjacent) {
    turn0 = turn1 = 16 * c < a.rot;
    f1 = turn0 ? f0 + half : 16 * c + 8;
    f0 = turn0 ? f0 : 16 * c;
  }
  const int heads = real ? a.Hq + a.Hk + (kCache ? a.Hk : 0) : 0;
  Piece<T> p0[U], p1[U];
  auto load = [&](int u, int h) {
    if (h >= heads) return;
    const bool key = h >= a.Hq, value = kCache && h >= a.Hq + a.Hk;
    const RopeRows& rows = key ? a.k : a.q;
    const T* from = static_cast<const T*>(rows.x) + b * rows.sb + (key ? h - a.Hq : h) * rows.sh +
                    s * rows.ss;
    if (value) from = static_cast<const T*>(a.v) + (h - a.Hq - a.Hk) * a.vh + s * a.vs;
    p0[u] = load_piece<kStream>(from + f0);
    p1[u] = load_piece<kStream>(from + f1);
  };
#pragma unroll
  for (int u = 0; u < U; ++u) load(u, row % kHeads + u * kHeads);

  int64_t k_at = 0, v_at = 0;  // the token's place in the caches
  bool stored = real;
  if constexpr (kCache) {
    const int64_t slot = a.slots[tok];
    stored = real && slot >= 0 && slot < a.num_slots;
    const SlotAt at(stored ? slot : 0, a.page);
    k_at = at.page * a.kp + at.in * a.kn;
    v_at = at.page * a.vp + at.in * a.vn;
  }
  float wq[16], wk[16];
  load_weights<T>(a, a.qw, f0, f1, wq);
  load_weights<T>(a, a.kw, f0, f1, wk);
  for (int i = threadIdx.x; i < kTokens * half; i += 256) {
    const int ti = i / half, f = i - ti * half;
    const uint32_t toki = t0 + ti < tokens ? t0 + ti : tokens - 1;
    const uint32_t bi = toki / uint32_t(a.S), si = toki - bi * uint32_t(a.S);
    turns[ti][f] = turn(a, bi, si, f);
  }
  lds_barrier();
  float2 cs[8];  // half: pairs 8c + e; adjacent: four of each piece
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int f = a.adjacent ? (e < 4 ? f0 / 2 + e : f1 / 2 + e - 4) : f0 + e;
    cs[e] = f < half ? turns[t][f] : make_float2(1.f, 0.f);
  }

  for (int h0 = row % kHeads; h0 < heads; h0 += kHeads * U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u * kHeads;
      if (h >= heads) break;
      const bool key = h >= a.Hq, value = kCache && h >= a.Hq + a.Hk;
      T* to = static_cast<T*>(key ? a.k.y : a.q.y);
      to += key ? b * a.k.tb + (h - a.Hq) * a.k.th + s * a.k.ts
                : b * a.q.tb + h * a.q.th + s * a.q.ts;
      if constexpr (kCache) {
        if (key) to = static_cast<T*>(a.kc) + k_at + (h - a.Hq) * a.kh;
        if (value) to = static_cast<T*>(a.vc) + v_at + (h - a.Hq - a.Hk) * a.vch;
      }
      Piece<T> y0 = p0[u], y1 = p1[u];
      load(u, h + kHeads * U);
      if (!value) {
        float x[16], y[16];
        unpack(y0, x);
        unpack(y1, x + 8);
        if (key ? a.kw : a.qw) {
          float sum = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) sum = __builtin_fmaf(x[e], x[e], sum);
          sum = row_sum<kLanes>(sum);
          const float inv = 1.f / __builtin_sqrtf(sum * (1.f / D) + a.eps);
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = x[e] * inv * (key ? wk[e] : wq[e]);
        }
        if (a.adjacent) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float p = x[2 * e], q = x[2 * e + 1];
            const bool on = e < 4 ? turn0 : turn1;
            y[2 * e] = on ? __builtin_fmaf(p, cs[e].x, -(q * cs[e].y)) : p;
            y[2 * e + 1] = on ? __builtin_fmaf(q, cs[e].x, p * cs[e].y) : q;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float p = x[e], q = x[e + 8];
            y[e] = turn0 ? __builtin_fmaf(p, cs[e].x, -(q * cs[e].y)) : p;
            y[e + 8] = turn0 ? __builtin_fmaf(q, cs[e].x, p * cs[e].y) : q;
          }
        }
        y0 = pack(y, T{});
        y1 = pack(y + 8, T{});
      }
      if (kCache && key) {
        if (stored) {
          store_piece<true>(to + f0, y0);
          store_piece<true>(to + f1, y1);
        }
      } else {
        store_piece<kStream>(to + f0, y0);
        store_piece<kStream>(to + f1, y1);
      }
    }
  }
}

// Keys and values of T tokens to their slots; a slot outside the cache takes
// nothing.  Element by element, for any stride and alignment.
template <typename E>
__global__ __launch_bounds__(256) void write_element_kernel(WriteArgs a) {
  const int64_t t = blockIdx.x;
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.num_slots) return;
  const int64_t page = slot / a.page, in = slot % a.page;
  const int n = a.Hk * a.D;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int h = i / a.D, f = i % a.D;
    static_cast<E*>(a.kc)[page * a.kp + in * a.kn + h * a.kch + f] =
        static_cast<const E*>(a.k)[t * a.ks + h * a.kh + f];
    static_cast<E*>(a.vc)[page * a.vp + in * a.vn + h * a.vch + f] =
        static_cast<const E*>(a.v)[t * a.vs + h * a.vh + f];
  }
}

// The same in 16-byte pieces.  `lanes` lanes (a power of two up to 64) walk the
// pieces of a token's keys and values, U tokens at a time with all their loads in
// flight: a copy is bound by memory alone.  The stores go past the caches, as
// above (32768 tokens of 4 heads of 128 in fp16: 29.8 -> 21.8 us; 613 tokens and
// 131072 the same).
constexpr int kWriteU = 4;
__global__ __launch_bounds__(256) void write_piece_kernel(WriteArgs a, int es, int lanes) {
  const int per = 16 / es;                          // elements of a piece
  const int row = a.D / per, pieces = a.Hk * row;   // pieces of a head's row, of a token
  const int side = 256 / lanes;                     // tokens side by side
  const int lane = threadIdx.x & (lanes - 1), t = threadIdx.x / lanes;
  int64_t tok[kWriteU], ko[kWriteU], vo[kWriteU];
  bool real[kWriteU];
#pragma unroll
  for (int u = 0; u < kWriteU; ++u) {
    const int64_t at = (int64_t(blockIdx.x) * kWriteU + u) * side + t;
    tok[u] = at < a.T ? at : a.T - 1;
    const int64_t slot = a.slots[tok[u]];
    real[u] = at < a.T && slot >= 0 && slot < a.num_slots;
    const SlotAt to(real[u] ? slot : 0, a.page);
    ko[u] = to.page * a.kp + to.in * a.kn;
    vo[u] = to.page * a.vp + to.in * a.vn;
  }
  for (int i = lane; i < pieces; i += lanes) {
    const int h = i / row, f = (i - h * row) * per;
    const int64_t from = int64_t(h) * a.kh + f, vfrom = int64_t(h) * a.vh + f;
    const int64_t to = int64_t(h) * a.kch + f, vto = int64_t(h) * a.vch + f;
    auto piece = [es](const void* p, int64_t e) {
      return reinterpret_cast<u32x4_t*>(static_cast<char*>(const_cast<void*>(p)) + e * es);
    };
    u32x4_t k[kWriteU], v[kWriteU];
#pragma unroll
    for (int u = 0; u < kWriteU; ++u) {
      k[u] = *piece(a.k, tok[u] * a.ks + from);
      v[u] = *piece(a.v, tok[u] * a.vs + vfrom);
    }
#pragma unroll
    for (int u = 0; u < kWriteU; ++u)
      if (real[u]) {
        __builtin_nontemporal_store(k[u], piece(a.kc, ko[u] + to));
        __builtin_nontemporal_store(v[u], piece(a.vc, vo[u] + vto));
      }
  }
}

static bool whole_pieces(int64_t es, std::initializer_list<const void*> bases,
                         std::initializer_list<int64_t> strides) {
  for (const void* p : bases)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int64_t s : strides)
    if (s * es % 16) return false;
  return true;
}

template <typename T, int D, bool kCache>
static void launch_rope_pieces(const RopeArgs& a, hipStream_t stream) {
  // Four tokens a work-group where that leaves every CU one, else one: us at 28 +
  // 4 heads of 128 in bf16, one token / four: 600 tokens 5.0 / 6.3, 1024 6.3 / 7.3,
  // 2333 13.1 / 11.3, 8192 34.6 / 27.0, 32760 138 / 101 (eight: 13.1, 26.2, 104).
  const int64_t tokens = a.B * a.S;
  if (tokens < 1536) {
    hipLaunchKernelGGL((rope_kernel<T, D, 1, kCache>), dim3(unsigned(tokens)), dim3(256), 0,
                       stream, a);
    return;
  }
  const dim3 grid{unsigned((tokens + 3) / 4)};
  // More than the Infinity Cache holds goes past it: with the producer before and a
  // reader behind, 32760 tokens of 12 + 12 heads 224 -> 213 us, 32768 of 28 + 4 287 ->
  // 258 (alone 87.7 -> 79.4, 97.9 -> 90.0); below that it costs the reader more than
  // it saves (8192 tokens 60.7 -> 64.8).
  if constexpr (!kCache) {
    if (2 * tokens * (a.Hq + a.Hk) * D * int64_t(sizeof(T)) > (256 << 20)) {
      hipLaunchKernelGGL((rope_kernel<T, D, 4, false, true>), grid, dim3(256), 0, stream, a);
      return;
    }
  }
  hipLaunchKernelGGL((rope_kernel<T, D, 4, kCache>), grid, dim3(256), 0, stream, a);
}

template <typename T>
static void launch_rope_t(const RopeArgs& a, hipStream_t stream) {
  const bool pieces =
      a.rot % 16 == 0 &&
      whole_pieces(sizeof(T), {a.q.x, a.q.y, a.k.x, a.k.y, a.v, a.kc, a.vc, a.qw, a.kw},
                   {a.q.sb, a.q.sh, a.q.ss, a.q.tb, a.q.th, a.q.ts, a.k.sb, a.k.sh, a.k.ss, a.k.tb,
                    a.k.th, a.k.ts, a.vh, a.vs, a.kp, a.kn, a.kh, a.vp, a.vn, a.vch});
  const bool cache = a.kc != nullptr;
  if (pieces && a.D == 64) {
    cache ? launch_rope_pieces<T, 64, true>(a, stream) : launch_rope_pieces<T, 64, false>(a, stream);
  } else if (pieces && a.D == 128) {
    cache ? launch_rope_pieces<T, 128, true>(a, stream)
          : launch_rope_pieces<T, 128, false>(a, stream);
  } else if (pieces && a.D == 256) {
    cache ? launch_rope_pieces<T, 256, true>(a, stream)
          : launch_rope_pieces<T, 256, false>(a, stream);
  } else {
    const int64_t rows = a.Hq + a.Hk + (cache ? a.Hk : 0);
    hipLaunchKernelGGL(rope_row_kernel<T>, dim3(unsigned(a.B * a.S * rows)), dim3(64), 0, stream,
                       a, rows);
  }
}

hipError_t launch_rope(int dtype, const RopeArgs& a, hipStream_t stream) {
  if (dtype == kBF16)
    launch_rope_t<bf16_t>(a, stream);
  else if (dtype == kF16)
    launch_rope_t<f16_t>(a, stream);
  else
    launch_rope_t<float>(a, stream);
  return hipGetLastError();
}

hipError_t launch_write_kv(int dtype, const WriteArgs& a, hipStream_t stream) {
  const int es = dtype == kF32 ? 4 : 2;
  const dim3 block{256};
  if (a.D * es % 16 == 0 &&
      whole_pieces(es, {a.k, a.v, a.kc, a.vc},
                   {a.ks, a.kh, a.vs, a.vh, a.kp, a.kn, a.kch, a.vp, a.vn, a.vch})) {
    const int64_t pieces = int64_t(a.Hk) * a.D * es / 16;
    int lanes = 1;
    while (lanes < 64 && lanes < pieces) lanes *= 2;
    const int64_t each = 256 / lanes * kWriteU;
    hipLaunchKernelGGL(write_piece_kernel, dim3(unsigned((a.T + each - 1) / each)), block, 0,
                       stream, a, es, lanes);
    return hipGetLastError();
  }
  const dim3 grid{unsigned(a.T)};
  if (dtype == kF32)
    hipLaunchKernelGGL(write_element_kernel<uint32_t>, grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL(write_element_kernel<uint16_t>, grid, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace va
