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
#include "paged_ops.h"

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

hipError_t launch_rope(int dtype, const RopeArgs& a, hipStream_t stream) {
  const int64_t rows = a.Hq + a.Hk + (a.kc ? a.Hk : 0);
  const unsigned grid = unsigned(a.B * a.S * rows);
  if (dtype == kBF16)
    hipLaunchKernelGGL(rope_row_kernel<bf16_t>, dim3(grid), dim3(64), 0, stream, a, rows);
  else if (dtype == kF16)
    hipLaunchKernelGGL(rope_row_kernel<f16_t>, dim3(grid), dim3(64), 0, stream, a, rows);
  else
    hipLaunchKernelGGL(rope_row_kernel<float>, dim3(grid), dim3(64), 0, stream, a, rows);
  return hipGetLastError();
}

hipError_t launch_write_kv(int dtype, const WriteArgs& a, hipStream_t stream) {
  const dim3 grid{unsigned(a.T)}, block{256};
  if (dtype == kF32)
    hipLaunchKernelGGL(write_element_kernel<uint32_t>, grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL(write_element_kernel<uint16_t>, grid, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace va
