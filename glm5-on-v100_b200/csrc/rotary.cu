// Rotary embedding of query / key heads, strided in and out.
//
// For token t, head h and pair i < r/2 of the rotary part [off, off + r) of a
// head: (x1, x2) = (x[off + 2i], x[off + 2i + 1]) (GPT-J order) or
// (x[off + i], x[off + i + r/2]) (NeoX order),
//   o1 = x1 cos - x2 sin,  o2 = x2 cos + x1 sin
// with cos | sin from row positions[t] of the f32 table, the other elements of
// the head copied. Products and sums round separately in f32 (no fused
// multiply-add), once more into the output type: the same bits as the cache
// writers' rotation. The table holds whatever scaling of the frequencies the
// model uses (rope.rope_cos_sin_cache).
//
// Bound by HBM: each element is read and written once. A thread owns one "unit" of
// the head, a 16-byte vector (GPT-J: whole pairs in it; NeoX: the two vectors of
// its pairs), of several heads of a token: the angles are loaded once and stay in
// registers, the heads' loads are in flight together with them, and in-place
// rotation reads both halves of a pair before it writes either. Rows whose
// strides, offset or widths are not multiples of 16 bytes take units of one pair
// (or one copied element) instead.
// Measured: 16384 tokens x 64 heads x 64 of 256-wide rows into 576-wide ones, bf16,
// 55 us = 5.0 TB/s (77% of a plain copy's rate; a head is 128 bytes of a row), 97 us
// when each thread looked its angles up per head; 4097 x 32 x 128, half rotated, 17 us
// (3.9 TB/s); 16 tokens: the call, 12 us of host time and 4 of the kernel.
#include <algorithm>
#include <cstdint>
#include <cstdlib>

#include "common.cuh"

namespace dsa {
namespace {

constexpr int kThreads = 256;  // at most, of a block: units x heads x tokens

struct RotaryArgs {
  void* out;
  const void* x;
  int64_t ot, oh, xt, xh;  // token / head strides, elements
  const int64_t* pos;
  const float* cos_sin;    // [max_pos, r]
  int64_t max_pos;
  int r, off, width;
  int n_tok, n_head;
  int units_rot, units;    // units of the rotary part / of a whole head
};

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ void rotate(float x1, float x2, float c, float s, float& o1, float& o2) {
  o1 = __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s));
  o2 = __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s));
}

// E elements of T in one 16-byte word (VEC) or one element.
template <typename T, bool VEC>
struct Chunk {
  static constexpr int E = VEC ? 16 / (int)sizeof(T) : 1;
  T v[E];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC)
      *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
    else
      v[0] = *p;
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (VEC)
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
    else
      *p = v[0];
  }
};

// Heads of a thread whose loads are in flight at once (NeoX loads two words each).
template <bool NEOX, bool VEC>
constexpr int kHeads = NEOX && VEC ? 2 : 4;

template <typename T, bool NEOX, bool VEC>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a) {
  using C = Chunk<T, VEC>;
  constexpr int E = C::E;
  constexpr int U = kHeads<NEOX, VEC>;
  constexpr bool TWO = NEOX || !VEC;       // a pair's elements in two chunks
  constexpr int P = TWO ? E : E / 2;       // pairs of a unit
  const int t = blockIdx.x * blockDim.z + threadIdx.z;
  if (t >= a.n_tok) return;
  const int64_t pos = a.pos[t];
  const float* cs = a.cos_sin + (pos < 0 ? 0 : (pos >= a.max_pos ? a.max_pos - 1 : pos)) * a.r;
  const int half = a.r >> 1;
  const int h0 = blockIdx.y * (U * blockDim.y) + threadIdx.y;
  for (int u = threadIdx.x; u < a.units; u += blockDim.x) {
    const bool rot = u < a.units_rot;
    int at;  // in the head: of the first chunk
    if (rot) {
      at = a.off + u * (NEOX ? E : VEC ? E : 2);
    } else {
      at = (u - a.units_rot) * E;
      if (at >= a.off) at += a.r;
    }
    const T* x = reinterpret_cast<const T*>(a.x) + (t * a.xt + h0 * a.xh + at);
    T* o = reinterpret_cast<T*>(a.out) + (t * a.ot + h0 * a.oh + at);
    const int64_t xs = a.xh * blockDim.y, os = a.oh * blockDim.y;
    C lo[U], hi[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (h0 + k * (int)blockDim.y >= a.n_head) continue;
      lo[k].load(x + k * xs);
      if (TWO && rot) hi[k].load(x + k * xs + (NEOX ? half : 1));
    }
    if (rot) {
      float c[P], s[P];
      const float* q = cs + u * P;
      if constexpr (P % 4 == 0) {
#pragma unroll
        for (int e = 0; e < P; e += 4) {
          *reinterpret_cast<float4*>(c + e) = __ldg(reinterpret_cast<const float4*>(q + e));
          *reinterpret_cast<float4*>(s + e) = __ldg(reinterpret_cast<const float4*>(q + half + e));
        }
      } else if constexpr (P == 2) {
        *reinterpret_cast<float2*>(c) = __ldg(reinterpret_cast<const float2*>(q));
        *reinterpret_cast<float2*>(s) = __ldg(reinterpret_cast<const float2*>(q + half));
      } else {
        c[0] = __ldg(q);
        s[0] = __ldg(q + half);
      }
#pragma unroll
      for (int k = 0; k < U; ++k)
#pragma unroll
        for (int e = 0; e < P; ++e) {
          T& x1 = TWO ? lo[k].v[e] : lo[k].v[(2 * e) % E];
          T& x2 = TWO ? hi[k].v[e] : lo[k].v[(2 * e + 1) % E];
          float o1, o2;
          rotate(to_f32(x1), to_f32(x2), c[e], s[e], o1, o2);
          x1 = from_f32<T>(o1);
          x2 = from_f32<T>(o2);
        }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (h0 + k * (int)blockDim.y >= a.n_head) continue;
      lo[k].store(o + k * os);
      if (TWO && rot) hi[k].store(o + k * os + (NEOX ? half : 1));
    }
  }
}

template <typename T, bool NEOX, bool VEC>
void launch(const RotaryArgs& a, cudaStream_t s) {
  constexpr int U = kHeads<NEOX, VEC>;
  // a block: the units of as many heads of a token as it takes, U a thread; where
  // that leaves threads over, more tokens
  const int x = std::min(a.units, kThreads);
  const int y = std::min((a.n_head + U - 1) / U, kThreads / x);
  const int z = std::min(std::min(kThreads / (x * y), 64), a.n_tok);
  const dim3 grid((unsigned)((a.n_tok + z - 1) / z), (unsigned)((a.n_head + U * y - 1) / (U * y)));
  rotary_kernel<T, NEOX, VEC><<<grid, dim3(x, y, z), 0, s>>>(a);
}

template <typename T>
void launch(const RotaryArgs& a, bool neox, bool vec, cudaStream_t s) {
  if (neox)
    vec ? launch<T, true, true>(a, s) : launch<T, true, false>(a, s);
  else
    vec ? launch<T, false, true>(a, s) : launch<T, false, false>(a, s);
}

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_rotary_embedding(void* out, int64_t out_tok_stride, int64_t out_head_stride, const void* x,
                                    int64_t x_tok_stride, int64_t x_head_stride, int dtype, const int64_t* positions,
                                    const float* cos_sin, int64_t max_pos, int rotary_dim, int rope_offset,
                                    int rope_neox, int n_tok, int n_head, int width, void* stream) {
  clear_error();
  DSA_REQUIRE(dtype == DSA_F16 || dtype == DSA_BF16 || dtype == DSA_F32, DSA_ERR_INVALID,
              "rotary_embedding: x must be f16, bf16 or f32");
  DSA_REQUIRE(n_tok >= 0 && n_head >= 0 && width > 0, DSA_ERR_INVALID,
              "rotary_embedding: bad sizes (tokens=%d heads=%d width=%d)", n_tok, n_head, width);
  DSA_REQUIRE(rotary_dim > 0 && rotary_dim % 2 == 0 && rope_offset >= 0 &&
                  (int64_t)rope_offset + rotary_dim <= width,
              DSA_ERR_INVALID, "rotary_embedding: rotary part [%d, %d) must be even and inside the head's %d elements",
              rope_offset, rope_offset + rotary_dim, width);
  DSA_REQUIRE(width <= 2048, DSA_ERR_UNSUPPORTED, "rotary_embedding: heads are at most 2048 wide (got %d)", width);
  DSA_REQUIRE(n_tok <= (1 << 28) && n_head <= 65535, DSA_ERR_UNSUPPORTED, "rotary_embedding: too many tokens or heads");
  if (n_tok == 0 || n_head == 0) return DSA_OK;
  // no two of out's heads share an element: the nearer of its strides spans a head,
  // the other all the heads at the nearer one
  const int64_t st = n_tok > 1 ? out_tok_stride : INT64_MAX, sh = n_head > 1 ? out_head_stride : INT64_MAX;
  const int64_t near = std::min(st, sh), far = std::max(st, sh), n_near = st <= sh ? n_tok : n_head;
  DSA_REQUIRE(near >= width && (far == INT64_MAX || (far - width) / (n_near - 1) >= near),
              DSA_ERR_INVALID, "rotary_embedding: heads of out overlap (strides %lld, %lld)", (long long)out_tok_stride,
              (long long)out_head_stride);
  const int item = dtype == DSA_F32 ? 4 : 2;
  const int e = 16 / item;
  // x moved against out by `d` elements, with out's strides: a head of one meets a head
  // of the other when d lies within a width of a distance between two heads
  if ((n_tok == 1 || out_tok_stride == x_tok_stride) && (n_head == 1 || out_head_stride == x_head_stride)) {
    const int64_t d = ((int64_t)reinterpret_cast<uintptr_t>(out) - (int64_t)reinterpret_cast<uintptr_t>(x)) / item;
    const int64_t n_far = st <= sh ? n_head : n_tok;
    bool meet = false;
    for (int64_t f = d / far - 1; d != 0 && f <= d / far + 1; ++f) {
      if (std::abs(f) >= n_far) continue;
      const int64_t r = d - (f == 0 ? 0 : f * far);
      for (int64_t k = r / near - 1; k <= r / near + 1; ++k)
        meet |= std::abs(k) < n_near && std::abs(r - (k == 0 ? 0 : k * near)) < width;
    }
    DSA_REQUIRE(!meet, DSA_ERR_INVALID, "rotary_embedding: out overlaps x without being x");
  }
  DSA_REQUIRE(out && x && positions && cos_sin && max_pos > 0, DSA_ERR_INVALID, "rotary_embedding: null pointer");
  auto is16 = [&](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = is16(out) && is16(x) && is16(cos_sin) && out_tok_stride % e == 0 && out_head_stride % e == 0 &&
                   x_tok_stride % e == 0 && x_head_stride % e == 0 && width % e == 0 && rope_offset % e == 0 &&
                   rotary_dim % (rope_neox ? 2 * e : e) == 0 && rotary_dim % 8 == 0;
  RotaryArgs a{};
  a.out = out;
  a.x = x;
  a.ot = out_tok_stride;
  a.oh = out_head_stride;
  a.xt = x_tok_stride;
  a.xh = x_head_stride;
  a.pos = positions;
  a.cos_sin = cos_sin;
  a.max_pos = max_pos;
  a.r = rotary_dim;
  a.off = rope_offset;
  a.width = width;
  a.n_tok = n_tok;
  a.n_head = n_head;
  const bool copy = !(out == x && out_tok_stride == x_tok_stride && out_head_stride == x_head_stride);
  a.units_rot = vec ? (rope_neox ? rotary_dim / 2 / e : rotary_dim / e) : rotary_dim / 2;
  a.units = a.units_rot + (copy ? (width - rotary_dim) / (vec ? e : 1) : 0);  // in place nothing is copied
  cudaStream_t s = as_stream(stream);
  if (dtype == DSA_F32)
    launch<float>(a, rope_neox != 0, vec, s);
  else if (dtype == DSA_F16)
    launch<__half>(a, rope_neox != 0, vec, s);
  else
    launch<__nv_bfloat16>(a, rope_neox != 0, vec, s);
  return check_launch("rotary_kernel");
}
