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
// Bound by HBM: each element is read and written once; the table row of a token
// stays in L1 over its heads. A block takes whole tokens, or a range of one
// token's heads, as "units" of one 16-byte vector (GPT-J: whole pairs in it;
// NeoX: the two vectors of its pairs), so every load and store is 16 bytes wide
// and in-place rotation reads both halves of a pair before it writes either.
// Rows whose strides, offset or widths are not multiples of 16 bytes take units
// of one pair (or one copied element) instead.
#include <algorithm>

#include "common.cuh"

namespace dsa {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;      // units whose loads are in flight at once
constexpr int kMaxUnits = 2048; // units per block: 8 per thread

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
  int tokens_per_block, heads_per_block;
  uint32_t mul_units;      // ceil(2^32 / units): exact quotients below 2^16
  int copy;                // 0: in place, nothing to copy
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

template <typename T, bool NEOX, bool VEC>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a) {
  using C = Chunk<T, VEC>;
  constexpr int E = C::E;
  const int t0 = blockIdx.x * a.tokens_per_block;
  const int h0 = blockIdx.y * a.heads_per_block;
  const int nt = min(a.tokens_per_block, a.n_tok - t0);
  const int nh = min(a.heads_per_block, a.n_head - h0);
  const int half = a.r >> 1;
  const int per_token = nh * a.units;
  const int n = nt * per_token;
  for (int base = threadIdx.x; base < n; base += kThreads * kUnroll) {
    C lo[kUnroll], hi[kUnroll];
    int first[kUnroll], token[kUnroll], unit[kUnroll];
    int64_t src[kUnroll], dst[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      int j = base + k * kThreads;
      token[k] = -1;
      if (j >= n) continue;
      int t = 0;
      if (nt > 1) {
        t = j / per_token;
        j -= t * per_token;
      }
      const int h = a.mul_units ? (int)__umulhi((uint32_t)j, a.mul_units) : j;
      const int u = j - h * a.units;
      if (u >= a.units_rot && !a.copy) continue;
      token[k] = t0 + t;
      unit[k] = u;
      src[k] = (int64_t)(t0 + t) * a.xt + (int64_t)(h0 + h) * a.xh;
      dst[k] = (int64_t)(t0 + t) * a.ot + (int64_t)(h0 + h) * a.oh;
      const T* x = reinterpret_cast<const T*>(a.x) + src[k];
      if (u < a.units_rot) {
        // the pair's two elements, or for GPT-J vectors the one word that holds E/2 pairs
        first[k] = a.off + (NEOX ? u * E : u * (VEC ? E : 2));
        lo[k].load(x + first[k]);
        if (NEOX || !VEC) hi[k].load(x + first[k] + (NEOX ? half : 1));
      } else {
        const int c = (u - a.units_rot) * E;
        first[k] = c < a.off ? c : c + a.r;
        lo[k].load(x + first[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      if (token[k] < 0) continue;
      T* o = reinterpret_cast<T*>(a.out) + dst[k] + first[k];
      if (unit[k] >= a.units_rot) {
        lo[k].store(o);
        continue;
      }
      int64_t p = a.pos[token[k]];
      p = p < 0 ? 0 : (p >= a.max_pos ? a.max_pos - 1 : p);
      const float* cs = a.cos_sin + p * a.r;
      if constexpr (VEC && !NEOX) {
        constexpr int P = E / 2;  // pairs in the word
        float c[P], s[P];
        const float* q = cs + unit[k] * P;
        if constexpr (P == 4) {
          *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(q);
          *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(q + half);
        } else {
          *reinterpret_cast<float2*>(c) = *reinterpret_cast<const float2*>(q);
          *reinterpret_cast<float2*>(s) = *reinterpret_cast<const float2*>(q + half);
        }
#pragma unroll
        for (int e = 0; e < P; ++e) {
          float o1, o2;
          rotate(to_f32(lo[k].v[2 * e]), to_f32(lo[k].v[2 * e + 1]), c[e], s[e], o1, o2);
          lo[k].v[2 * e] = from_f32<T>(o1);
          lo[k].v[2 * e + 1] = from_f32<T>(o2);
        }
        lo[k].store(o);
      } else {
        float c[E], s[E];
        const float* q = cs + unit[k] * E;
        if constexpr (VEC) {
#pragma unroll
          for (int e = 0; e < E; e += 4) {
            *reinterpret_cast<float4*>(c + e) = *reinterpret_cast<const float4*>(q + e);
            *reinterpret_cast<float4*>(s + e) = *reinterpret_cast<const float4*>(q + half + e);
          }
        } else {
          c[0] = q[0];
          s[0] = q[half];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float o1, o2;
          rotate(to_f32(lo[k].v[e]), to_f32(hi[k].v[e]), c[e], s[e], o1, o2);
          lo[k].v[e] = from_f32<T>(o1);
          hi[k].v[e] = from_f32<T>(o2);
        }
        lo[k].store(o);
        hi[k].store(o + (NEOX ? half : 1));
      }
    }
  }
}

template <typename T>
void launch(const RotaryArgs& a, bool neox, bool vec, dim3 grid, cudaStream_t s) {
  if (neox)
    vec ? rotary_kernel<T, true, true><<<grid, kThreads, 0, s>>>(a)
        : rotary_kernel<T, true, false><<<grid, kThreads, 0, s>>>(a);
  else
    vec ? rotary_kernel<T, false, true><<<grid, kThreads, 0, s>>>(a)
        : rotary_kernel<T, false, false><<<grid, kThreads, 0, s>>>(a);
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
  DSA_REQUIRE(out && x && positions && cos_sin && max_pos > 0, DSA_ERR_INVALID, "rotary_embedding: null pointer");
  const int item = dtype == DSA_F32 ? 4 : 2;
  const int e = 16 / item;
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
  a.copy = !(out == x && out_tok_stride == x_tok_stride && out_head_stride == x_head_stride);
  a.units_rot = vec ? (rope_neox ? rotary_dim / 2 / e : rotary_dim / e) : rotary_dim / 2;
  a.units = a.units_rot + (a.copy ? (width - rotary_dim) / (vec ? e : 1) : 0);
  // units per block: 256 a pass, up to eight passes while the blocks still fill the GPU about four times
  const int64_t total = (int64_t)n_tok * n_head * a.units;
  const int nsm = sm_count(current_device());
  const int64_t want = std::min<int64_t>(kMaxUnits, std::max<int64_t>(kThreads, total / ((int64_t)nsm * 4)));
  a.heads_per_block = (int)std::min<int64_t>(n_head, std::max<int64_t>(1, want / a.units));
  a.tokens_per_block = a.heads_per_block == n_head
                           ? (int)std::min<int64_t>(n_tok, std::max<int64_t>(1, want / ((int64_t)n_head * a.units)))
                           : 1;
  a.mul_units = a.units == 1 ? 0u : (uint32_t)(((1ull << 32) + a.units - 1) / a.units);  // 0: the quotient is j
  const dim3 grid((unsigned)((n_tok + a.tokens_per_block - 1) / a.tokens_per_block),
                  (unsigned)((n_head + a.heads_per_block - 1) / a.heads_per_block));
  cudaStream_t s = as_stream(stream);
  if (dtype == DSA_F32)
    launch<float>(a, rope_neox != 0, vec, grid, s);
  else if (dtype == DSA_F16)
    launch<__half>(a, rope_neox != 0, vec, grid, s);
  else
    launch<__nv_bfloat16>(a, rope_neox != 0, vec, grid, s);
  return check_launch("rotary_kernel");
}
