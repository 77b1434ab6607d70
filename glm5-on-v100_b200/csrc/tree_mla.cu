// Attention of a tree of drafted tokens over the paged latent cache.
//
// Request b has s = seq_lens[b] positions, the last n = draft_lens[b] of them
// its drafts. Row (i, h), the query of draft i and head h, sees position p when
// p < s - n, or when bit p - (s - n) of tree_mask[b, i] is set:
//   z_p = scale * q[b,i,h,:576] . kv_p,  lse = log sum_p exp(z_p),
//   o = sum_p exp(z_p - lse) kv_p[:512];  nothing visible: o = 0, lse = -inf.
//
// One block: 16 rows of one request, keys in tiles of 16 held as f32 in shared
// memory, the softmax's running maximum and sum in f32.
#include "common.cuh"

namespace dsa {
namespace {

constexpr int TR = 16, TK = 16, DK = 576, DV = 512, NT = 256;

struct TreeArgs {
  const void* q;
  const uint8_t* kv;
  const int32_t* bt;
  const int32_t* seq_lens;
  const int32_t* draft_lens;
  const int64_t* mask;
  void* o;
  float* lse;
  int64_t n_kv_rows, bt_stride, mask_stride;
  int fmt, page, max_blocks, T, H, q_bf16, o_bf16;
  float scale_log2;
};

__device__ float kv_value(const TreeArgs& p, int64_t row, int d) {
  if (row < 0) return 0.f;
  if (p.fmt == DSA_FP8_DS_MLA) {
    const uint8_t* r = p.kv + row * 656;
    if (d >= 512) return __half2float(reinterpret_cast<const __half*>(r + 528)[d - 512]);
    const __half_raw h = __nv_cvt_fp8_to_halfraw(r[d], __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half*>(&h)) * reinterpret_cast<const float*>(r + 512)[d >> 7];
  }
  if (p.fmt == DSA_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.kv)[row * DK + d]);
  return __half2float(reinterpret_cast<const __half*>(p.kv)[row * DK + d]);
}

__global__ void __launch_bounds__(NT) tree_simple_kernel(const TreeArgs p) {
  extern __shared__ float sm[];
  float* q = sm;                 // [TR][DK]
  float* kv = q + TR * DK;       // [TK][DK]
  float* s = kv + TK * DK;       // [TR][TK]
  float* m = s + TR * TK;        // [TR]
  float* l = m + TR;
  float* al = l + TR;
  const int b = blockIdx.y, r0 = blockIdx.x * TR, R = p.T * p.H;
  const int nd = p.draft_lens ? min(max(p.draft_lens[b], 0), p.T) : p.T;
  const int seq = p.seq_lens[b], pre = seq - nd;
  for (int i = threadIdx.x; i < TR * DK; i += NT) {
    const int r = r0 + i / DK;
    float v = 0.f;
    if (r < R) {
      const int64_t at = ((int64_t)b * R + r) * DK + i % DK;
      v = p.q_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.q)[at])
                   : __half2float(reinterpret_cast<const __half*>(p.q)[at]);
    }
    q[i] = v;
  }
  if (threadIdx.x < TR) {
    m[threadIdx.x] = -INFINITY;
    l[threadIdx.x] = 0.f;
  }
  uint64_t seen = 0;  // draft columns that some row of the request sees: the others are not read
  for (int t = 0; t < nd; ++t) seen |= (uint64_t)p.mask[(int64_t)b * p.mask_stride + t];
  float acc[TR][2] = {};
  const int row = threadIdx.x / TK, key = threadIdx.x % TK;
  const int gr = r0 + row, i = gr / p.H;
  const uint64_t bits = (gr < R && i < nd) ? (uint64_t)p.mask[(int64_t)b * p.mask_stride + i] : 0;
  for (int k0 = 0; k0 < seq; k0 += TK) {
    __syncthreads();
    for (int e = threadIdx.x; e < TK * DK; e += NT) {
      const int pos = k0 + e / DK;
      int64_t phys = -1;
      if (pos < seq && pos / p.page < p.max_blocks && (pos < pre || ((seen >> (pos - pre)) & 1))) {
        phys = (int64_t)p.bt[(int64_t)b * p.bt_stride + pos / p.page] * p.page + pos % p.page;
        if (phys < 0 || phys >= p.n_kv_rows) phys = -1;
      }
      kv[e] = kv_value(p, phys, e % DK);
    }
    __syncthreads();
    float z = 0.f;
    for (int d = 0; d < DK; ++d) z += q[row * DK + d] * kv[key * DK + d];
    const int pos = k0 + key;
    const bool sees = gr < R && i < nd && pos < seq && (pos < pre || ((bits >> (pos - pre)) & 1));
    s[row * TK + key] = sees ? z * p.scale_log2 : -INFINITY;
    __syncthreads();
    if (threadIdx.x < TR) {
      float mx = m[threadIdx.x];
      for (int k = 0; k < TK; ++k) mx = fmaxf(mx, s[threadIdx.x * TK + k]);
      const float a = m[threadIdx.x] == -INFINITY ? 0.f : exp2f(m[threadIdx.x] - mx);
      float sum = l[threadIdx.x] * a;
      for (int k = 0; k < TK; ++k) {
        const float v = s[threadIdx.x * TK + k];
        const float e = v == -INFINITY ? 0.f : exp2f(v - mx);
        s[threadIdx.x * TK + k] = e;
        sum += e;
      }
      m[threadIdx.x] = mx;
      l[threadIdx.x] = sum;
      al[threadIdx.x] = a;
    }
    __syncthreads();
    for (int r = 0; r < TR; ++r)
      for (int c = 0; c < 2; ++c) {
        float v = acc[r][c] * al[r];
        for (int k = 0; k < TK; ++k) v += s[r * TK + k] * kv[k * DK + threadIdx.x + 256 * c];
        acc[r][c] = v;
      }
  }
  __syncthreads();
  for (int r = 0; r < TR && r0 + r < R; ++r) {
    const float inv = l[r] > 0.f ? 1.f / l[r] : 0.f;
    const int64_t at = ((int64_t)b * R + r0 + r);
    for (int c = 0; c < 2; ++c) {
      const int64_t e = at * DV + threadIdx.x + 256 * c;
      if (p.o_bf16)
        reinterpret_cast<__nv_bfloat16*>(p.o)[e] = __float2bfloat16_rn(acc[r][c] * inv);
      else
        reinterpret_cast<__half*>(p.o)[e] = __float2half_rn(acc[r][c] * inv);
    }
    if (threadIdx.x == 0) p.lse[at] = l[r] > 0.f ? (m[r] + log2f(l[r])) * 0.69314718055994530942f : -INFINITY;
  }
}

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" size_t dsa_tree_mla_decode_workspace_bytes(int B, int T, int n_head) { return 0; }

extern "C" int dsa_tree_mla_decode(void* o, int o_dtype, float* lse, const void* q, int q_dtype, const void* kv_cache,
                                   int kv_format, int64_t n_kv_rows, int page_size, const int32_t* block_table,
                                   int64_t bt_stride, int max_blocks, const int32_t* seq_lens,
                                   const int32_t* draft_lens, const int64_t* tree_mask, int64_t mask_stride, int B,
                                   int T, int n_head, double scale, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  clear_error();
  DSA_REQUIRE(B >= 0 && T >= 0 && n_head >= 0, DSA_ERR_INVALID, "tree_mla_decode: negative size (B=%d T=%d n_head=%d)",
              B, T, n_head);
  DSA_REQUIRE(T <= 64, DSA_ERR_UNSUPPORTED, "tree_mla_decode: at most 64 drafts a request (got %d)", T);
  DSA_REQUIRE(q_dtype == DSA_F16 || q_dtype == DSA_BF16, DSA_ERR_INVALID, "tree_mla_decode: q must be f16 or bf16");
  DSA_REQUIRE(o_dtype == DSA_F16 || o_dtype == DSA_BF16, DSA_ERR_INVALID, "tree_mla_decode: o must be f16 or bf16");
  DSA_REQUIRE(kv_format == DSA_F16 || kv_format == DSA_BF16 || kv_format == DSA_FP8_DS_MLA, DSA_ERR_INVALID,
              "tree_mla_decode: kv_cache must be f16, bf16 or fp8_ds_mla (u8 656)");
  DSA_REQUIRE(!(kv_format == DSA_BF16 && q_dtype == DSA_F16), DSA_ERR_UNSUPPORTED,
              "tree_mla_decode: a bf16 cache needs bf16 q");
  DSA_REQUIRE(page_size > 0 && max_blocks >= 0 && n_kv_rows >= 0 && n_kv_rows <= 0x7fffffff &&
                  bt_stride >= max_blocks && mask_stride >= T,
              DSA_ERR_INVALID, "tree_mla_decode: bad cache geometry or strides (page=%d max_blocks=%d rows=%lld)",
              page_size, max_blocks, (long long)n_kv_rows);
  if (B == 0 || T == 0 || n_head == 0) return DSA_OK;
  DSA_REQUIRE(n_head <= 1024 && B <= 65535, DSA_ERR_UNSUPPORTED, "tree_mla_decode: at most 65535 requests of 1024 heads");
  DSA_REQUIRE(o && lse && q && seq_lens && tree_mask && (n_kv_rows == 0 || kv_cache) && (max_blocks == 0 || block_table),
              DSA_ERR_INVALID, "tree_mla_decode: null pointer");
  DSA_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)kv_cache & 15) == 0 && ((uintptr_t)o & 15) == 0, DSA_ERR_INVALID,
              "tree_mla_decode: q, kv_cache and o must be 16-byte aligned");
  TreeArgs p{q, reinterpret_cast<const uint8_t*>(kv_cache), block_table, seq_lens, draft_lens, tree_mask, o, lse,
             n_kv_rows, bt_stride, mask_stride, kv_format, page_size, max_blocks, T, n_head, q_dtype == DSA_BF16,
             o_dtype == DSA_BF16, (float)(scale * 1.4426950408889634)};
  constexpr int kSmem = (TR * DK + TK * DK + TR * TK + 3 * TR) * 4;
  DSA_CUDA_TRY(cudaFuncSetAttribute(tree_simple_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem),
               "tree_mla_decode setup");
  tree_simple_kernel<<<dim3((T * n_head + TR - 1) / TR, B), NT, kSmem, as_stream(stream)>>>(p);
  return check_launch("tree_simple_kernel");
}
