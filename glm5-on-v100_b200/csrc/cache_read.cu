// Reading the paged caches back, and moving rows inside them.
//
// 1. dsa_gather_cache: output row i belongs to the request b with
//    cu[b] <= i < cu[b+1] and holds position p = start[b] + i - cu[b], i.e.
//    cache row block_table[b, p / page] * page + p % page, dequantised:
//    value = e4m3(code) * f32 scale of its 128-wide group, one product in f32,
//    rounded once to the output type (the f16 rotary tail and 16-bit caches are
//    converted or copied).
//    Bound by HBM: a latent row is 656 B in, 1,152 B out. A block resolves 64
//    output rows (search in cu, block table) into shared memory, then its
//    threads take 8 output values each: 8 bytes in, 16 bytes out, both
//    contiguous over the warp, six loads in flight.
//    Measured: 131,072 latent rows to bf16 44 us of kernel, 47 a call = 5.0 TB/s (78%
//    of a plain copy's rate); 7 x 4099 ragged indexer rows 6 us, 16 a call.
// 2. dsa_commit_draft_rows: after a tree of drafts is verified, the k-th
//    accepted draft's row moves from position pre + accepted[b, k] to pre + k
//    in every cache of a list (one per layer), as raw bytes: nothing is
//    quantised again. A source may be another move's destination, so one block
//    holds all the rows of a request and cache in registers before it writes
//    any. Bound by latency: one launch for up to 128 caches, block = (request,
//    cache).
//    Measured: 8 requests x 48 caches 7 us of kernel, 43 a call (the checks and
//    the passing of 48 tensors); one cache 3 us, 15 a call.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace dsa {
namespace {

// Cache row of position p of request b, or -1 outside the table or the cache.
__device__ __forceinline__ int64_t cache_row(const int32_t* __restrict__ bt, int64_t bt_stride, int max_blocks,
                                             int page, int64_t n_rows, int b, int64_t p) {
  if (p < 0) return -1;
  const int64_t blk = p / page;
  if (blk >= max_blocks) return -1;
  const int64_t r = (int64_t)bt[(int64_t)b * bt_stride + blk] * page + (p - blk * page);
  return r >= 0 && r < n_rows ? r : -1;
}

// ------------------------------------------------------------------ gather
constexpr int kGatherRows = 64;
constexpr int kGatherThreads = 256;
constexpr int kGatherUnroll = 6;

struct GatherArgs {
  uint8_t* out;
  int64_t out_stride;  // elements
  int n_out;
  const uint8_t* cache;
  int64_t n_rows;
  int page, max_blocks;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* cu;
  const int32_t* starts;
  int B;
  int width;           // values per row
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) { return pack_half2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Four e4m3 codes times `scale` -> two packed words of T.
template <typename T>
__device__ __forceinline__ void dequant4(uint32_t codes, float scale, uint32_t& w0, uint32_t& w1) {
  __half2 lo, hi;
  e4m3x4_to_half2x2(codes, lo, hi);
  const float2 a = __half22float2(lo), b = __half22float2(hi);
  w0 = pack2<T>(__fmul_rn(a.x, scale), __fmul_rn(a.y, scale));
  w1 = pack2<T>(__fmul_rn(b.x, scale), __fmul_rn(b.y, scale));
}

// Eight 16-bit values of type S as T.
template <typename S, typename T>
__device__ __forceinline__ uint4 convert8(uint4 v) {
  if constexpr (sizeof(S) == sizeof(T) && std::is_same<S, T>::value) {
    return v;
  } else {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const S* s = reinterpret_cast<const S*>(&w[i]);
      w[i] = pack2<T>(to_f32(s[0]), to_f32(s[1]));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int FMT, typename T>
__global__ void __launch_bounds__(kGatherThreads) gather_cache_kernel(const GatherArgs a) {
  __shared__ int64_t rows[kGatherRows];  // cache row, -1: zeros, -2: not an output row of any request
  const int i0 = blockIdx.x * kGatherRows;
  if (threadIdx.x < kGatherRows) {
    const int i = i0 + threadIdx.x;
    int64_t r = -2;
    if (i < a.n_out && i >= a.cu[0] && i < a.cu[a.B]) {
      int lo = 0, hi = a.B;  // cu[lo] <= i < cu[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= i) lo = mid; else hi = mid;
      }
      const int64_t p = (int64_t)(a.starts ? a.starts[lo] : 0) + (i - a.cu[lo]);
      r = cache_row(a.bt, a.bt_stride, a.max_blocks, a.page, a.n_rows, lo, p);
    }
    rows[threadIdx.x] = r;
  }
  __syncthreads();
  const int chunks = FMT == DSA_FP8_DS_MLA ? 72 : FMT == DSA_FP8_IDXK ? 16 : a.width >> 3;
  const int n = min(kGatherRows, a.n_out - i0) * chunks;
  for (int base = threadIdx.x; base < n; base += kGatherThreads * kGatherUnroll) {
    uint4 v[kGatherUnroll];
    float sc[kGatherUnroll];
    int row[kGatherUnroll], ch[kGatherUnroll];
#pragma unroll
    for (int k = 0; k < kGatherUnroll; ++k) {
      const int j = base + k * kGatherThreads;
      row[k] = -1;
      v[k] = make_uint4(0, 0, 0, 0);
      sc[k] = 0.f;
      if (j >= n) continue;
      const int i = j / chunks, c = j - i * chunks;
      const int64_t r = rows[i];
      if (r == -2) continue;
      row[k] = i;
      ch[k] = c;
      if (r < 0) continue;
      if constexpr (FMT == DSA_FP8_DS_MLA) {
        const uint8_t* p = a.cache + r * 656;
        if (c < 64) {
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(p + 8 * c));
          v[k].x = w.x;
          v[k].y = w.y;
          sc[k] = __ldg(reinterpret_cast<const float*>(p + 512) + (c >> 4));
        } else {
          v[k] = __ldg(reinterpret_cast<const uint4*>(p + 528 + 16 * (c - 64)));
        }
      } else if constexpr (FMT == DSA_FP8_IDXK) {  // rows are only 4-byte aligned
        const uint8_t* p = a.cache + r * 132;
        v[k].x = __ldg(reinterpret_cast<const uint32_t*>(p + 8 * c));
        v[k].y = __ldg(reinterpret_cast<const uint32_t*>(p + 8 * c + 4));
        sc[k] = __ldg(reinterpret_cast<const float*>(p + 128));
      } else {
        v[k] = __ldg(reinterpret_cast<const uint4*>(a.cache + (r * a.width + 8 * c) * 2));
      }
    }
#pragma unroll
    for (int k = 0; k < kGatherUnroll; ++k) {
      if (row[k] < 0) continue;
      uint4 o;
      if constexpr (FMT == DSA_F16) {
        o = convert8<__half, T>(v[k]);
      } else if constexpr (FMT == DSA_BF16) {
        o = convert8<__nv_bfloat16, T>(v[k]);
      } else {
        if (FMT == DSA_FP8_IDXK || ch[k] < 64) {
          dequant4<T>(v[k].x, sc[k], o.x, o.y);
          dequant4<T>(v[k].y, sc[k], o.z, o.w);
        } else {
          o = convert8<__half, T>(v[k]);
        }
      }
      *reinterpret_cast<uint4*>(a.out + ((int64_t)(i0 + row[k]) * a.out_stride + 8 * ch[k]) * 2) = o;
    }
  }
}

template <int FMT>
void launch_gather(const GatherArgs& a, bool bf16, cudaStream_t s) {
  const unsigned grid = (unsigned)((a.n_out + kGatherRows - 1) / kGatherRows);
  if (bf16)
    gather_cache_kernel<FMT, __nv_bfloat16><<<grid, kGatherThreads, 0, s>>>(a);
  else
    gather_cache_kernel<FMT, __half><<<grid, kGatherThreads, 0, s>>>(a);
}

// ------------------------------------------------------------------ commit
constexpr int kMaxCaches = 128;   // pointers in one launch's parameters
constexpr int kMaxAccept = 64;
constexpr int kCommitThreads = 512;

struct CommitArgs {
  uint8_t* cache[kMaxCaches];
  int64_t n_rows;
  int page, max_blocks, row_bytes;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* seq_lens;
  const int32_t* draft_lens;
  int n_drafts;
  const int32_t* accepted;
  int64_t acc_stride;
  int n_accept;
};

// V: the word a row is moved in; K: words a thread holds.
template <typename V, int K>
__global__ void __launch_bounds__(kCommitThreads) commit_rows_kernel(const __grid_constant__ CommitArgs a) {
  __shared__ int64_t src[kMaxAccept], dst[kMaxAccept];
  __shared__ int n_moves;
  const int b = blockIdx.x;
  if (threadIdx.x == 0) n_moves = 0;
  __syncthreads();
  if (threadIdx.x < a.n_accept) {
    const int k = threadIdx.x;
    const int nd = a.draft_lens ? min(max(a.draft_lens[b], 0), a.n_drafts) : a.n_drafts;
    const int64_t pre = (int64_t)a.seq_lens[b] - nd;
    const int from = a.accepted[(int64_t)b * a.acc_stride + k];
    if (from >= 0 && from < nd && k < nd && from != k && pre >= 0) {
      const int64_t r = cache_row(a.bt, a.bt_stride, a.max_blocks, a.page, a.n_rows, b, pre + from);
      const int64_t w = cache_row(a.bt, a.bt_stride, a.max_blocks, a.page, a.n_rows, b, pre + k);
      if (r >= 0 && w >= 0) {
        const int m = atomicAdd(&n_moves, 1);  // order is of no account: all sources are read first
        src[m] = r;
        dst[m] = w;
      }
    }
  }
  __syncthreads();
  uint8_t* cache = a.cache[blockIdx.y];
  const int words = a.row_bytes / (int)sizeof(V);
  const int n = n_moves * words;
  V v[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int j = threadIdx.x + k * kCommitThreads;
    if (j < n) v[k] = *reinterpret_cast<const V*>(cache + src[j / words] * a.row_bytes + (j % words) * (int)sizeof(V));
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int j = threadIdx.x + k * kCommitThreads;
    if (j < n) *reinterpret_cast<V*>(cache + dst[j / words] * a.row_bytes + (j % words) * (int)sizeof(V)) = v[k];
  }
}

constexpr int kCommitWords16 = 9;  // 64 rows x 72 words of 16 bytes (1,152-byte rows) / 512 threads
constexpr int kCommitWords4 = 5;   // 64 rows x 33 words of 4 bytes (132-byte rows) / 512 threads

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_gather_cache(void* out, int out_dtype, int64_t out_stride, int n_out, const void* cache,
                                int cache_format, int64_t n_rows, int page_size, int width,
                                const int32_t* block_table, int64_t bt_stride, int max_blocks,
                                const int32_t* cu_seq_lens, const int32_t* seq_starts, int B, void* stream) {
  clear_error();
  DSA_REQUIRE(out_dtype == DSA_F16 || out_dtype == DSA_BF16, DSA_ERR_INVALID, "gather_cache: out must be f16 or bf16");
  DSA_REQUIRE(cache_format == DSA_F16 || cache_format == DSA_BF16 || cache_format == DSA_FP8_DS_MLA ||
                  cache_format == DSA_FP8_IDXK,
              DSA_ERR_INVALID, "gather_cache: cache must be f16, bf16, fp8_ds_mla or fp8 indexer-K");
  const int need = cache_format == DSA_FP8_DS_MLA ? 576 : cache_format == DSA_FP8_IDXK ? 128 : width;
  DSA_REQUIRE(width == need && width > 0 && width % 8 == 0, DSA_ERR_INVALID,
              "gather_cache: rows of this cache hold %d values (a multiple of 8; got width %d)", need, width);
  DSA_REQUIRE(n_out >= 0 && B >= 0 && n_rows >= 0 && page_size > 0 && max_blocks >= 0 &&
                  row_stride_ok(bt_stride, max_blocks) && out_stride >= width,
              DSA_ERR_INVALID, "gather_cache: bad sizes or strides");
  if (n_out == 0 || B == 0) return DSA_OK;
  DSA_REQUIRE(out && cu_seq_lens && (n_rows == 0 || cache) && (max_blocks == 0 || block_table), DSA_ERR_INVALID,
              "gather_cache: null pointer");
  DSA_REQUIRE(((uintptr_t)out & 15) == 0 && out_stride % 8 == 0 &&
                  ((uintptr_t)cache & (cache_format == DSA_FP8_IDXK ? 3 : 15)) == 0,
              DSA_ERR_INVALID, "gather_cache: out rows and cache must be 16-byte aligned (132-byte rows: 4)");
  GatherArgs a{reinterpret_cast<uint8_t*>(out), out_stride, n_out, reinterpret_cast<const uint8_t*>(cache), n_rows,
               page_size, max_blocks, block_table, bt_stride, cu_seq_lens, seq_starts, B, width};
  cudaStream_t s = as_stream(stream);
  const bool bf16 = out_dtype == DSA_BF16;
  switch (cache_format) {
    case DSA_FP8_DS_MLA: launch_gather<DSA_FP8_DS_MLA>(a, bf16, s); break;
    case DSA_FP8_IDXK: launch_gather<DSA_FP8_IDXK>(a, bf16, s); break;
    case DSA_F16: launch_gather<DSA_F16>(a, bf16, s); break;
    default: launch_gather<DSA_BF16>(a, bf16, s); break;
  }
  return check_launch("gather_cache_kernel");
}

extern "C" int dsa_commit_draft_rows(void* const* caches, int n_caches, int64_t n_rows, int page_size, int row_bytes,
                                     const int32_t* block_table, int64_t bt_stride, int max_blocks,
                                     const int32_t* seq_lens, const int32_t* draft_lens, int n_drafts,
                                     const int32_t* accepted, int64_t acc_stride, int n_accept, int B, void* stream) {
  clear_error();
  DSA_REQUIRE(n_caches >= 0 && B >= 0 && n_accept >= 0 && n_drafts >= 0 && n_rows >= 0 && page_size > 0 &&
                  max_blocks >= 0 && row_stride_ok(bt_stride, max_blocks) && row_stride_ok(acc_stride, n_accept),
              DSA_ERR_INVALID, "commit_draft_rows: bad sizes or strides");
  // requests whose drafts are the same rows would move them under one another
  DSA_REQUIRE(B <= 1 || max_blocks == 0 || bt_stride > 0, DSA_ERR_INVALID,
              "commit_draft_rows: each request needs its own row of the block table");
  DSA_REQUIRE(n_drafts <= kMaxAccept && n_accept <= kMaxAccept, DSA_ERR_UNSUPPORTED,
              "commit_draft_rows: at most 64 drafts (got %d, %d accepted)", n_drafts, n_accept);
  const bool wide = row_bytes % 16 == 0;
  DSA_REQUIRE(row_bytes > 0 && row_bytes % 4 == 0 && row_bytes <= (wide ? 1152 : 132), DSA_ERR_UNSUPPORTED,
              "commit_draft_rows: rows are at most 1152 bytes in multiples of 16, or 132 in multiples of 4 (got %d)",
              row_bytes);
  if (n_caches == 0 || B == 0 || n_accept == 0 || n_drafts == 0 || n_rows == 0 || max_blocks == 0) return DSA_OK;
  DSA_REQUIRE(caches && block_table && seq_lens && accepted, DSA_ERR_INVALID, "commit_draft_rows: null pointer");
  CommitArgs a{};
  a.n_rows = n_rows;
  a.page = page_size;
  a.max_blocks = max_blocks;
  a.row_bytes = row_bytes;
  a.bt = block_table;
  a.bt_stride = bt_stride;
  a.seq_lens = seq_lens;
  a.draft_lens = draft_lens;
  a.n_drafts = n_drafts;
  a.accepted = accepted;
  a.acc_stride = acc_stride;
  a.n_accept = n_accept;
  for (int i = 0; i < n_caches; ++i)
    DSA_REQUIRE(caches[i] && ((uintptr_t)caches[i] & (wide ? 15 : 3)) == 0, DSA_ERR_INVALID,
                "commit_draft_rows: cache %d is null or not aligned to its rows' words", i);
  for (int i0 = 0; i0 < n_caches; i0 += kMaxCaches) {
    const int n = std::min(kMaxCaches, n_caches - i0);
    for (int i = 0; i < n; ++i) a.cache[i] = reinterpret_cast<uint8_t*>(caches[i0 + i]);
    const dim3 grid((unsigned)B, (unsigned)n);
    if (wide)
      commit_rows_kernel<uint4, kCommitWords16><<<grid, kCommitThreads, 0, as_stream(stream)>>>(a);
    else
      commit_rows_kernel<uint32_t, kCommitWords4><<<grid, kCommitThreads, 0, as_stream(stream)>>>(a);
    const int st = check_launch("commit_rows_kernel");
    if (st != DSA_OK) return st;
  }
  return DSA_OK;
}
