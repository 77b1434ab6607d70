// Attention of a tree of drafted tokens over the paged latent cache, on the
// 5th-generation tensor cores (tcgen05 + TMEM, CTA pairs).
//
// Request b has s = seq_lens[b] positions, the last n = draft_lens[b] of them
// its drafts. Row (i, h), the query of draft i and head h, sees position p when
// p < s - n, or when bit p - (s - n) of tree_mask[b, i] is set:
//   z_p = scale * q[b,i,h,:576] . kv_p,  lse = log sum_p exp(z_p),
//   o = sum_p exp(z_p - lse) kv_p[:512];  nothing visible: o = 0, lse = -inf.
//
// All T * H rows of a request read the same keys, so rows are the M side: one
// cluster of two CTAs takes 128 consecutive rows (64 per CTA) and a run of
// 128-key tiles, one pass with a running maximum and sum. Per tile
//   S[128 x 128]  = Q[128 x 576] . K^T     each CTA holds 64 of the keys
//   O[128 x 512] += P[128 x 128] . V       each CTA holds 256 of the columns
// as cta_group::2 MMAs (M = 128, N = 128 and 2 x 256). Why pairs: an f32 state
// of 512 columns lets an SM hold 64 rows (half of TMEM, the other half S), and
// alone such an SM would read every key operand from its own shared memory for
// 64 rows only; in a pair each SM stores half of each operand and the hardware
// shares it.
//
// Work split: the (request, row tile, key tile) triples of a call form one
// list; pair p of P takes an equal run of it, whatever the lengths of the
// requests are. A run that holds all key tiles of a row tile writes o and lse;
// the first and last segments of a run may hold only some, and leave their
// unnormalised state in one of the pair's two workspace slots for the merge
// kernel, which is told where the runs start (no counters, nothing to reset, the
// same bits in every run).
//
// Roles (28 warps, 72 registers): the row warp walks the run, turns positions into
// cache rows, and has this CTA's 64 rows of an fp8 tile copied as they lie into one
// raw buffer (bulk copies; loads would go through the 28 KB that L1 has left),
// prefetched into L2 while the buffer is still in use (8 heads ragged 100 -> 96 us
// from memory; 1 - 2% slower where the cache lies in L2 already). Warps 0-15, four
// keys each, take the codes into registers, expand them and store K (keys x 576,
// K-major) and V (this CTA's 256 columns, MN-major): its own keys' from the same
// registers, the other CTA's by loads a tile ahead, which hit L2 (passing them
// between the CTAs' shared memory took 6600 cycles a tile). Two tail warps copy the
// rotary part. 16-bit rows go to K and V by cp.async. Warps 16-23 are the softmax,
// a thread a row and 32 keys (rows are TMEM lanes: no shuffles), read into
// registers once, so that S is free at once. One warp of CTA 0 issues the MMAs, in
// uniform control flow with one elected lane (80-130 cycles each otherwise, 45-64
// now). Q lies in tensor memory but for three of its nine 64-column blocks. QK(t+1)
// is issued before PV(t), so K(t+1) is stored under PV(t-1), V(t) under QK(t+1),
// and the softmax of t runs under PV(t-1). The roles meet at mbarriers and run on
// through the segments. Every wait is bounded.
//
// Arithmetic: f16 operands (bf16 for a bf16 cache), f32 sums, maximum and state. An
// fp8 value code * scale rounded once to f16 is off by up to half a step, 2^-11, which
// puts up to 2^-11 * scale * sum_d |q_d kv_d| on a score, 2e-4 for N(0, 1) rows and
// queries. Rows that weigh many keys average it (lse 1e-6 at 25,000 positions); where
// one key carries the row, lse and the weights keep it: with queries 4 times as large
// lse is off by 9e-4 (rms) and f16 o by 7e-4 of its norm at 32,769 positions, by 3e-5
// and 3e-4 at 32,768; bf16 o by 1.8e-3 and 1.7e-3. Beyond 32768 positions a score
// takes that one product all the same, because the second costs half as much
// again there (131,072 positions x 32 x 64: 584 us, 870 with two). Up to 32768 it takes
// two: the scale is cut into hi (7 bits: code * hi is exact in f16) and lo, and K is
// stored and multiplied with lo, then with hi, into the same S (the small products
// first: the sum keeps them): 2^-16 of a value, 2^-15 where scales are below 2^-8.
// Up to 1024 positions the second product is the rounding's own remainder, and V's is
// multiplied too (fewer keys average less). N(0, 1) rows, 8 heads x 16 drafts, 8
// requests of 13,824 to 24,576 positions: one product 74 us and lse within 1.1e-6, two
// 100 us and 1.5e-7; 64 heads x 8 drafts, 4 x 24,576: 133 us and 9.5e-7, 188 us and
// 1.7e-7. V's values are rounded to f16 once beyond 1024 positions (f16 o 14 - 45%
// farther from 64 bits than the plain form's), a bf16 cache's probabilities to bf16, as both
// operands of a product have one type (o 14 - 25% farther). bf16 q is shifted by a power of two
// per row into f16's range, which the row's scale undoes exactly.
// Probabilities are 2^(z - m) with m 7 below the running maximum, in log2 units, and
// m moves only when a score exceeds it by 15: P <= 2^15 uses f16's range at both ends,
// and O is rarely rescaled. Without the 7 the faint keys of a long context became zeros
// in P while the sum kept them: one key 17.5 nats above 131,071 others of value 1, its
// own 1/2, gave o = 0.4983 for 0.5016; 0.5005 now. What is left is the tensor cores'
// f32 accumulator, which cuts a product two bits below its own last place.
//
// Measured (times with the merge): 32 drafts x 64 heads over 131,072 positions, fp8
// 584 - 598 us = 1.0 PFLOP/s, 61% of the rate of a plain matrix product (686 in a
// long loop, whose clocks the power limit lowers), 16-bit cache 584 - 608 us. A tile
// takes a CTA 5000 cycles, the tensor cores 2700 of them: the bound is the
// producers' chain, K and V of a tile after one another, each store (8 x 8 codes a
// lane) 1300 cycles of issue and latency and 700 of waits and fences. With two
// products K is stored twice, 7800 cycles. The code of the loops counts: an SM's
// instruction cache misses go to a cache that several share, and took 76% of its
// rate before the loops were cut (23% now), so the usual path has no calls, the
// others (remainders, scales below 2^-10 or above 128) are rolled, and a wait is three
// instructions. A producer warp with one such scale among its tile's takes the rolled
// path. N(0, 1) rows have none; rows a tenth as large, or with one of the four groups so
// quiet, have them in every tile: 8 heads ragged 98 -> 182 us, 64 heads 189 -> 401,
// long context 598 -> 1450; with 1% of the rows all zero 130, 276 and 813.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <mutex>

#include "sparse_mla.cuh"
#include "tc_common.cuh"

namespace dsa {
namespace {

using namespace tc;

constexpr int kPairRows = 128;  // rows of a cluster
constexpr int kRows = 64;       // rows of a CTA
constexpr int kKeys = 128;      // keys of a tile
constexpr int DK = 576, DV = 512;
constexpr int kProducers = 16;  // warps 0-15
constexpr int kSoftmax0 = 16, kSoftmaxWarps = 8;
constexpr int kMmaWarp = 24, kRowWarp = 25;
constexpr int kTail0 = 26, kTailWarps = 2;  // fp8: the rotary part of K; 16-bit: L2 prefetch
constexpr int kRing = 3;        // 16-bit caches: tiles whose rows are known ahead
constexpr int kThreads = 28 * 32;
constexpr uint32_t kBlk = 64 * 128;    // 64 rows x 64 16-bit values: 8 KB
constexpr uint32_t kVBlk = 128 * 128;  // 128 keys x 64 columns: 16 KB
constexpr int kQtBlks = 6;             // 64-column blocks of Q in tensor memory; the other three in shared memory
constexpr uint32_t SM_Q = 0;
constexpr uint32_t SM_K = SM_Q + (9 - kQtBlks) * kBlk;
constexpr uint32_t SM_V = SM_K + 9 * kBlk;
constexpr uint32_t SM_P = SM_V + 4 * kVBlk;
constexpr uint32_t SM_RAW = SM_P + 2 * kBlk;       // fp8: this CTA's 64 cache rows as they lie in the cache
constexpr uint32_t SM_RING = SM_RAW + 64 * 656;    // 16-bit: rows[kRing][128]; fp8: rows[64] of the other CTA's keys
constexpr uint32_t SM_MISC = SM_RING + kRing * kKeys * 4;
constexpr int kSegs = 6;        // segment descriptors kept: the row warp is at most five tiles ahead of an epilogue
constexpr int kQeSegs = 3;      // Q is at most two segments ahead of the softmax
// the misc block: mbarriers | TMEM base, tiles of the run, valid rows | qe | row maxima / sums | segments
constexpr uint32_t kBarAt = 0, kWordsAt = 192, kQeAt = 224, kRowxAt = kQeAt + kQeSegs * 64, kSegAt = kRowxAt + 4 * 64 * 4;
constexpr uint32_t S_COL = 256, Q_COL = 320;  // O half h at [128h, +128), S at [256, +64), Q at [320, +192)
constexpr uint32_t TMEM_COLS = 512;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kNoMax = -1e30f;
constexpr int kMaxSeq = 0x7fffff00;   // tile ends stay in 32 bits
constexpr float kHead = 7.0f;          // log2 units: a new maximum's probability is 2^kHead
constexpr float kRescale = 15.0f;      // and none is above 2^kRescale, inside f16
constexpr int kTwoPassKeys = 32768;    // fp8: two products to a score up to here
constexpr int kFineKeys = 1024;        // and up to here the second is the rounding's remainder
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr int kSlotF = DV + 2;         // f32 of a row's partial state: o, then m and l

// Where a pair's run starts: key tile `tile` of `nt` in a row tile (0 also for an
// empty run); the other pairs' runs follow at distances of `chunk`.
struct Cut {
  int b, rt, tile, nt;
  int chunk, pad[3];
};

struct TreeArgs {
  const void* q;
  const uint8_t* kv;
  const int32_t* bt;
  const int32_t* seq_lens;
  const int32_t* draft_lens;
  const int64_t* mask;
  void* o;
  float* lse;
  float* part_o;   // [2 * pairs][512 / 4][slot_rows][4]
  float* part_ml;  // [2 * pairs][slot_rows][2]
  Cut* cuts;       // [pairs]
  int64_t n_kv_rows, bt_stride, mask_stride;
  int page, page_shift, max_blocks, B, T, H, pairs, slot_rows;  // page_shift < 0: no power of two
  int q_bf16, o_bf16;
  uint32_t q_sign;   // 0x80008000 for a negative scale
  float scale_log2;  // its magnitude
};

// Request b's size: key tiles and row tiles (0 tiles: nothing to do).
struct Req {
  int seq, nd, nt, nrt;
};
__device__ __forceinline__ Req load_req(const TreeArgs& p, int b) {
  Req r;
  r.seq = min(max(p.seq_lens[b], 0), kMaxSeq);
  r.nd = p.draft_lens ? min(max(p.draft_lens[b], 0), p.T) : p.T;
  r.nrt = (r.nd * p.H + kPairRows - 1) / kPairRows;
  r.nt = r.nd > 0 ? (int)(((int64_t)r.seq + kKeys - 1) / kKeys) : 0;
  return r;
}

// Sum of nt * nrt over requests [0, n), by one warp; every lane gets it.
__device__ __forceinline__ long long warp_work(const TreeArgs& p, int n, int lane) {
  long long w = 0;
  for (int b = lane; b < n; b += 32) {
    const Req r = load_req(p, b);
    w += (long long)r.nt * r.nrt;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
  return w;
}

__device__ __forceinline__ long long chunk_of(long long work, int pairs) { return (work + pairs - 1) / pairs; }

// A run of key tiles of one row tile, as the row warp hands it to the others.
struct Segment {
  int b, rt;
  int n;      // key tiles
  int pre;    // context positions less those before the first tile
  int nd;     // drafts of the request
  int flags;  // kTwo: two-pass products, kFine: of the rounding's remainder | kFull: every key tile of the row tile
};
enum { kTwo = 1, kFull = 2, kFine = 4 };
constexpr uint32_t SMEM_BYTES = SM_MISC + kSegAt + kSegs * (uint32_t)sizeof(Segment);
static_assert(SMEM_BYTES <= 232448, "shared memory budget");

// One pair's walk over its run of tiles.
struct Cursor {
  int chunk;       // tiles of a full run
  int left;        // tiles left, this one included
  int b, rt, tile;
  bool first;      // first tile of a segment
  Req r;
  __device__ __forceinline__ void next(const TreeArgs& p) {
    first = false;
    ++tile;
    if (--left == 0) return;
    if (tile == r.nt) {
      tile = 0;
      first = true;
      if (++rt == r.nrt) {
        rt = 0;
        do r = load_req(p, ++b);
        while (r.nt == 0 || r.nrt == 0);
      }
    }
  }
};

// The segment that starts at c.
template <bool FP8>
__device__ __forceinline__ Segment segment_of(const Cursor& c) {
  Segment sg;
  sg.b = c.b;
  sg.rt = c.rt;
  sg.n = min(c.r.nt - c.tile, c.left);
  sg.pre = c.r.seq - c.r.nd - c.tile * kKeys;
  sg.nd = c.r.nd;
  sg.flags = (FP8 && c.r.seq <= kTwoPassKeys ? kTwo : 0) | (FP8 && c.r.seq <= kFineKeys ? kFine : 0) | (sg.n == c.r.nt ? kFull : 0);
  return sg;
}

// The start of a pair's run, by one warp.
__device__ __forceinline__ Cursor find_run(const TreeArgs& p, int pair, int lane) {
  const long long work = warp_work(p, p.B, lane);
  const long long chunk = chunk_of(work, p.pairs);
  const long long w0 = chunk * pair;
  Cursor c{};
  c.chunk = (int)min(chunk, 0x7fffffffll);
  c.left = (int)max(min(chunk, work - w0), 0ll);
  c.first = true;
  if (c.left == 0) return c;
  long long before = 0;
  for (int b0 = 0;; b0 += 32) {
    Req r{0, 0, 0, 0};
    if (b0 + lane < p.B) r = load_req(p, b0 + lane);
    const long long mine = (long long)r.nt * r.nrt;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + incl > w0);
    if (hit) {
      const int src = __ffs(hit) - 1;
      c.b = b0 + src;
      c.r = load_req(p, c.b);
      const long long at = w0 - (before + __shfl_sync(0xffffffffu, incl - mine, src));
      c.rt = (int)(at / c.r.nt);
      c.tile = (int)(at % c.r.nt);
      return c;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
}

// A value that a warp's lanes have in common, in a register of the warp: where branches
// are known to be uniform, warp-wide instructions need no code to gather their lanes.
__device__ __forceinline__ int uniform(uint32_t x) { return (int)__reduce_or_sync(0xffffffffu, x); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two f32 lanes per instruction, and a maximum of three (sm_100).
__device__ __forceinline__ uint64_t pack64(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack64(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// How codes are expanded to f16: the product code * scale rounded once, by f16
// arithmetic where the scale's parts and the products stay in f16's range (groups whose
// largest value lies between 0.44 and 57344), by f32 elsewhere: twice the time, figures
// above.
__device__ __forceinline__ bool fast_scale(float sc) { return sc >= 0x1p-10f && sc <= 128.0f; }

// A scale cut in two f16 parts, hi (low half word) with 7 significant bits and lo the
// rest: a code (4 bits) times hi is exact in f16's 11 bits, so fma(code, lo, code *
// hi) rounds the whole product once (lo keeps the scale to 2^-15 of it or better).
__device__ __forceinline__ uint32_t cut_scale(float sc) {
  const float h = __uint_as_float(__float_as_uint(sc) & 0xFFFE0000u);
  return pack_half2(h, sc - h);
}

// Eight codes -> eight f16 values.
__device__ __forceinline__ uint4 dequant8(uint2 v, uint32_t cut) {
  const __half2 c = *reinterpret_cast<const __half2*>(&cut);
  const __half2 hi = __low2half2(c), lo = __high2half2(c);
  __half2 x[4];
  e4m3x4_to_half2x2(v.x, x[0], x[1]);
  e4m3x4_to_half2x2(v.y, x[2], x[3]);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = __hfma2(x[e], lo, __hmul2(x[e], hi));
  return *reinterpret_cast<const uint4*>(x);
}

// With one of the two parts, as f16 (hi: exact). lo has at most 2^-6 of the scale, so as
// f16 it keeps the scale to 2^-18, and its product with a code is rounded by 2^-17 of
// the value; a lo below 2^-14 (scales below 2^-7) is off by up to 2^-25, which is 2^-17
// of a scale of 2^-8 and 2^-15 of the smallest, 2^-10, alike for the group's 128 values.
__device__ __forceinline__ uint4 dequant8_part(uint2 v, __half part) {
  __half2 x[4];
  e4m3x4_to_half2x2(v.x, x[0], x[1]);
  e4m3x4_to_half2x2(v.y, x[2], x[3]);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = __hmul2(x[e], __half2half2(part));
  return *reinterpret_cast<const uint4*>(x);
}

// The scale's part after hi times 256, itself cut in two: 29 bits of the scale in all.
__device__ __forceinline__ uint32_t cut_rest(float sc) {
  const float lo = (sc - __uint_as_float(__float_as_uint(sc) & 0xFFFE0000u)) * 256.f;
  const __half h = __float2half_rn(lo);
  return pack_half2(__half2float(h), lo - __half2float(h));
}

// What dequant8's rounding left, itself rounded. Its value y lies so near code * hi
// that the difference is exact; the small parts take code / 256.
__device__ __forceinline__ uint4 rest8(uint2 v, uint32_t cut, uint32_t small) {
  const __half2 c = *reinterpret_cast<const __half2*>(&cut), d = *reinterpret_cast<const __half2*>(&small);
  const __half2 hi = __low2half2(c), lo = __high2half2(c), lo1 = __low2half2(d), lo2 = __high2half2(d);
  __half2 x[4];
  e4m3x4_to_half2x2(v.x, x[0], x[1]);
  e4m3x4_to_half2x2(v.y, x[2], x[3]);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const __half2 y = __hfma2(x[e], lo, __hmul2(x[e], hi));
    const __half2 z = __hmul2(x[e], __float2half2_rn(0x1p-8f));
    x[e] = __hfma2(z, lo2, __hfma2(z, lo1, __hfma2(x[e], hi, __hneg2(y))));
  }
  return *reinterpret_cast<const uint4*>(x);
}

// The same for any scale, or with `rest` what that rounding left, itself rounded.
// Kept out of the loops' code, which has to fit the instruction cache.
__device__ __noinline__ uint4 dequant8_any(uint2 v, float sc, bool rest, bool fast) {
  if (fast) return rest8(v, cut_scale(sc), cut_rest(sc));
  __half2 x[4];
  e4m3x4_to_half2x2(v.x, x[0], x[1]);
  e4m3x4_to_half2x2(v.y, x[2], x[3]);
  uint32_t q[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(x[e]);
    q[e] = pack_half2(f.x * sc, f.y * sc);
    if (rest) {
      const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&q[e]));
      q[e] = pack_half2(fmaf(f.x, sc, -y.x), fmaf(f.y, sc, -y.y));
    }
  }
  return make_uint4(q[0], q[1], q[2], q[3]);
}

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

__device__ __forceinline__ float lds4(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

__device__ __forceinline__ uint2 lds8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

__device__ __forceinline__ uint2 ldg_nc8_or_zero(const void* p, bool on) {
  uint2 v;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %3, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\t"
      "@q ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];\n\t}"
      : "=&r"(v.x), "=&r"(v.y)
      : "l"(p), "r"((uint32_t)on));
  return v;
}

// Bytes of global memory (both 16-byte aligned, a multiple of 16) into this CTA's shared memory.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t mbar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(mbar)
               : "memory");
}

__device__ __forceinline__ void sts16(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

__device__ __forceinline__ void cp_async16_zfill(uint32_t saddr, const void* gptr, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(saddr), "l"(gptr), "r"(on ? 16 : 0));
}

// Draft columns of request b that some draft sees (the others are not read).
__device__ __forceinline__ uint64_t seen_columns(const TreeArgs& p, int b, int nd, int lane) {
  uint64_t m = 0;
  for (int i = lane; i < nd; i += 32) m |= (uint64_t)p.mask[(int64_t)b * p.mask_stride + i];
  const uint32_t lo = __reduce_or_sync(0xffffffffu, (uint32_t)m);
  const uint32_t hi = __reduce_or_sync(0xffffffffu, (uint32_t)(m >> 32));
  return ((uint64_t)hi << 32) | lo;
}

// Cache rows of positions pos0 + 32k + lane, k < 4, or -1 (reads as zeros); the
// block-table loads are in flight together.
__device__ __forceinline__ void row_codes(const TreeArgs& p, int b, const Req& r, uint64_t seen, int pos0, int lane,
                                          int (&code)[4]) {
  const int32_t* bt = p.bt + (int64_t)b * p.bt_stride;
  int blk[4], page_row[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int pos = pos0 + 32 * k + lane;
    blk[k] = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page;
    page_row[k] = p.max_blocks > 0 ? __ldg(bt + min(blk[k], p.max_blocks - 1)) : -1;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int pos = pos0 + 32 * k + lane;
    const int j = pos - (r.seq - r.nd);
    const int64_t row = (int64_t)page_row[k] * p.page + (pos - blk[k] * p.page);
    const bool on = pos < r.seq && (j < 0 || ((seen >> j) & 1)) && blk[k] < p.max_blocks && row >= 0 && row < p.n_kv_rows;
    code[k] = on ? (int)row : -1;
  }
}

__device__ __forceinline__ void prefetch_line(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// This CTA's 64 query rows (f16, or bf16 as it is), by the producer warps: the last
// three 64-column blocks into shared memory, the others by way of the K buffer,
// which is free then, into tensor memory (twice, for its two lane halves). Warp w
// loads rows 4w + lane / 8, eight lanes a row. qe[row]: the power of two that a
// bf16 row was divided by.
constexpr int kQLoads = 3;  // loads in flight, of 9
template <int FMT>
__device__ __forceinline__ void load_q(const TreeArgs& p, uint32_t base, uint32_t tmem, int8_t* qe, int b, int row0, int w,
                                       int lane) {
  const int row = 4 * w + (lane >> 3), l8 = lane & 7;
  const bool on = row0 + row < p.T * p.H;
  const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(p.q) +
                                                    ((int64_t)b * p.T * p.H + row0 + row) * DK * 2);
  auto at = [&](int c) {
    return base + (c < kQtBlks ? SM_K + c * kBlk : SM_Q + (c - kQtBlks) * kBlk) + sw128_off(row, l8);
  };
  if (on) {  // the row's nine lines come from memory together
    prefetch_line(src + 8 * l8);
    if (l8 == 0) prefetch_line(src + 64);
  }
  const bool scaled = FMT != DSA_BF16 && p.q_bf16;
  uint32_t bits = 0;
#pragma unroll 1
  for (int c0 = 0; c0 < 9; c0 += kQLoads) {
    uint4 v[kQLoads];
#pragma unroll
    for (int k = 0; k < kQLoads; ++k)
      v[k] = on && c0 + k < 9 ? __ldg(src + l8 + 8 * (c0 + k)) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < kQLoads; ++k) {
      if (scaled) bits = max(bits, bf16x8_max_abs_bits(v[k]));
      v[k] = make_uint4(v[k].x ^ p.q_sign, v[k].y ^ p.q_sign, v[k].z ^ p.q_sign, v[k].w ^ p.q_sign);
      if (c0 + k < 9) sts16(at(c0 + k), v[k]);
    }
  }
  int e = 0;
  if (scaled) {
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 2));
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 4));
    e = bf16_fp16_shift(bits);
#pragma unroll 3
    for (int c = 0; c < 9; ++c) sts16(at(c), bf16x8_to_half8_scaled(lds16(at(c)), e));
  }
  if (l8 == 0) qe[row] = (int8_t)e;
  named_bar(2, kProducers * 32);
  // four warps a sub-partition: blocks w / 4 and w / 4 + 4
  const int sp = w & 3, trow = (32 * sp + lane) & 63;
#pragma unroll 1
  for (int c = 2 * (w >> 2); c < 2 * kQtBlks; c += (c & 1) ? 7 : 1) {  // half blocks: 32 columns of Q
    uint32_t r[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint4 v = lds16(base + SM_K + (c >> 1) * kBlk + sw128_off(trow, 4 * (c & 1) + k));
      r[4 * k] = v.x;
      r[4 * k + 1] = v.y;
      r[4 * k + 2] = v.z;
      r[4 * k + 3] = v.w;
    }
    tmem_st16(tmem + ((uint32_t)(32 * sp) << 16) + Q_COL + 16 * c, r);
  }
  tmem_wait_st();
  named_bar(2, kProducers * 32);  // the K buffer has been read
}

// FMT: the cache's format.
template <int FMT>
__global__ void __launch_bounds__(kThreads, 1) tree_mla_kernel(const TreeArgs p, int32_t* err) {
  constexpr bool kFp8 = FMT == DSA_FP8_DS_MLA;
  constexpr bool kBf16 = FMT == DSA_BF16;
  constexpr int kRowBytes = kFp8 ? 656 : 2 * DK;
  constexpr uint32_t IDESC_QK = idesc_f16(kPairRows, kKeys, false, false, kBf16);
  constexpr uint32_t IDESC_PV = idesc_f16(kPairRows, 256, false, true, kBf16);
  extern __shared__ __align__(1024) uint8_t sm[];  // 1024: the swizzle atoms' alignment
  const uint32_t base = smem_u32(sm);
  if (base & 1023u) {  // never, with no static shared memory in this kernel
    if (threadIdx.x == 0) atomicExch(err, (int32_t)DSA_ERR_CUDA);
    return;
  }
  uint8_t* misc = sm + SM_MISC;
  const uint32_t mb = smem_u32(misc) + kBarAt;
  const uint32_t mb_k_full = mb, mb_k_free = mb + 8, mb_v_full = mb + 16, mb_v_free = mb + 24, mb_p_full = mb + 32,
                 mb_o_free = mb + 40, mb_done = mb + 48, mb_s_full = mb + 56, mb_s_free = mb + 64,
                 mb_q_full = mb + 72 /* [3] */, mb_r_full = mb + 96 /* [3] */, mb_r_free = mb + 120 /* [3] */,
                 mb_raw_full = mb + 144, mb_raw_free = mb + 152, mb_pv = mb + 160;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + kWordsAt);
  int* run_tiles = reinterpret_cast<int*>(misc + kWordsAt + 8);
  uint32_t* raw_valid = reinterpret_cast<uint32_t*>(misc + kWordsAt + 16);  // [2]: rows that lie in the raw buffer
  int8_t* qe = reinterpret_cast<int8_t*>(misc + kQeAt);         // [kQeSegs][64]
  float* rowx = reinterpret_cast<float*>(misc + kRowxAt);       // [4][64]
  int* ring = reinterpret_cast<int*>(sm + SM_RING);             // [kRing][128]
  Segment* segs = reinterpret_cast<Segment*>(misc + kSegAt);    // [kSegs]

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rank = uniform(cluster_rank());
  const int pair = blockIdx.x >> 1;

  Cursor c{};  // the row warp's
  if (warp == 0) {
    if (lane == 0) {
      mbar_init(mb_k_full, 2 * (kProducers + (kFp8 ? kTailWarps : 0)));
      mbar_init(mb_k_free, 1);
      mbar_init(mb_v_full, 2 * kProducers);
      mbar_init(mb_v_free, 1);
      mbar_init(mb_p_full, 2 * kSoftmaxWarps);
      mbar_init(mb_o_free, 2 * kSoftmaxWarps);
      mbar_init(mb_done, 1);
      mbar_init(mb_s_full, 1);
      mbar_init(mb_s_free, 2 * kSoftmaxWarps);
      for (int x = 0; x < kQeSegs; ++x) mbar_init(mb_q_full + 8 * x, kProducers);
      for (int x = 0; x < kRing; ++x) {
        mbar_init(mb_r_full + 8 * x, 1);
        mbar_init(mb_r_free + 8 * x, kProducers + (kFp8 ? 0 : kTailWarps));
      }
      mbar_init(mb_pv, 1);
      mbar_init(mb_raw_full, 1);
      mbar_init(mb_raw_free, kProducers + kTailWarps);
      mbar_init_fence();
    }
    __syncwarp();
    tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLS);
  } else if (warp == kRowWarp) {
    for (int i = lane; i < kRing * kKeys; i += 32) ring[i] = -1;
    for (int i = lane; i < kSegs * (int)(sizeof(Segment) / 4); i += 32) reinterpret_cast<int*>(segs)[i] = 0;
    __syncwarp();
    c = find_run(p, pair, lane);
    if (lane == 0) {
      *run_tiles = c.left;
      if (c.left > 0) segs[0] = segment_of<kFp8>(c);
      if (rank == 0) p.cuts[pair] = Cut{c.b, c.rt, c.tile, c.r.nt, c.chunk, {0, 0, 0}};
    }
  }
  fence_before_sync();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist and TMEM is allocated
  fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const int total = uniform(*run_tiles);

  // After a wait that ran out, `more` is 0: its thread's later waits return after one
  // try, and it goes on through its role's barriers and arrivals with whatever is
  // there. That is safe: rows in the ring and segment descriptors are valid from
  // the start, and what a segment's loops go by is read only while no thread of the
  // role has failed. The MMA and row warps stop instead (`ok`, uniform).
  uint32_t more = 1u << 20;
  auto wait = [&](uint32_t mbar, uint32_t parity) { mbar_wait_sticky(mbar, parity, more); };
  auto wait_ok = [&](uint32_t mbar, uint32_t parity) {
    mbar_wait_sticky(mbar, parity, more);
    return __all_sync(0xffffffffu, more != 0);
  };
  if (warp < kProducers) {
    // ------------------------------------------------------------- producers
    // K(t+1) is stored under PV(t-1), V(t) under QK(t+1); with two passes the first
    // of K(t+1) under QK(t), the second under PV(t).
    const int w = warp;
    const uint32_t k_full0 = cluster_map(mb_k_full, 0), v_full0 = cluster_map(mb_v_full, 0);
    int seg = 0, left = 0;  // the segment of the next K store, and its tiles left
    // The flags of the next K's segment, those of the next V's three bits up, and the
    // parities of the number of K and of V stores so far. A wait for the buffer's next
    // release goes by the parity's complement: at once before the first.
    constexpr int kVShift = 3, kKOdd = 64, kVOdd = 128;
    int st = 0;
    auto wait_k = [&]() { wait(mb_k_free, st & kKOdd ? 0 : 1); };
    auto wait_v = [&]() { wait(mb_v_free, st & kVOdd ? 0 : 1); };
    // the next segment's Q, through the K buffer
    auto enter = [&]() {
      const Segment& sg = segs[seg % kSegs];  // visible: the wait for this tile's rows
      const bool live = !named_bar_or(2, kProducers * 32, more == 0);  // all take the same number of barriers
      left = live ? uniform(sg.n) : 1 << 30;
      st = (st & ~(kTwo | kFine | kFull)) | (live ? uniform(sg.flags) : 0);
      if (live)
        load_q<FMT>(p, base, tmem, qe + 64 * (seg % kQeSegs), sg.b, sg.rt * kPairRows + kRows * rank, w, lane);
      more = live ? more : 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(mb_q_full + 8 * (seg % kQeSegs));
      ++seg;
    };
    if constexpr (kFp8) {
      // This CTA's 64 keys land in shared memory as they lie in the cache, by bulk
      // copies: loads would go through an L1 of 28 KB, whose lines they fill faster
      // than they arrive. Rows 4w + x are this warp's. A lane takes 8 codes of each
      // half row, which is one 16-byte chunk of f16, so a store writes whole 128-byte
      // rows of four 64-column blocks. In registers the codes serve K and, the half that
      // is this CTA's columns, V a tile later; V of the other CTA's keys is loaded a
      // tile ahead.
      uint2 kd[4][2], vd[4], pd[4];  // K: [row][half] | V: own rows | the other CTA's rows
      // their scales: lane 4x + g < 16 holds row x, group g; of the other CTA's rows
      // lane 2x + g < 8, of this CTA's columns
      float ks = 1.f, vs = 1.f, ps = 1.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) kd[x][0] = kd[x][1] = vd[x] = pd[x] = make_uint2(0, 0);
      int4 oc = make_int4(-1, -1, -1, -1);  // the other CTA's rows of the tile last stored as K
      int os = -1;
      auto load_others = [&]() {
        const uint8_t* at = p.kv + 256 * rank + 8 * lane;
        const int code[4] = {oc.x, oc.y, oc.z, oc.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) pd[x] = ldg_nc8_or_zero(at + (int64_t)code[x] * kRowBytes, code[x] >= 0);
        ps = 1.f;
        if (lane < 8 && os >= 0)
          ps = __ldg(reinterpret_cast<const float*>(p.kv + (int64_t)os * kRowBytes + 512) + 2 * rank + (lane & 1));
      };
      // chunk lane & 7 of block lane / 8, row 4w: row x further on moves the swizzle by x
      const uint32_t k_at = base + SM_K + (lane >> 3) * kBlk + sw128_off(4 * w, lane & 7);
      const uint32_t v_at = base + SM_V + (lane >> 3) * kVBlk + sw128_off(4 * w, lane & 7);
      // The loops below for any scales are rolled, with row 0's registers taken and the
      // others moved down, so that they cost little code.
      auto put_v = [&](bool rest) {
        const bool fast = __all_sync(0xffffffffu, fast_scale(vs) && fast_scale(ps));
        if (fast && !rest) {
          const uint32_t vcut = cut_scale(vs), pcut = cut_scale(ps);
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t at = (v_at ^ (16 * x)) + 128 * x;
            const uint32_t s0 = __shfl_sync(0xffffffffu, vcut, 4 * x + 2 * rank + (lane >> 4));
            const uint32_t s1 = __shfl_sync(0xffffffffu, pcut, 2 * x + (lane >> 4));
            sts16(at + 8192 * rank, dequant8(vd[x], s0));
            sts16(at + 8192 * (rank ^ 1), dequant8(pd[x], s1));
          }
          return;
        }
#pragma unroll 1
        for (int x = 0; x < 8; ++x) {  // own rows, then the other CTA's
          const bool own = x < 4;
          const float sc = __shfl_sync(0xffffffffu, own ? vs : ps, (own ? 4 * x + 2 * rank : 2 * (x - 4)) + (lane >> 4));
          const uint4 v = dequant8_any(vd[0], sc, rest, fast);
          sts16((v_at ^ (16 * (x & 3))) + 128 * (x & 3) + 8192 * (own ? rank : rank ^ 1), v);
          const uint2 first = vd[0];
          vd[0] = vd[1], vd[1] = vd[2], vd[2] = vd[3], vd[3] = pd[0];
          pd[0] = pd[1], pd[1] = pd[2], pd[2] = pd[3], pd[3] = first;
        }
      };
      auto take = [&](int t) {
        wait(mb_raw_full, t & 1);
        const uint32_t valid = raw_valid[w >> 3] >> (4 * w & 31);
        const uint32_t raw = base + SM_RAW + 4 * w * 656;
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int h = 0; h < 2; ++h) kd[x][h] = lds8(raw + 656 * x + 256 * h + 8 * lane);
        ks = lds4(raw + 656 * ((lane >> 2) & 3) + 512 + 4 * (lane & 3));
        oc = *reinterpret_cast<const int4*>(ring + 4 * w);
        os = ring[4 * w + ((lane >> 1) & 3)];
        if ((valid & 15u) != 15u) {  // the others read as zeros
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (!((valid >> x) & 1)) kd[x][0] = kd[x][1] = make_uint2(0, 0);
          if (!((valid >> ((lane >> 2) & 3)) & 1)) ks = 1.f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(mb_raw_free);
      };
      // `rest`: what rounding takes away
      auto put_k = [&](bool rest) {
        const bool fast = __all_sync(0xffffffffu, fast_scale(ks));
        const uint32_t cut = cut_scale(ks);
        if (fast && (!(st & kTwo) || (!rest && (st & kFine)))) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              sts16((k_at ^ (16 * x)) + 128 * x + 4 * kBlk * h,
                    dequant8(kd[x][h], __shfl_sync(0xffffffffu, cut, 4 * x + 2 * h + (lane >> 4))));
          return;
        }
        if (fast && !(st & kFine)) {
          const uint32_t part = rest ? cut >> 16 : cut;
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              sts16((k_at ^ (16 * x)) + 128 * x + 4 * kBlk * h,
                    dequant8_part(kd[x][h], __ushort_as_half((unsigned short)__shfl_sync(
                                                0xffffffffu, part, 4 * x + 2 * h + (lane >> 4)))));
          return;
        }
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
          const int x = i >> 1, h = i & 1;
          const float sc = __shfl_sync(0xffffffffu, ks, 4 * x + 2 * h + (lane >> 4));
          const uint4 v = dequant8_any(kd[0][0], sc, rest, fast);
          sts16((k_at ^ (16 * x)) + 128 * x + 4 * kBlk * h, v);
          const uint2 first = kd[0][0];
          kd[0][0] = kd[0][1], kd[0][1] = kd[1][0], kd[1][0] = kd[1][1], kd[1][1] = kd[2][0];
          kd[2][0] = kd[2][1], kd[2][1] = kd[3][0], kd[3][0] = kd[3][1], kd[3][1] = first;
        }
      };
      auto begin_k = [&](int t) {
        if (left <= 0) {
          if (t > 0) {
            wait(mb_raw_full, t & 1);  // the segment's descriptor is visible
            wait_k();
          }
          enter();
        }
        take(t);
        --left;
      };
#pragma unroll 1
      for (int t = 0; t <= total; ++t) {
        if (t < total) begin_k(t);
        // K of tile t, or first what rounding takes from it; V of tile t - 1; then K
#pragma unroll 1
        for (int s = 0; s < 2; ++s) {
          if (t < total && (s == 0 || (st & kTwo))) {
            wait_k();
            put_k(s == 0 && (st & kTwo));
            fence_proxy_async();
            fence_before_sync();  // Q's tensor-memory stores
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(k_full0);
            st ^= kKOdd;
          }
          if (s == 0 && t > 0) {
#pragma unroll 1
            for (int x = st & (kFine << kVShift) ? 0 : 1; x < 2; ++x) {
              wait_v();
              put_v(x == 0);
              fence_proxy_async();
              __syncwarp();
              if (lane == 0) mbar_arrive_cluster(v_full0);
              st ^= kVOdd;
            }
          }
        }
        if (t < total) {
#pragma unroll
          for (int x = 0; x < 4; ++x) vd[x] = rank ? kd[x][1] : kd[x][0];
          vs = ks;
          st = (st & ~(7 << kVShift)) | (st & 7) << kVShift;
          load_others();
        }
      }
    } else {
      const int r4 = lane >> 3, l8 = lane & 7;  // eight lanes a row, 16 bytes each
      auto rows_of = [&](int t) { return ring + (t % kRing) * kKeys; };
      auto free_rows = [&](int t) {
        __syncwarp();
        if (lane == 0) mbar_arrive(mb_r_free + 8 * (t % kRing));
      };
      auto store_k = [&](int t) {
        if (left <= 0 && t == 0) enter();
        wait(mb_r_full + 8 * (t % kRing), (t / kRing) & 1);
        const int code = rows_of(t)[64 * rank + 4 * w + r4];
        wait_k();
        if (left <= 0) enter();
        {
          const uint8_t* row = p.kv + (int64_t)max(code, 0) * kRowBytes + 16 * l8;
#pragma unroll
          for (int x = 0; x < 9; ++x)
            cp_async16_zfill(base + SM_K + x * kBlk + sw128_off(4 * w + r4, l8), row + 128 * x, code >= 0);
        }
        cp_async_commit();
        cp_async_wait<0>();
        fence_proxy_async();
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(k_full0);
        st ^= kKOdd;
        --left;
      };
#pragma unroll 1
      for (int t = -1; t < total; ++t) {
        if (t + 1 < total) store_k(t + 1);
        if (t < 0) continue;
        int code[2];
        code[0] = rows_of(t)[8 * w + r4];
        code[1] = rows_of(t)[8 * w + r4 + 4];
        free_rows(t);
        if (t > 0) wait(mb_v_free, (t - 1) & 1);
        {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint8_t* row = p.kv + (int64_t)max(code[i], 0) * kRowBytes + 512 * rank + 16 * l8;
#pragma unroll
            for (int x = 0; x < 4; ++x)
              cp_async16_zfill(base + SM_V + x * kVBlk + sw128_off(8 * w + 4 * i + r4, l8), row + 128 * x, code[i] >= 0);
          }
        }
        cp_async_commit();
        cp_async_wait<0>();
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(v_full0);
      }
    }
  } else if (warp == kRowWarp) {
    // ------------------------------------------------------ rows of the tiles
    // Block table -> cache rows. 16-bit: into the ring, kRing tiles ahead. fp8: this
    // CTA's keys are copied into the raw buffer as soon as the tile before has been
    // read, with the rows of the other CTA's keys beside it.
    uint64_t seen = 0;
    int seg = 0, t = 0;
    bool ok = true;
#pragma unroll 1
    for (; t < total; ++t) {
      if (c.first) seen = seen_columns(p, c.b, c.r.nd, lane);
      int code[4];
      row_codes(p, c.b, c.r, seen, c.tile * kKeys, lane, code);
      int mine[2];
      bool run[2];  // 32 neighbouring rows are one copy
      uint32_t valid[2];
      if constexpr (kFp8) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          mine[k] = rank ? code[2 + k] : code[k];
          valid[k] = __ballot_sync(0xffffffffu, mine[k] >= 0);
          const int head = __shfl_sync(0xffffffffu, mine[k], 0);
          run[k] = __all_sync(0xffffffffu, mine[k] >= 0 && mine[k] == head + lane);
          // the raw buffer is still in use: into L2
          if (run[k] ? lane == 0 : mine[k] >= 0)
            prefetch_l2(p.kv + (int64_t)mine[k] * kRowBytes, (run[k] ? 32 : 1) * kRowBytes);
        }
        if (t > 0) ok = wait_ok(mb_raw_free, (t - 1) & 1);
      } else {
        if (t >= kRing) ok = wait_ok(mb_r_free + 8 * (t % kRing), (t / kRing - 1) & 1);
      }
      if (!ok) break;
      if (c.first && t > 0 && lane == 0) segs[seg % kSegs] = segment_of<kFp8>(c);
      if constexpr (kFp8) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          ring[32 * k + lane] = rank ? code[k] : code[2 + k];  // the other CTA's keys
          if (lane == 0) raw_valid[k] = valid[k];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_expect_tx(mb_raw_full, (__popc(valid[0]) + __popc(valid[1])) * kRowBytes);
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (run[k] ? lane == 0 : mine[k] >= 0)
            bulk_load(base + SM_RAW + (32 * k + lane) * kRowBytes, p.kv + (int64_t)mine[k] * kRowBytes,
                      (run[k] ? 32 : 1) * kRowBytes, mb_raw_full);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) ring[(t % kRing) * kKeys + 32 * k + lane] = code[k];
        __syncwarp();
        if (lane == 0) mbar_arrive(mb_r_full + 8 * (t % kRing));
      }
      if (c.first) ++seg;
      c.next(p);
    }
    if (kFp8 && t > 0) mbar_wait_drain(mb_raw_full, (t - 1) & 1, kWaitNs);  // the last copies have landed
  } else if (warp >= kTail0) {
    const int w = warp - kTail0;
    if constexpr (kFp8) {
      // ------------------------------------------------- rotary part of K
      // Rows 32w + 4x + lane / 8, 16 bytes a lane: copied, they are 16-bit in the cache.
      const uint32_t k_full0 = cluster_map(mb_k_full, 0);
      int kc = 0, seg = 0, left = 0;
      bool two = false;
#pragma unroll 1
      for (int t = 0; t < total; ++t) {
        wait(mb_raw_full, t & 1);
        if (left == 0) {
          left = uniform(segs[seg % kSegs].n);
          two = (uniform(segs[seg % kSegs].flags) & kTwo) != 0;
          ++seg;
        }
        const uint32_t raw = base + SM_RAW + (32 * w + (lane >> 3)) * 656 + 528 + 16 * (lane & 7);
        const uint32_t at = base + SM_K + 8 * kBlk + sw128_off(32 * w + (lane >> 3), lane & 7);
        const uint32_t valid = raw_valid[w] >> (lane >> 3);
#pragma unroll 1
        for (int s = two ? 0 : 1; s < 2; ++s) {
          if (kc > 0) wait(mb_k_free, (kc - 1) & 1);
          // (Q passes through the K buffer's other blocks only)
          {
#pragma unroll 2
            for (int x = 0; x < 8; ++x) {  // four rows on: half a swizzle atom, chunks flip bit 2
              uint4 d = lds16(raw + 4 * 656 * x);
              if (s == 0 || !((valid >> (4 * x)) & 1)) d = make_uint4(0, 0, 0, 0);
              sts16((at + 512 * x) ^ (64 * (x & 1)), d);
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(k_full0);
          ++kc;
        }
        if (lane == 0) mbar_arrive(mb_raw_free);
        --left;
      }
    } else {
      // 16-bit rows go to shared memory when their buffer is free, without a stop in
      // registers: these warps bring this CTA's half of the tile's keys into L2 (the
      // other CTA brings the rest of V's).
#pragma unroll 1
      for (int t = 0; t < total; ++t) {
        wait(mb_r_full + 8 * (t % kRing), (t / kRing) & 1);
        const int code = ring[(t % kRing) * kKeys + 64 * rank + 32 * w + lane];
        __syncwarp();
        if (lane == 0) mbar_arrive(mb_r_free + 8 * (t % kRing));
        if (code >= 0) prefetch_l2(p.kv + (int64_t)code * kRowBytes, kRowBytes);
      }
    }
  } else if (warp == kMmaWarp) {
    // ----------------------------------------------------------- MMA issue
    if (rank == 0) {
      const uint32_t leader = elect_one();
      const uint32_t tm = __reduce_or_sync(0xffffffffu, tmem);  // in a uniform register
      const uint64_t dq = sw128_desc(base + SM_Q, 16, 1024), dk = sw128_desc(base + SM_K, 16, 1024);
      const uint64_t dp = sw128_desc(base + SM_P, 16, 1024), dv = sw128_desc(base + SM_V, kVBlk, 1024);
      int kc = 0, gq = 0;
      bool ok = true;
      int qseg = 0, qleft = 0;  // segment of the next QK
      bool two = false;
      int pseg = 0, pleft = 0, vc = 0;  // of the next PV
      bool fine = false;
#pragma unroll 1
      for (int g = -1; g < total && ok; ++g) {
        // QK of tile g + 1, or of two passes the first; PV of tile g; then the second
#pragma unroll 1
        for (int s = 0; s < 2; ++s) {
          if (g + 1 < total && (s == 0 || two)) {
            ok = wait_ok(mb_k_full, kc & 1);
            if (!ok) break;
            if (s == 0) {
              if (qleft == 0) {  // its first tile is stored, so its descriptor is visible
                qleft = uniform(segs[qseg % kSegs].n);
                two = (uniform(segs[qseg % kSegs].flags) & kTwo) != 0;
                ++qseg;
              }
              --qleft;
              if (gq > 0) ok = wait_ok(mb_s_free, (gq - 1) & 1);  // the softmax has read S(gq - 1)
              if (!ok) break;
              ++gq;
            }
            fence_after_sync();
            uint64_t a = dq, b = dk;
#pragma unroll 1
            for (int kb = 0; kb < kQtBlks; ++kb, b += kBlk >> 4)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma_f16_ts_pair(tm + S_COL, tm + Q_COL + 32 * kb + 8 * k, b + 2 * k, IDESC_QK, (kb | k) != 0 || s > 0,
                                leader);
#pragma unroll 1
            for (int kb = kQtBlks; kb < 9; ++kb, a += kBlk >> 4, b += kBlk >> 4)
#pragma unroll
              for (int k = 0; k < 4; ++k) mma_f16_ss_pair(tm + S_COL, a + 2 * k, b + 2 * k, IDESC_QK, 1, leader);
            mma_commit_pair(mb_k_free, leader);
            ++kc;
            if (s > 0 || !two) mma_commit_pair(mb_s_full, leader);
          }
          if (s == 0 && g >= 0) {
            const bool first = pleft == 0;
            ok = wait_ok(mb_p_full, g & 1);
            if (!ok) break;
            if (first) {
              // the accumulator of the segment before has been read
              if (pseg > 0) ok = wait_ok(mb_o_free, (pseg - 1) & 1);
              if (!ok) break;
              pleft = uniform(segs[pseg % kSegs].n);
              fine = (uniform(segs[pseg % kSegs].flags) & kFine) != 0;
              ++pseg;
            }
#pragma unroll 1
            for (int y = fine ? 0 : 1; y < 2; ++y) {
              ok = wait_ok(mb_v_full, vc & 1);
              if (!ok) break;
              fence_after_sync();
              const uint32_t keep = !first || (fine && y > 0);
#pragma unroll 1
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int x = 0; x < kKeys / 16; ++x)
                  mma_f16_ss_pair(tm + 128 * h, dp + (((x >> 2) * kBlk + 32 * (x & 3)) >> 4),
                                  dv + h * (2 * kVBlk >> 4) + (2048 * x >> 4), IDESC_PV, x > 0 ? 1 : keep, leader);
              mma_commit_pair(mb_v_free, leader);
              ++vc;
            }
            mma_commit_pair(mb_pv, leader);
            --pleft;
          }
        }
      }
      mma_commit_pair(mb_done, leader);  // every MMA of this thread
    }
    __syncwarp();
  } else if (warp >= kSoftmax0 && warp < kSoftmax0 + kSoftmaxWarps) {
    // ------------------------------------------------------------- softmax
    const int sp = warp & 3;                    // TMEM sub-partition: lanes [32 sp, +32)
    const int hh = (warp - kSoftmax0) >> 2;     // S columns [32 hh, +32), O half hh
    const int row = 32 * (sp & 1) + lane;       // of this CTA
    const int q4 = 2 * (sp >> 1) + hh;          // this thread's quarter of the row's keys
    const int kofs = 64 * (sp >> 1) + 32 * hh;  // its first key
    const uint32_t t_sp = tmem + ((uint32_t)(32 * sp) << 16);
    const uint32_t p_full0 = cluster_map(mb_p_full, 0), o_free0 = cluster_map(mb_o_free, 0),
                   s_free0 = cluster_map(mb_s_free, 0);
    uint8_t* prow = sm + SM_P + (sp >> 1) * kBlk;
    int g = 0;
#pragma unroll 1
    for (int seg = 0; g < total; ++seg) {
      wait(mb_q_full + 8 * (seg % kQeSegs), (seg / kQeSegs) & 1);
      const bool live = !named_bar_or(1, kSoftmaxWarps * 32, more == 0);  // all take the same number of barriers
      more = live ? more : 0;
      const Segment& sg = segs[seg % kSegs];
      const int end = live ? g + uniform(sg.n) : total;
      // positions before the drafts, from this thread's first key of the tile on
      int d = -64;
      if (live && (sg.rt * kPairRows + kRows * rank + row) / p.H < sg.nd) d = max(sg.pre - kofs, -64);
      // not 0, so that a hidden key's -inf stays one
      const float rs = fmaxf(p.scale_log2 * __int_as_float((127 + (int)qe[64 * (seg % kQeSegs) + row]) << 23), FLT_MIN);
      float m = kNoMax, L = 0.f;
      bool first = true;
#pragma unroll 1
      for (; g < end; ++g) {
        // keys this thread's row sees, one bit each
        uint32_t allow = d >= 32 ? 0xffffffffu : d > 0 ? (1u << d) - 1 : 0u;
        if (d < 32 && d > -64) {  // drafts among the keys
          const int draft = min((sg.rt * kPairRows + kRows * rank + row) / p.H, p.T - 1);
          uint64_t bits = (uint64_t)p.mask[(int64_t)sg.b * p.mask_stride + draft];
          if (sg.nd < 64) bits &= (1ull << sg.nd) - 1;
          allow |= (uint32_t)(d >= 0 ? bits << d : bits >> -d);
        }
        d = max(d - kKeys, -64);
        wait(mb_s_full, g & 1);
        fence_after_sync();
        // this thread's scores, in registers from here on: S is free for the next tile
        uint32_t s[32];
        tmem_ld32(t_sp + S_COL + 32 * hh, s);
        tmem_wait_ld();
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(s_free0);
        if (allow != 0xffffffffu) {
#pragma unroll
          for (int j = 0; j < 32; ++j) s[j] = (allow >> j) & 1 ? s[j] : 0xff800000u;
        }
        float mx = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
#pragma unroll
        for (int j = 2; j < 32; j += 2) mx = max3(mx, __uint_as_float(s[j]), __uint_as_float(s[j + 1]));
        mx *= rs;  // rs >= 0
        float alpha = 1.f;
        const bool any = named_bar_or(1, kSoftmaxWarps * 32, mx > m + kRescale);
        if (any) {
          rowx[64 * q4 + row] = mx;
          named_bar(1, kSoftmaxWarps * 32);
          const float rm = fmaxf(fmaxf(rowx[row], rowx[64 + row]), fmaxf(rowx[128 + row], rowx[192 + row]));
          if (rm > m + kRescale) {
            alpha = ex2(m - (rm - kHead));
            m = rm - kHead;
            L *= alpha;
          }
        }
        const uint64_t rs2 = pack64(rs, rs), nm2 = pack64(-m, -m);
        uint64_t sum2 = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) {  // the probabilities' pairs take the scores' places
          float a, b;
          unpack64(fma2(pack64(__uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1])), rs2, nm2), a, b);
          a = ex2(a);
          b = ex2(b);
          sum2 = add2(sum2, pack64(a, b));
          if (kBf16) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
            s[j] = *reinterpret_cast<const uint32_t*>(&t);
          } else {
            s[j] = pack_half2(a, b);
          }
        }
        {
          float a, b;
          unpack64(sum2, a, b);
          L += a + b;
        }
        // P's buffer and O are free once PV(t-1) has completed (the epilogue waited for a segment's last)
        if (!first) wait(mb_pv, (g - 1) & 1);
        {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<uint4*>(prow + sw128_off(row, 4 * hh + k)) =
                make_uint4(s[4 * k], s[4 * k + 1], s[4 * k + 2], s[4 * k + 3]);
          if (!first && __any_sync(0xffffffffu, alpha != 1.f)) {
            fence_after_sync();
#pragma unroll 1
            for (int k = 0; k < 8; ++k) {
              uint32_t o[16];
              const uint32_t at = t_sp + 128 * hh + 16 * k;
              tmem_ld16(at, o);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
              tmem_st16(at, o);
            }
            tmem_wait_st();
          }
        }
        fence_proxy_async();
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(p_full0);
        first = false;
      }
      // ------------------------------------------- epilogue of the segment
      named_bar(1, kSoftmaxWarps * 32);  // rowx: every thread is past its use as maxima
      rowx[64 * q4 + row] = L;
      named_bar(1, kSoftmaxWarps * 32);
      L = (rowx[row] + rowx[64 + row]) + (rowx[128 + row] + rowx[192 + row]);
      wait(mb_pv, (g - 1) & 1);
      const bool good = !named_bar_or(1, kSoftmaxWarps * 32, more == 0);
      if (good) {
        fence_after_sync();
        const bool mine = sg.rt * kPairRows + kRows * rank + row < p.T * p.H;
        const bool full = (sg.flags & kFull) != 0;
        const int slot = 2 * pair + (seg == 0 ? 0 : 1);
        const int col0 = 256 * (sp >> 1) + 128 * hh;  // lanes 64-127: CTA 1's columns
        const int64_t grow = (int64_t)sg.b * p.T * p.H + sg.rt * kPairRows + kRows * rank + row;
        const int64_t prow_i = (int64_t)slot * p.slot_rows + kRows * rank + row;
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld32(t_sp + 128 * hh + 32 * k, o);
          tmem_wait_ld();
          if (mine && full) {
            uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p.o) + (grow * DV + col0 + 32 * k) * 2);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t v[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const float a = __uint_as_float(o[8 * e + 2 * x]) * inv, b = __uint_as_float(o[8 * e + 2 * x + 1]) * inv;
                if (p.o_bf16) {
                  const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
                  v[x] = *reinterpret_cast<const uint32_t*>(&t);
                } else {
                  v[x] = pack_half2(a, b);
                }
              }
              dst[e] = make_uint4(v[0], v[1], v[2], v[3]);
            }
          } else if (mine) {
            uint4* dst = reinterpret_cast<uint4*>(p.part_o) + ((int64_t)slot * (DV / 4) + (col0 + 32 * k) / 4) * p.slot_rows +
                         kRows * rank + row;
#pragma unroll
            for (int e = 0; e < 8; ++e)
              dst[(int64_t)e * p.slot_rows] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
        if (mine && q4 == 0) {
          if (full) {
            p.lse[grow] = L == 0.f ? -INFINITY : (m + log2f(L)) * kLn2;
          } else {
            p.part_ml[prow_i * 2] = m;
            p.part_ml[prow_i * 2 + 1] = L;
          }
        }
      }
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(o_free0);
    }
  }
  if (more == 0) atomicExch(err, (int32_t)DSA_ERR_TIMEOUT);
  // every MMA has completed before TMEM is released, and no CTA leaves while the
  // other may still read its shared memory or arrive on its barriers
  __syncthreads();
  mbar_wait_drain(mb_done, 0, kWaitNs);
  fence_before_sync();
  __syncthreads();
  cluster_sync();
  if (warp == 0) {
    fence_after_sync();
    tmem_dealloc_pair(tmem, TMEM_COLS);
  }
}

// Row tiles whose key tiles lie in several segments: o = sum_s w_s o_s / sum_s w_s
// l_s with w_s = 2^(m_s - max m). A lane takes a row and 8 columns of it, so that
// a warp reads 32 rows' neighbouring vectors. Such a tile is cut where a pair's run
// starts inside it; kMergeBlocks blocks belong to each of these starts, and those
// of a tile's first one merge it. The last B * tiles blocks write the row tiles
// that no segment holds: o = 0, lse = -inf.
constexpr int kMergeWarps = 8;
constexpr int kMergeCols = 8;                                                   // of a lane
constexpr int kMergeBlocks = (kPairRows / 32) * (DV / kMergeCols) / kMergeWarps;
__device__ __forceinline__ uint32_t pack_out(const TreeArgs& p, float a, float b) {
  if (!p.o_bf16) return pack_half2(a, b);
  const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&x);
}

__global__ void __launch_bounds__(32 * kMergeWarps) tree_merge_kernel(const TreeArgs p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows = p.T * p.H;
  const int cuts = (p.pairs - 1) * kMergeBlocks;
  cudaGridDependencySynchronize();  // the main kernel's results
  if ((int64_t)blockIdx.x >= cuts) {
    const int tiles = (rows + kPairRows - 1) / kPairRows;
    const int64_t i = (int64_t)blockIdx.x - cuts;
    const int b = (int)(i / tiles), rt = (int)(i % tiles);
    const Req q = load_req(p, b);
    if (q.nt > 0 && rt < q.nrt) return;
    const int end = min(rows, (rt + 1) * kPairRows);
    for (int r = rt * kPairRows + warp; r < end; r += kMergeWarps) {
      const int64_t grow = (int64_t)b * rows + r;
      uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p.o) + grow * DV * 2);
      o[lane] = make_uint4(0, 0, 0, 0);
      o[lane + 32] = make_uint4(0, 0, 0, 0);
      if (lane == 0) p.lse[grow] = -INFINITY;
    }
    return;
  }
  const int pair = 1 + blockIdx.x / kMergeBlocks;
  const Cut cut = p.cuts[pair];
  if (cut.tile == 0 || cut.tile > cut.chunk) return;  // no cut, or not the tile's first
  const int item = (int)(blockIdx.x % kMergeBlocks) * kMergeWarps + warp;
  const int row = 32 * (item % (kPairRows / 32)) + lane;  // of the row tile
  const int col = kMergeCols * (item / (kPairRows / 32));
  if (cut.rt * kPairRows + row >= rows) return;
  const int n = 1 + (int)(((long long)cut.nt - cut.tile + cut.chunk - 1) / cut.chunk);  // segments
  // the first one is slot 0 if the tile starts where its pair's run does, else slot 1
  auto slot = [&](int i) { return 2 * (pair - 1 + i) + (i == 0 && cut.tile < cut.chunk ? 1 : 0); };
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + row;
  float M = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float2 x = ml[(int64_t)slot(i) * p.slot_rows];
    if (x.y > 0.f) M = fmaxf(M, x.x);
  }
  float L = 0.f;
  float acc[kMergeCols];
#pragma unroll
  for (int c = 0; c < kMergeCols; ++c) acc[c] = 0.f;
  const float4* po = reinterpret_cast<const float4*>(p.part_o) + (int64_t)(col / 4) * p.slot_rows + row;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float2 x = ml[(int64_t)slot(i) * p.slot_rows];
    const float4* at = po + (int64_t)slot(i) * (DV / 4) * p.slot_rows;
    float4 v[kMergeCols / 4];
#pragma unroll
    for (int c = 0; c < kMergeCols / 4; ++c) v[c] = at[(int64_t)c * p.slot_rows];
    // 0: saw nothing; a NaN stays one
    const float w = x.y == 0.f ? 0.f : x.y > 0.f ? exp2f(x.x - M) : 1.f;
    L += x.y * w;
#pragma unroll
    for (int c = 0; c < kMergeCols / 4; ++c) {
      acc[4 * c] = x.y == 0.f ? acc[4 * c] : fmaf(v[c].x, w, acc[4 * c]);
      acc[4 * c + 1] = x.y == 0.f ? acc[4 * c + 1] : fmaf(v[c].y, w, acc[4 * c + 1]);
      acc[4 * c + 2] = x.y == 0.f ? acc[4 * c + 2] : fmaf(v[c].z, w, acc[4 * c + 2]);
      acc[4 * c + 3] = x.y == 0.f ? acc[4 * c + 3] : fmaf(v[c].w, w, acc[4 * c + 3]);
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const int64_t grow = (int64_t)cut.b * rows + cut.rt * kPairRows + row;
  uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p.o) + (grow * DV + col) * 2);
#pragma unroll
  for (int c = 0; c < kMergeCols / 8; ++c) {
    uint32_t v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = pack_out(p, acc[8 * c + 2 * e] * inv, acc[8 * c + 2 * e + 1] * inv);
    o[c] = make_uint4(v[0], v[1], v[2], v[3]);
  }
  if (col == 0) p.lse[grow] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
}

std::once_flag g_once[kMaxDevices];
int g_status[kMaxDevices];
int32_t* g_err[kMaxDevices];
int g_pairs[kMaxDevices];

template <int FMT>
cudaError_t setup_kernel() {
  return cudaFuncSetAttribute(tree_mla_kernel<FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES);
}

cudaLaunchConfig_t pair_config(int pairs, cudaStream_t s, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * pairs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = s;
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = 2;
  attr->val.clusterDim.y = 1;
  attr->val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

int ensure_setup(int dev) {
  if (dev < 0 || dev >= kMaxDevices) {
    set_error("tree_mla_decode: device index %d out of range", dev);
    return DSA_ERR_UNSUPPORTED;
  }
  std::call_once(g_once[dev], [dev] {
    cudaError_t e = setup_kernel<DSA_FP8_DS_MLA>();
    if (e == cudaSuccess) e = setup_kernel<DSA_F16>();
    if (e == cudaSuccess) e = setup_kernel<DSA_BF16>();
    int n = 0;
    if (e == cudaSuccess) {
      cudaLaunchAttribute attr{};
      const cudaLaunchConfig_t cfg = pair_config(sm_count(dev) / 2, nullptr, &attr);
      e = cudaOccupancyMaxActiveClusters(&n, tree_mla_kernel<DSA_FP8_DS_MLA>, &cfg);
    }
    if (e == cudaSuccess && tc_error_word(dev, &g_err[dev]) != DSA_OK) e = cudaErrorUnknown;
    g_pairs[dev] = n;
    g_status[dev] = (int)e;
  });
  if (g_status[dev] != 0 || g_pairs[dev] <= 0) {
    set_error("tree_mla_decode setup: %s (%d clusters of two CTAs fit)", cudaGetErrorString((cudaError_t)g_status[dev]),
              g_pairs[dev]);
    return DSA_ERR_CUDA;
  }
  return DSA_OK;
}

template <int FMT>
cudaError_t launch_main(const TreeArgs& p, int dev, cudaStream_t s) {
  cudaLaunchAttribute attr{};
  const cudaLaunchConfig_t cfg = pair_config(p.pairs, s, &attr);
  return cudaLaunchKernelEx(&cfg, tree_mla_kernel<FMT>, p, g_err[dev]);
}

}  // namespace
}  // namespace dsa

using namespace dsa;

// Two partial states per pair, of the rows that a pair can hold.
static size_t tree_workspace(int T, int n_head, int pairs) {
  const int64_t rows = std::min<int64_t>(kPairRows, (int64_t)T * n_head);
  return (size_t)pairs * sizeof(Cut) + (size_t)2 * pairs * rows * kSlotF * sizeof(float);
}

extern "C" size_t dsa_tree_mla_decode_workspace_bytes(int B, int T, int n_head) {
  if (B <= 0 || T <= 0 || n_head <= 0) return 0;
  return tree_workspace(T, n_head, sm_count(current_device()) / 2);
}

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
                  row_stride_ok(bt_stride, max_blocks) && row_stride_ok(mask_stride, T),
              DSA_ERR_INVALID, "tree_mla_decode: bad cache geometry or strides (page=%d max_blocks=%d rows=%lld)",
              page_size, max_blocks, (long long)n_kv_rows);
  const float scale_log2 = (float)(std::fabs(scale) * 1.4426950408889634);
  DSA_REQUIRE(std::isfinite(scale_log2), DSA_ERR_INVALID, "tree_mla_decode: scale must be finite, in f32 too");
  if (B == 0 || T == 0 || n_head == 0) return DSA_OK;
  DSA_REQUIRE(n_head <= 1024 && B <= 65535, DSA_ERR_UNSUPPORTED, "tree_mla_decode: at most 65535 requests of 1024 heads");
  DSA_REQUIRE(o && lse && q && seq_lens && tree_mask && (n_kv_rows == 0 || kv_cache) && (max_blocks == 0 || block_table),
              DSA_ERR_INVALID, "tree_mla_decode: null pointer");
  DSA_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)kv_cache & 15) == 0 && ((uintptr_t)o & 15) == 0, DSA_ERR_INVALID,
              "tree_mla_decode: q, kv_cache and o must be 16-byte aligned");
  const int64_t most = (int64_t)B * (((int64_t)T * n_head + kPairRows - 1) / kPairRows) *
                       std::max<int64_t>(1, ((int64_t)max_blocks * page_size + kKeys - 1) / kKeys);
  const int dev = current_device();
  const int st = ensure_setup(dev);
  if (st != DSA_OK) return st;
  TreeArgs p{};
  p.q = q;
  p.kv = reinterpret_cast<const uint8_t*>(kv_cache);
  p.bt = block_table;
  p.seq_lens = seq_lens;
  p.draft_lens = draft_lens;
  p.mask = tree_mask;
  p.o = o;
  p.lse = lse;
  p.n_kv_rows = n_kv_rows;
  p.bt_stride = bt_stride;
  p.mask_stride = mask_stride;
  p.page = page_size;
  p.page_shift = -1;
  for (int k = 0; k < 31; ++k)
    if (page_size == 1 << k) p.page_shift = k;
  p.max_blocks = max_blocks;
  p.B = B;
  p.T = T;
  p.H = n_head;
  p.pairs = (int)std::min<int64_t>(std::min(g_pairs[dev], sm_count(dev) / 2), most);
  p.slot_rows = (int)std::min<int64_t>(kPairRows, (int64_t)T * n_head);
  p.q_bf16 = q_dtype == DSA_BF16;
  p.o_bf16 = o_dtype == DSA_BF16;
  p.q_sign = scale < 0 ? 0x80008000u : 0u;
  p.scale_log2 = scale_log2;
  const size_t need = tree_workspace(T, n_head, p.pairs);
  DSA_REQUIRE(workspace != nullptr && workspace_bytes >= need, DSA_ERR_WORKSPACE,
              "tree_mla_decode: workspace needs %zu bytes, got %zu", need, workspace_bytes);
  DSA_REQUIRE(((uintptr_t)workspace & 15) == 0, DSA_ERR_INVALID, "tree_mla_decode: workspace must be 16-byte aligned");
  p.cuts = reinterpret_cast<Cut*>(workspace);
  p.part_o = reinterpret_cast<float*>(p.cuts + p.pairs);
  p.part_ml = p.part_o + (size_t)2 * p.pairs * p.slot_rows * DV;
  cudaStream_t s = as_stream(stream);
  const cudaError_t e = kv_format == DSA_FP8_DS_MLA ? launch_main<DSA_FP8_DS_MLA>(p, dev, s)
                        : kv_format == DSA_F16      ? launch_main<DSA_F16>(p, dev, s)
                                                    : launch_main<DSA_BF16>(p, dev, s);
  if (e != cudaSuccess) {
    set_error("tree_mla_kernel launch: %s", cudaGetErrorString(e));
    return DSA_ERR_CUDA;
  }
  const int rt = (T * n_head + kPairRows - 1) / kPairRows;
  // launched while the main kernel's last blocks run
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((int64_t)B * rt + (int64_t)(p.pairs - 1) * kMergeBlocks));
  cfg.blockDim = dim3(32 * kMergeWarps);
  cfg.stream = s;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  const cudaError_t em = cudaLaunchKernelEx(&cfg, tree_merge_kernel, p);
  if (em != cudaSuccess) {
    set_error("tree_merge_kernel launch: %s", cudaGetErrorString(em));
    return DSA_ERR_CUDA;
  }
  return check_launch("tree_merge_kernel");
}
