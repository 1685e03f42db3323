// Causal GQA attention for a prefill chunk on the 5th-generation tensor cores: tcgen05.mma with the score
// tile S, the probability tile P and the output accumulator O all in tensor memory.
//
// A pair of CTAs (cta_group::2) = 2 x 128 query rows over the same keys: the same rows of two query heads of a kv head, or, where a kv
// head has an odd number of them, two row tiles of a head.  It walks the visible keys in tiles of 128:
//     S = Q K^T   tcgen05.mma kind::f16, A = Q (shared memory, resident), B = K tile, 64 keys from each CTA; M 256, N 128, K = D in
//                 steps of 16; fp32 S in tensor memory (two buffers)
//     softmax     eight warps, thread = query row = TMEM lane, two warps share a row (64 keys each): tcgen05.ld S, running maximum
//                 in the log2 domain, P = 2^(S - m) rounded to fp16 and written over the scores with tcgen05.st
//     O += P V    tcgen05.mma with the A operand read from TENSOR MEMORY (the P tile) and B = V^T tile, half of the dimensions from
//                 each CTA; M 256, N D, K = 128 keys in steps of 16; fp32 O in tensor memory
// The cache holds fp8 e4m3 rows in 16-token pages.  Eight conversion warps widen this CTA's half of each K tile to fp16 in the
// canonical K-major 128-byte-swizzled layout, and write its half of the V tile TRANSPOSED ([dimension][token]) so that V is a plain
// K-major B operand as well; the raw bytes of the next tile wait in registers.  Q is pre-multiplied by softmax scale x log2(e) x the
// K descale while it is converted, so scores need no further scaling.  The issuer keeps one S tile ahead of the softmax (S_j+1 is
// issued before P_j V_j), V's conversion runs up to two tiles ahead and K's three.
//
// Why pairs and 128 keys: one CTA with 64 keys a tile spent 92 clocks on the issue of each of its 20 products a tile (its scores
// read 6 KB of shared memory for 32 clocks of work) and all of its conversion warps' time on K and V that the neighbour converted
// too: 3440 clocks for 64 keys, where the products take 1024.  In pairs each product is twice as long, reads half of B and meets half
// of the conversions.  What bounds it now is the chain scores -> softmax -> products over two score buffers (the accumulator takes the
// other half of tensor memory): 3300 clocks from announced probabilities to the scores after next, about as many in the softmax,
// whose 128 x 128 exponentials alone take 1024.  Output gates (of the fp8 cache) wait in K's buffers and output rows leave as one copy per row
// half: read and written directly by the lanes that own the rows, they took 25k clocks a CTA.
// 8192 rows, 24 heads over 4, D = 256: 1623 -> 953 us (865 TFLOP/s); 1024 rows after 29000 1499 -> 916; 333 rows 50 -> 29;
// 32 heads over 8, D = 128, 8192 rows 1304 -> 913.
//
// Rescaling of O when a row maximum grows is lazy: P is computed against the maximum in use, and only when some
// row's true maximum has moved more than 8 (a factor 256, harmless in fp16 / fp32) does the warp wait for the
// outstanding P V products, rescale its 32 rows of O in tensor memory and adopt the new maximum.
// Every wait is bounded; a wait that runs out sets the status word and the CTA unwinds (frees tensor memory).
//
// The reference's counterpart is a query-tiled WMMA kernel (reference:
// third_party/libr4d/r4d_attn_prefill_h256_gqa6.hip:112); nothing is shared with it.
#include <type_traits>

#include "common.cuh"
#include "kv4.cuh"
#include "sm100_ptx.cuh"

namespace r4dxb {
namespace {

constexpr int kQRows = 128;               // of a CTA
constexpr int kKvTile = 128;              // keys of a step; each CTA of the pair prepares half of K's rows and half of V's columns
constexpr int kHalfTile = kKvTile / 2;
constexpr int kPage = 16;
constexpr int kSoftmaxWarps = 8;          // warp w: rows 32 (w % 4) .., keys 64 (w / 4) ..
constexpr int kMmaWarp = kSoftmaxWarps;
constexpr int kConvWarps = 8;
constexpr int kConvThreads = kConvWarps * 32;
constexpr int kThreads = (kSoftmaxWarps + 1 + kConvWarps) * 32;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kSCol = 256;           // S buffers: 256 + 128 b; P overwrites the scores that its own warp has read
constexpr float kRescaleStep = 8.f;

struct TcArgs {
  const __nv_bfloat16* q;      // [T, Hq, D] normed + roped
  const __nv_bfloat16* qg;     // [T, Hq, 2D] (gate in the upper half), may be null when !gated
  const uint8_t* cache;        // [page][Hkv][2][16][D] fp8
  const int* block_table;
  const float* k_descale;
  const float* v_descale;
  __nv_bfloat16* out;          // [T, Hq, D]
  int T, Hq, Hkv, pos0, gated, window;
  int by_head;                 // a pair is two query heads of a kv head over the same rows, else two row tiles of a head
  int* status;
};

struct Kv4Args : TcArgs {
  kv4::Table table;
  const int* key_limit;        // [T] or null: row t also sees this call's keys up to that position
  int splits;                  // pairs that share the keys of a row tile; more than one: partial results
  float* part_acc;             // [splits][T][Hq][D]
  float2* part_ml;             // [splits][T][Hq]: maximum (log2 domain) and sum
};
// (what a kernel is given differs, not only the code: with the longer arguments the fp8 kernels spilled 60 bytes where they spill 24)
template <bool KV4>
using Args = std::conditional_t<KV4, Kv4Args, TcArgs>;

struct Control {
  uint64_t q_full, k_full[2], v_full[2], p_full[2];      // those of the first CTA count both
  uint64_t s_full[2], pv_done[2], o_final;               // commits, to both CTAs
  uint64_t gates;                                        // the output gates lie in K's buffers (this CTA only)
  uint32_t tmem_base;
  int abort_flag;
  float row[2][2][kQRows];                               // [tile parity][half of the keys]: what the two warps of a row exchange
};
struct Kv4Control : Control {
  float inv[kQRows];                                     // 1 / l of the rows
  float q_scale[kQRows];                                 // what takes a row's scores to the log2 domain
  int nan_groups[kQRows];                                // groups of 64 columns in which the row sees a NaN among the values
  uint32_t tops[kConvWarps][4];                          // largest scales and low ends that a warp has met
  float k_back;                                          // 1 / the power of two that the keys are taken by
  float v_back[4];                                       // 1 / the power of two that the group's values are taken by
};

__device__ __forceinline__ uint32_t Fp8x2Bits(uint32_t v16) {
  __half2_raw r = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v16 & 0xFFFFu), __NV_E4M3);
  return *reinterpret_cast<uint32_t*>(&r);
}
// four e4m3 bytes of one word -> two half2 words (bytes 0-1, bytes 2-3), without shifts or masks
__device__ __forceinline__ void Fp8x4ToHalf(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h; }"
      : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ float Exp2Approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// without the division's dozen instructions (its result is off by 2^-22)
__device__ __forceinline__ float SigmoidApprox(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.0f + __expf(-x)));
  return y;
}
// offset of 16-byte chunk c of row r inside a [rows][128 B] tile in the K-major 128-byte-swizzled UMMA layout
__device__ __forceinline__ int Sw128(int r, int c) { return (r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4); }

// offset of gates 8 c .. 8 c + 7 of row r: rows of 2 D bytes whose 16-byte chunks are permuted, so that 32 lanes reading the same
// columns of 32 rows reach all banks
template <int D>
__device__ __forceinline__ int GateChunk(int r, int c) { return r * 2 * D + ((c ^ (r & 7)) << 4); }

// the bits of a flag word in one of the two CTAs' shared memory
__device__ __forceinline__ void OrRemote(uint32_t addr, uint32_t bits) {
  asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(addr), "r"(bits) : "memory");
}

__device__ __forceinline__ void StoreRemote(uint32_t addr, float x) {
  asm volatile("st.relaxed.cluster.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(x) : "memory");
}
// scale and low end of a pair, both times a power of two (exact)
__device__ __forceinline__ uint32_t Mul2Bf16(uint32_t pair, uint32_t power) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(pair), "r"(power));
  return r;
}
// of a pair without its signs, or the largest halves of several: is one infinite or NaN?
__device__ __forceinline__ bool NoNumber(uint32_t pair) { return (pair & 0xffffu) >= 0x7f80u || pair >= 0x7f800000u; }

// Four code pairs of a 4-bit word (codes i and i + 4 in the halves of result i) as fp16 values n s + lo: the codes enter the mantissa of
// 1024 (or, where they lie four bits higher, as 1024 + 16 n), come back out exactly, and one fma rounds to fp16.
__device__ __forceinline__ __half2 AsHalf2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ uint32_t Bits(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
__device__ __forceinline__ uint32_t AndOr(uint32_t a, uint32_t b, uint32_t c) {        // (one instruction: two where the compiler folds constants)
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ void Kv4ToHalf(uint32_t w, __half2 s, __half2 lo, uint32_t (&h)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const uint32_t x = w >> (4 * i);
    const __half2 n0 = __hsub2(AsHalf2(AndOr(x, 0x000f000fu, 0x64006400u)), AsHalf2(0x64006400u));
    const __half2 n1 = __hfma2(AsHalf2(AndOr(x, 0x00f000f0u, 0x64006400u)), AsHalf2(0x2c002c00u), AsHalf2(0xd400d400u));     // / 16 - 64
    h[i] = Bits(__hfma2(n0, s, lo));
    h[i + 1] = Bits(__hfma2(n1, s, lo));
  }
}

// The largest of what scales and low ends may stand for among the keys (or values) of positions `begin` .. `end` - 1, in one group of channels (or all:
// -1), as the exponent of a float, 15 .. 254; by all conversion warps.  The pairs of a head's block b lie at pairs + b page_words.  Called where
// keys or values are tiny, and kept out of line: its registers are not the kernel's.
__device__ __forceinline__ float Bound(uint32_t pair) { return fmaf(15.f, BfLo(pair), BfHi(pair)); }       // of a pair without signs
template <int D>
__device__ __noinline__ int TopExponent(Kv4Control* ctl, kv4::Table table, const uint32_t* pairs, size_t page_words, int begin, int end, int tid, int group) {
  constexpr int NG = kv4::Shape<D>::kGroups, kPieces = 4 * NG;        // pieces: 16 bytes of a block's pairs
  uint32_t top[NG] = {};
#pragma unroll 1
  for (int b = begin / kv4::kBlock + tid / kPieces; b * kv4::kBlock < end; b += kConvThreads / kPieces) {
    const int blk = table.BlockAt(b);
    if (blk < 0) continue;
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(pairs + blk * page_words) + tid % kPieces);
    const uint32_t w[4] = {x.x & 0x7fff7fffu, x.y & 0x7fff7fffu, x.z & 0x7fff7fffu, x.w & 0x7fff7fffu};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int kp = b * kv4::kBlock + (tid % kPieces * 4 + i) / NG;
      if (!NoNumber(w[i]) && kp >= begin && kp < end) top[i % NG] = __vmaxu2(top[i % NG], w[i]);
    }
  }
  asm volatile("bar.sync 6, %0;" ::"n"(kConvThreads) : "memory");      // (the last call's are read)
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const uint32_t t = __reduce_max_sync(0xffffffffu, top[g] & 0xffffu) | __reduce_max_sync(0xffffffffu, top[g] >> 16) << 16;
    if (tid % 32 == 0) ctl->tops[tid / 32][g] = t;
  }
  asm volatile("bar.sync 6, %0;" ::"n"(kConvThreads) : "memory");
  uint32_t most = 0u;
#pragma unroll
  for (int w = 0; w < kConvWarps; ++w)
#pragma unroll
    for (int g = 0; g < NG; ++g)
      if (group < 0 || group == g) most = __vmaxu2(most, ctl->tops[w][g]);
  return min(max(static_cast<int>(__float_as_uint(Bound(most)) >> 23), 15), 254);
}

// Eight channels of a query row times a power of two, as fp16 in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ void StoreQuery(unsigned char* at, const uint4& v, float power) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t h[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = Bits(__floats2half2_rn(BfLo(w[j]) * power, BfHi(w[j]) * power));
  *reinterpret_cast<uint4*>(at) =
      make_uint4(__byte_perm(h[0], h[2], 0x5410), __byte_perm(h[0], h[2], 0x7632), __byte_perm(h[1], h[3], 0x5410), __byte_perm(h[1], h[3], 0x7632));
}
// larger and smaller magnitudes of two pairs of bf16 (their signs mean nothing; a NaN counts for nothing)
__device__ __forceinline__ uint32_t MaxAbs2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t MinAbs2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// A softmax warp's rows (those of its part of the loop in the kernel) once more where some value is small or very large: each row times the power
// of two that brings its largest value to 2^14 .. 2^15, in which fp16 holds bf16 as it is, and what takes its scores back.  (Out of line: the
// rows' maxima for every call took 1 us of the 15 of 333 rows.)
template <int D>
__device__ __noinline__ void ScaleQueries(unsigned char* Qs, float* q_scale, const __nv_bfloat16* q, size_t stride, int rows, float score_scale) {
  constexpr int kLanes = D / 8;
#pragma unroll 1
  for (int i = threadIdx.x; i < kQRows * kLanes; i += kSoftmaxWarps * 32) {
    const int row = i / kLanes, c = i % kLanes;
    const uint4 v = row < rows ? __ldg(reinterpret_cast<const uint4*>(q + row * stride + c * 8)) : make_uint4(0u, 0u, 0u, 0u);
    uint32_t top = MaxAbs2(MaxAbs2(v.x, v.y), MaxAbs2(v.z, v.w)) & 0x7fff7fffu;
    top = max(top >> 16, top & 0xffffu);
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const uint32_t exponent = top >> 7, p = exponent == 255u ? 127u : min(268u - exponent, 253u);
    StoreQuery(Qs + (c >> 3) * (kQRows * 128) + Sw128(row, c & 7), v, __uint_as_float(p << 23));
    if (c == 0) q_scale[row] = score_scale * __uint_as_float((254u - p) << 23);
  }
}

// KV4: the 4-bit cache (kv4.cuh) in place of the fp8 one; only what the conversion warps load and store differs, and
//   - keys enter with the channels of every eight in the order 0 4 1 5 2 6 3 7 (that of Kv4ToHalf), and so does Q;
//   - a value group that is NaN is stored as zeros, and noted for the rows that see it: 0 x NaN would reach the rows that do not.
//     (NaN keys need nothing: a score that a row does not see is replaced before it is used.)
//   - values in front of the first row's window, whose bytes may be anything, are not loaded: 0 x infinity would reach every row;
//   - pages that the table or pool does not have are NaN keys;
//   - the softmax warps bring Q, and all 16 warps write whole rows at the end, their gates loaded ahead: of a CTA of one tile (24 heads over 4 of
//     256) 26000 clocks became 21500, half of which are start and end.
// The same chain bounds it as the fp8 cache's (1024 rows after 8000 keys: tensor pipe 44 %, issue slots 51 %); widening codes costs the conversion
// warps no more than widening fp8 does.  24 heads over 4 of 256: 333 rows 15.4 us, 1024 after 29000 722 to 767, 8192 819 to 899 by the power that
// the chip is left; 32 over 8 of 128, 8192 rows 759; of 64 712.
template <int D, bool KV4>
__global__ void __launch_bounds__(kThreads, 1) AttnPrefillTcKernel(Args<KV4> a) {
  constexpr int NS = D / 64;                          // 64-dimension slabs (one 128-byte swizzle row of fp16 each)
  [[maybe_unused]] const float score_scale = rsqrtf(static_cast<float>(D)) * 1.4426950408889634f;       // of the scores of the 4-bit cache, to the log2 domain
  constexpr int kQBytes = NS * kQRows * 128;
  constexpr int kKBytes = NS * kHalfTile * 128;       // [slab][64 keys][128 B]
  constexpr int kVSlab = D / 2 * 128;                 // V^T: [64-key slab][half of the dimensions][128 B]
  constexpr int kVBytes = 2 * kVSlab;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  unsigned char* Qs = smem;
  unsigned char* Ks = Qs + kQBytes;                   // [2][kKBytes]
  unsigned char* Vs = Ks + 2 * kKBytes;               // [2][kVBytes]
  using Ctl = std::conditional_t<KV4, Kv4Control, Control>;
  Ctl* ctl = reinterpret_cast<Ctl*>(Vs + 2 * kVBytes);
  volatile int* abort_flag = &ctl->abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1;
  const int hq = a.by_head ? blockIdx.x : blockIdx.x >> 1;
  const int hkv = hq / (a.Hq / a.Hkv);
  const int step = static_cast<int>(gridDim.y - 1 - blockIdx.y);            // the rows with the most keys start first, in all heads
  const int first_row = step * (a.by_head ? kQRows : 2 * kQRows);           // of the pair
  const int q0 = a.by_head ? first_row : first_row + rank * kQRows;
  const int rows = max(0, min(kQRows, a.T - q0));
  const int kv_limit = a.pos0 + a.T;                  // tokens present in the cache
  int splits = 1;
  const int* key_limit = nullptr;
  if constexpr (KV4) {
    splits = a.splits;
    key_limit = a.key_limit;
  }
  const bool limits = KV4 && key_limit != nullptr, partial = KV4 && splits > 1;
  const int kv_end = limits ? kv_limit : a.pos0 + min(a.T, first_row + (a.by_head ? kQRows : 2 * kQRows));      // first key no row of the pair may see
  const int kv_first = a.window > 0 ? max(0, a.pos0 + first_row - a.window + 1) : 0;
  // (a pair that shares the keys with others has one part of their tiles, `per` of them at most)
  const int tiles = (kv_end + kKvTile - 1) / kKvTile - kv_first / kKvTile;  // at least 1
  const int per = KV4 ? (tiles + splits - 1) / splits : tiles, skip = KV4 ? static_cast<int>(blockIdx.z) * per : 0;
  const int tile0 = kv_first / kKvTile + skip, ntiles = min(per, tiles - skip);
  if constexpr (KV4) {
    // Before the allocation of tensor memory, too: a kernel that this one waits for may still have its own before it.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (ntiles <= 0) {                                // no tile is left for this part: no row sees any of it
      for (int r = threadIdx.x; r < rows; r += kThreads)
        a.part_ml[(static_cast<size_t>(blockIdx.z) * a.T + q0 + r) * a.Hq + hq] = make_float2(-INFINITY, 0.f);
      return;
    }
  }

  if (threadIdx.x == 0) {
    ptx::MbarInit(&ctl->q_full, 2 * kConvWarps);
    for (int b = 0; b < 2; ++b) {
      ptx::MbarInit(&ctl->k_full[b], 2 * kConvWarps);
      ptx::MbarInit(&ctl->v_full[b], 2 * kConvWarps);
      ptx::MbarInit(&ctl->p_full[b], 2 * kSoftmaxWarps);
      ptx::MbarInit(&ctl->s_full[b], 1);
      ptx::MbarInit(&ctl->pv_done[b], 1);
    }
    ptx::MbarInit(&ctl->o_final, 1);
    ptx::MbarInit(&ctl->gates, kConvWarps);
    ctl->abort_flag = 0;
    ptx::MbarFenceInit();
  }
  if constexpr (KV4) {
    if (threadIdx.x < kQRows) ctl->nan_groups[threadIdx.x] = 0;
    if (threadIdx.x < 4) ctl->v_back[threadIdx.x] = 1.f;
    if (threadIdx.x == 0) ctl->k_back = 1.f;
    if (threadIdx.x < kQRows) ctl->q_scale[threadIdx.x] = score_scale;
  }
  if (warp == kMmaWarp) {
    ptx::TmemAllocPair(&ctl->tmem_base, kTmemCols);
    ptx::TmemRelinquishPair();
  }
  ptx::TcFenceBefore();
  // The partner's barriers exist before anything arrives at them.  (4-bit cache: each role waits for that, and for tensor memory, which takes
  // 1500 clocks, with its first loads under way.)
  uint32_t tbase = 0u;
  auto join = [&]() {
    ptx::ClusterWait();
    ptx::TcFenceAfter();
    tbase = ctl->tmem_base;
  };
  if constexpr (KV4) {
    ptx::ClusterArrive();
  } else {
    __syncthreads();
    ptx::ClusterSync();
    ptx::TcFenceAfter();
    tbase = ctl->tmem_base;
  }

  if (warp > kMmaWarp) {
    // ---------------- conversion warps: Q once, then this CTA's half of K and of V^T of every key tile ----------------
    const int tid = threadIdx.x - (kMmaWarp + 1) * 32, cw = warp - (kMmaWarp + 1);
    [[maybe_unused]] const uint32_t q_full = ptx::MapToRank(ptx::SmemAddr(&ctl->q_full), 0);
    const uint32_t k_full = ptx::MapToRank(ptx::SmemAddr(&ctl->k_full[0]), 0), v_full = ptx::MapToRank(ptx::SmemAddr(&ctl->v_full[0]), 0);
    // K: a thread owns 16 dimensions of KI consecutive keys (16 lanes read a row); which of two neighbouring keys it stores first
    // depends on its slab, so that the 32 stores of an instruction spread over all banks.
    constexpr int CH = D / 16, KI = D / 64;
    const int ch = tid % CH, key0 = tid / CH * KI, flip = (ch >> 2) & 1;
    // V: a thread owns VD dimensions of 8 consecutive keys and turns them into VD rows of 16 bytes; the byte it starts with depends on
    // its lane, and the two halves of a warp are 4 key groups apart, for the same reason.
    constexpr int VD = D / 32, VW = VD >= 4 ? VD / 4 : 1;
    const int dq = lane & 15, tg = (cw & 3) + ((lane >> 4) << 2) + ((cw >> 2) << 3);
    const size_t page_bytes = static_cast<size_t>(a.Hkv) * 2 * kPage * D;
    const uint8_t* cache_k = a.cache + static_cast<size_t>(hkv) * 2 * kPage * D + ch * 16;
    const uint8_t* cache_v = a.cache + static_cast<size_t>(hkv) * 2 * kPage * D + kPage * D + rank * (D / 2) + dq * VD;
    uint4 kraw[KI];
    uint32_t vraw[8][VW];
    // 4-bit cache.  K: a thread owns the words of channels 8 kc .. of every 32 of one key (the keys of eight lanes are 4 apart, for the
    // banks of its stores).  V: word vword (of this CTA's half) of VT consecutive tokens, turned into eight rows of VT fp16 values; the
    // lanes of a store have the tokens of half a tile (all banks), the words of a warp lie in the same 32 bytes of the cache.
    constexpr int NJ = D / 32, NG = kv4::Shape<D>::kGroups, VT = D / 32, VWords = D / 16;
    const int kc = tid & 3, kkey = (tid >> 5) * 8 + ((tid >> 3) & 3) + (tid & 4);
    constexpr int VUnits = kHalfTile / VT;       // groups of tokens in half a tile: 8, 16 or 32 lanes
    const int vsub = lane / VUnits;         // warps 0 .. 3: the first half of the tile
    const int vword = D == 256 ? (cw & 3) * 2 + (vsub & 1) + (vsub >> 1) * 8 : (cw & 3) * (VWords / 4) + vsub;
    const int vtok = (cw >> 2) * kHalfTile + lane % VUnits * VT, vgroup = (rank * VWords + vword) >> 3;
    uint32_t kcodes[NJ], kpairs[NG], vcodes[VT], vpairs[VT];
    // the blocks of the next tiles' keys and values are looked up a tile ahead: an address that waits for its table entry held a warp up
    // for a quarter of a tile's time
    auto block_index = [&](int b) {
      if constexpr (KV4) return a.table.BlockAt(b);
      else return 0;
    };
    auto block_of = [&](int j, int first) { return block_index(((tile0 + j) * kKvTile + first) >> 4); };
    const int kfirst = rank * kHalfTile + kkey;
    int kblk = block_of(0, kfirst), vblk = block_of(0, vtok);
    // where a thread's words lie in a block: the same in every tile, since tiles begin with blocks
    int kword[2] = {}, vwords[VT] = {};
    if constexpr (KV4) {
      kword[0] = kv4::Word<D, false>(kfirst & 15, kc);
      kword[1] = kv4::Word<D, false>(kfirst & 15, D == 256 ? 16 + kc : kc);
#pragma unroll
      for (int t = 0; t < VT; ++t) vwords[t] = kv4::Word<D, true>((vtok & 15) + t, rank * VWords + vword);
    }
    const int kpair = 2 * D + (kfirst & 15) * NG, vpair = kv4::Shape<D>::kPart / 4 + 2 * D + (vtok & 15) * NG + vgroup;
    const uint32_t* cache4 = reinterpret_cast<const uint32_t*>(a.cache) + static_cast<size_t>(hkv) * (kv4::Shape<D>::kRun / 4);
    const size_t page_words = static_cast<size_t>(a.Hkv) * (kv4::Shape<D>::kRun / 4);
    // raw bytes of a tile into registers, zeros past the last token
    auto load_k = [&](int j) {
      if constexpr (KV4) {
        const int kp = (tile0 + j) * kKvTile + kfirst, blk = kblk;
        kblk = block_of(j + 1, kfirst);
#pragma unroll
        for (int i = 0; i < NJ; ++i) kcodes[i] = 0u;
#pragma unroll
        for (int i = 0; i < NG; ++i) kpairs[i] = 0u;
        if (j < ntiles && kp < kv_limit) {
          if (blk < 0) {
#pragma unroll
            for (int i = 0; i < NG; ++i) kpairs[i] = 0x7fc07fc0u;
          } else {
            const uint32_t* at = cache4 + blk * page_words;
            if constexpr (D == 256) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(at + kword[h]));
                kcodes[4 * h] = v.x; kcodes[4 * h + 1] = v.y; kcodes[4 * h + 2] = v.z; kcodes[4 * h + 3] = v.w;
              }
              const uint4 p = __ldg(reinterpret_cast<const uint4*>(at + kpair));
              kpairs[0] = p.x; kpairs[1] = p.y; kpairs[2] = p.z; kpairs[3] = p.w;
            } else if constexpr (D == 128) {
              const uint4 v = __ldg(reinterpret_cast<const uint4*>(at + kword[0]));
              kcodes[0] = v.x; kcodes[1] = v.y; kcodes[2] = v.z; kcodes[3] = v.w;
              const uint2 p = __ldg(reinterpret_cast<const uint2*>(at + kpair));
              kpairs[0] = p.x; kpairs[1] = p.y;
            } else {
              const uint2 v = __ldg(reinterpret_cast<const uint2*>(at + kword[0]));
              kcodes[0] = v.x; kcodes[1] = v.y;
              kpairs[0] = __ldg(at + kpair);
            }
          }
        }
        return;
      }
      const int kp0 = (tile0 + j) * kKvTile + rank * kHalfTile + key0;
#pragma unroll
      for (int i = 0; i < KI; ++i) kraw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (j < ntiles && kp0 < kv_limit) {
        const uint8_t* base = cache_k + a.block_table[kp0 >> 4] * page_bytes;
#pragma unroll
        for (int i = 0; i < KI; ++i) {
          const int kp = kp0 + (i ^ flip);
          if (kp < kv_limit) kraw[i] = __ldg(reinterpret_cast<const uint4*>(base + (kp & 15) * D));
        }
      }
    };
    const uint32_t v_whole = max(kv_limit - kv_first - VT + 1, 0);
    auto load_v = [&](int j) {
      if constexpr (KV4) {
        const int kp0 = (tile0 + j) * kKvTile + vtok, blk = vblk;
        vblk = block_of(j + 1, vtok);
#pragma unroll
        for (int t = 0; t < VT; ++t) vcodes[t] = vpairs[t] = 0u;
        if (j < ntiles && kp0 < kv_limit) {
          if (blk >= 0) {
            const uint32_t* at = cache4 + blk * page_words;
            const uint32_t from = kp0 - kv_first;                              // (of the keys from kv_first on; large in front of it)
            if (from < v_whole) {
#pragma unroll
              for (int t = 0; t < VT; ++t) {
                vcodes[t] = __ldg(at + kv4::Shape<D>::kPart / 4 + vwords[t]);
                vpairs[t] = __ldg(at + vpair + t * NG);
              }
            } else {
#pragma unroll
              for (int t = 0; t < VT; ++t)
                if (from + t < static_cast<uint32_t>(kv_limit - kv_first)) {
                  vcodes[t] = __ldg(at + kv4::Shape<D>::kPart / 4 + vwords[t]);
                  vpairs[t] = __ldg(at + vpair + t * NG);
                }
            }
          }
        }
        return;
      }
      const int kp0 = (tile0 + j) * kKvTile + tg * 8;
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int w = 0; w < VW; ++w) vraw[t][w] = 0u;
      if (j < ntiles && kp0 < kv_limit) {
        const uint8_t* base = cache_v + a.block_table[kp0 >> 4] * page_bytes + (kp0 & 15) * D;
#pragma unroll
        for (int t = 0; t < 8; ++t)
          if (kp0 + t < kv_limit) {
            if constexpr (VW == 2) {
              const uint2 v = __ldg(reinterpret_cast<const uint2*>(base + t * D));
              vraw[t][0] = v.x;
              vraw[t][1] = v.y;
            } else {
              vraw[t][0] = __ldg(reinterpret_cast<const uint32_t*>(base + t * D));
            }
          }
      }
    };
    // 4-bit cache: keys and values of ordinary size are widened as they are, none being above 2^15: fp16 keeps those above 6e-5 with all their bits and is
    // off by 2^-25 at most below.  Where most of the first 32 keys are below 2^-12 throughout, or their values below 2^-6 throughout a group of 64
    // columns, that is no small part of them: the pair then looks through the scales and low ends of all of them and takes the keys, or the
    // group's values, times the power of two that brings the largest to 2^14 .. 2^15, and the scores, or the sums, back in the end.  (Such a look
    // ahead of every call took 10 us of a CTA of 8192 keys at D = 256: 885 us instead of 803 for 8192 rows of 24 heads over 4; a look at every tile's
    // keys, with a power each, 3 to 10 %.  Each warp looks at the 32 keys for itself: the eight run apart, and a barrier of theirs once in the
    // beginning, which brings them in step, took 3 %.)
    const int v_begin = max(kv_first, tile0 * kKvTile), v_end = min((tile0 + ntiles) * kKvTile, kv_limit);      // of the keys whose values are loaded
    constexpr int kOwnGroups = NG > 1 ? NG / 2 : 1;      // of this CTA's columns of the values
    uint32_t k_power = 0x3f803f80u, v_power = 0x3f803f80u;                 // as two bf16; of this thread's group
    uint32_t k_sample[NG] = {}, v_sample[kOwnGroups] = {};                 // the pairs of one of the 32 keys
    auto load_sample = [&]() {
      if constexpr (KV4) {
        const int kp = v_begin + lane, blk = block_index(kp < v_end ? kp >> 4 : -1);
        if (blk >= 0) {
          const uint32_t* at = cache4 + blk * page_words + 2 * D + (kp & 15) * NG;
#pragma unroll
          for (int g = 0; g < NG; ++g) k_sample[g] = __ldg(at + g);
#pragma unroll
          for (int g = 0; g < kOwnGroups; ++g) v_sample[g] = __ldg(at + kv4::Shape<D>::kPart / 4 + rank * NG / 2 + g);
        }
      }
    };
    auto choose_powers = [&]() {
      if constexpr (KV4) {
        auto most_of = [&](bool some) { return 2 * __popc(__ballot_sync(0xffffffffu, some && v_begin + lane < v_end)) > min(32, v_end - v_begin); };
        uint32_t top = 0u;
#pragma unroll
        for (int g = 0; g < NG; ++g) top = __vmaxu2(top, k_sample[g] & 0x7fff7fffu);
        bool tiny = false;                       // (the same for all warps, and the first the same for both CTAs)
#pragma unroll
        for (int g = 0; g < kOwnGroups; ++g) tiny |= most_of(Bound(v_sample[g] & 0x7fff7fffu) < 0.015625f);
        if (most_of(Bound(top) < 0.000244140625f)) {
          const int exponent = TopExponent<D>(ctl, a.table, cache4 + 2 * D, page_words, v_begin, v_end, tid, -1);
          k_power = static_cast<uint32_t>((268 - exponent) << 7) * 0x10001u;
          if (tid == 0) ctl->k_back = __uint_as_float(static_cast<uint32_t>(exponent - 14) << 23);
        }
        asm volatile("bar.arrive 7, %0;" ::"n"((kSoftmaxWarps + kConvWarps) * 32) : "memory");
        if (tiny) {
          const int exponent = TopExponent<D>(ctl, a.table, cache4 + kv4::Shape<D>::kPart / 4 + 2 * D, page_words, v_begin, v_end, tid, vgroup);
          v_power = static_cast<uint32_t>((268 - exponent) << 7) * 0x10001u;
          if (lane % VUnits == 0 && cw < 4 && (vword & 7) == 0) {
            // each CTA's rows have all the columns
            for (int peer = 0; peer < 2; ++peer)
              StoreRemote(ptx::MapToRank(ptx::SmemAddr(&ctl->v_back[vgroup]), peer), __uint_as_float(static_cast<uint32_t>(exponent - 14) << 23));
            asm volatile("fence.acq_rel.cluster;" ::: "memory");
          }
        }
      }
    };
    unsigned char* k_dst = Ks + (ch >> 2) * (kHalfTile * 128);
    auto store_k = [&](int j) {
      if constexpr (KV4) {
        unsigned char* at = Ks + (j & 1) * kKBytes;
#pragma unroll
        for (int i = 0; i < NG; ++i) kpairs[i] = Mul2Bf16(kpairs[i], k_power);
#pragma unroll
        for (int i = 0; i < NJ; ++i) {
          const uint32_t pair = kpairs[i >> 1];
          uint32_t h[4];
          Kv4ToHalf(kcodes[i], __float2half2_rn(BfLo(pair)), __float2half2_rn(BfHi(pair)), h);
          *reinterpret_cast<uint4*>(at + (i >> 1) * (kHalfTile * 128) + Sw128(kkey, (i & 1) * 4 + kc)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        ptx::FenceProxyAsyncShared();
        __syncwarp();
        if (lane == 0) ptx::MbarArriveRemote(k_full + (j & 1) * 8);
        return;
      }
      unsigned char* at = k_dst + (j & 1) * kKBytes;
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int off = Sw128(key0 + (i ^ flip), (ch & 3) * 2);              // the second chunk sits at off ^ 16
        uint4 lo, hi;
        Fp8x4ToHalf(kraw[i].x, lo.x, lo.y);
        Fp8x4ToHalf(kraw[i].y, lo.z, lo.w);
        Fp8x4ToHalf(kraw[i].z, hi.x, hi.y);
        Fp8x4ToHalf(kraw[i].w, hi.z, hi.w);
        *reinterpret_cast<uint4*>(at + off) = lo;
        *reinterpret_cast<uint4*>(at + (off ^ 16)) = hi;
      }
      ptx::FenceProxyAsyncShared();
      __syncwarp();
      if (lane == 0) ptx::MbarArriveRemote(k_full + (j & 1) * 8);
    };
    unsigned char* v_dst = Vs + (tg >> 3) * kVSlab;
    auto store_v = [&](int j) {
      if constexpr (KV4) {
        unsigned char* at = Vs + (j & 1) * kVBytes + (vtok >> 6) * kVSlab;
        uint32_t top = 0u;
#pragma unroll
        for (int t = 0; t < VT; ++t) top = __vmaxu2(top, vpairs[t] & 0x7fff7fffu);
        if (NoNumber(top)) {
#pragma unroll
          for (int t = 0; t < VT; ++t)
            if (NoNumber(vpairs[t] & 0x7fff7fffu)) {
              vpairs[t] = 0u;
              const int kp = (tile0 + j) * kKvTile + vtok + t;
              if ((vword & 7) == 0)              // one of the threads of the group
                for (int peer = 0; peer < 2; ++peer) {
                  const int first = a.by_head ? first_row : first_row + peer * kQRows;
                  const uint32_t flags = ptx::MapToRank(ptx::SmemAddr(&ctl->nan_groups[0]), peer);
                  for (int r = 0; r < kQRows && first + r < a.T; ++r) {
                    const int qpos = a.pos0 + first + r, last = limits ? max(qpos, key_limit[first + r]) : qpos;
                    if (kp <= last && (a.window == 0 || kp > qpos - a.window)) OrRemote(flags + 4 * r, 1u << vgroup);
                  }
                }
            }
          asm volatile("fence.acq_rel.cluster;" ::: "memory");
        }
#pragma unroll
        for (int t = 0; t < VT; ++t) vpairs[t] = Mul2Bf16(vpairs[t], v_power);
        __half2 s2[VT / 2], lo2[VT / 2];
#pragma unroll
        for (int t = 0; t < VT / 2; ++t) {
          s2[t] = __floats2half2_rn(BfLo(vpairs[2 * t]), BfLo(vpairs[2 * t + 1]));
          lo2[t] = __floats2half2_rn(BfHi(vpairs[2 * t]), BfHi(vpairs[2 * t + 1]));
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {            // channels 0 .. 3 and 4 .. 7: a half of each token's word
          uint32_t h[VT / 2][4];
#pragma unroll
          for (int t = 0; t < VT / 2; ++t) Kv4ToHalf(__byte_perm(vcodes[2 * t], vcodes[2 * t + 1], q == 0 ? 0x5410 : 0x7632), s2[t], lo2[t], h[t]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            unsigned char* dst = at + Sw128(vword * 8 + 4 * q + i, (vtok >> 3) & 7) + (vtok & 7) * 2;
            if constexpr (VT == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(h[0][i], h[1][i], h[2][i], h[3][i]);
            else if constexpr (VT == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(h[0][i], h[1][i]);
            else *reinterpret_cast<uint32_t*>(dst) = h[0][i];
          }
        }
        ptx::FenceProxyAsyncShared();
        __syncwarp();
        if (lane == 0) ptx::MbarArriveRemote(v_full + (j & 1) * 8);
        return;
      }
      unsigned char* at = v_dst + (j & 1) * kVBytes;
#pragma unroll
      for (int s = 0; s < VD; ++s) {
        const int byte = (s + dq) & 3;
        const uint32_t sel = byte * 0x11 + 0x40;                             // that byte of both words
        uint32_t h[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) h[t] = Fp8x2Bits(__byte_perm(vraw[2 * t][s >> 2], vraw[2 * t + 1][s >> 2], sel));
        *reinterpret_cast<uint4*>(at + Sw128(dq * VD + (s & 4) + byte, tg & 7)) = make_uint4(h[0], h[1], h[2], h[3]);
      }
      ptx::FenceProxyAsyncShared();
      __syncwarp();
      if (lane == 0) ptx::MbarArriveRemote(v_full + (j & 1) * 8);
    };

    load_k(0);
    load_sample();
    if constexpr (KV4) join();
    if constexpr (!KV4) {
      const float scale = rsqrtf(static_cast<float>(D)) * 1.4426950408889634f * a.k_descale[hkv];
      auto widen = [&](const uint4& v) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __half2 p = __floats2half2_rn(BfLo(w[j]) * scale, BfHi(w[j]) * scale);
          h[j] = *reinterpret_cast<const uint32_t*>(&p);
        }
        return make_uint4(h[0], h[1], h[2], h[3]);
      };
#pragma unroll 4
      for (int i = tid; i < kQRows * (D / 8); i += kConvThreads) {
        const int r = i / (D / 8), c = i % (D / 8);
        uint4 o = make_uint4(0u, 0u, 0u, 0u);
        if (r < rows) o = widen(*reinterpret_cast<const uint4*>(a.q + (static_cast<size_t>(q0 + r) * a.Hq + hq) * D + c * 8));
        *reinterpret_cast<uint4*>(Qs + (c >> 3) * (kQRows * 128) + Sw128(r, c & 7)) = o;
      }
      ptx::FenceProxyAsyncShared();
      __syncwarp();
      if (lane == 0) ptx::MbarArriveRemote(q_full);
    }
    // K runs two tiles ahead of V: K's buffer is free when the scores are done, one product earlier than V's
    if constexpr (KV4) choose_powers();
    store_k(0);
    load_k(1);
    load_v(0);
    if (ntiles > 1) {
      store_k(1);
      load_k(2);
    }
    bool ok = true;
    for (int j = 0; j < ntiles && ok; ++j) {
      const uint32_t ph = static_cast<uint32_t>(j >> 1) & 1u;
      if (j >= 2) ok = ptx::WarpMbarWait(&ctl->pv_done[j & 1], ph ^ 1u, abort_flag, 12);    // P_(j-2) V_(j-2) has consumed the buffer
      if (!ok) break;
      store_v(j);
      load_v(j + 1);
      if (j + 2 < ntiles) {
        ok = ptx::WarpMbarWait(&ctl->s_full[j & 1], ph, abort_flag, 11);                    // S_j has consumed the buffer
        if (!ok) break;
        store_k(j + 2);
        load_k(j + 3);
      }
    }
    // the output gates of this CTA's rows, into K's buffers once the last scores have read them
    if constexpr (!KV4) {
      if (ok && a.gated) ok = ptx::WarpMbarWait(&ctl->s_full[(ntiles - 1) & 1], static_cast<uint32_t>((ntiles - 1) >> 1) & 1u, abort_flag, 13);
      if (ok && a.gated) {
#pragma unroll 4
        for (int i = tid; i < rows * (D / 8); i += kConvThreads) {
          const int r = i / (D / 8), c = i % (D / 8);
          const __nv_bfloat16* src = a.qg + ((static_cast<size_t>(q0 + r) * a.Hq + hq) * 2 + 1) * D + c * 8;
          uint4 g;
          if (reinterpret_cast<uintptr_t>(a.qg) % 16 == 0) {
            g = *reinterpret_cast<const uint4*>(src);
          } else {                              // (their base may lie at any 4 bytes)
            const uint32_t* w = reinterpret_cast<const uint32_t*>(src);
            g = make_uint4(w[0], w[1], w[2], w[3]);
          }
          *reinterpret_cast<uint4*>(Ks + GateChunk<D>(r, c)) = g;
        }
        __syncwarp();
        if (lane == 0) ptx::MbarArrive(&ctl->gates);
      }
    }
  } else if (warp == kMmaWarp) {
    // ---------------- MMA issuer (one thread of the first CTA) ----------------
    if constexpr (KV4) join();
    if (rank == 0 && lane == 0) {
      constexpr uint32_t idesc_s = ptx::UmmaInstrDescF16(2 * kQRows, kKvTile, false);
      constexpr uint32_t idesc_o = ptx::UmmaInstrDescF16(2 * kQRows, D, false);
      const uint64_t qd = ptx::UmmaDescSw128(ptx::SmemAddr(Qs)), kd = ptx::UmmaDescSw128(ptx::SmemAddr(Ks));
      const uint64_t vd = ptx::UmmaDescSw128(ptx::SmemAddr(Vs));       // (the address is the low field, in units of 16 bytes)
      const uint32_t s_full = ptx::SmemAddr(&ctl->s_full[0]), pv_done = ptx::SmemAddr(&ctl->pv_done[0]);
      auto scores = [&](int b) {
        ptx::TcFenceAfter();
        const uint64_t kb = kd + b * (kKBytes / 16);
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            ptx::UmmaF16Pair(tbase + kSCol + b * kKvTile, qd + (s * (kQRows * 128) + k * 32) / 16, kb + (s * (kHalfTile * 128) + k * 32) / 16,
                             idesc_s, (s > 0 || k > 0) ? 1u : 0u);
        ptx::UmmaCommitPairAt(s_full + b * 8, 3);
      };
      bool ok = ptx::MbarWait(&ctl->q_full, 0, abort_flag, 1) && ptx::MbarWait(&ctl->k_full[0], 0, abort_flag, 2);
      if (ok) scores(0);
      for (int j = 0; j < ntiles && ok; ++j) {
        const int b = j & 1;
        const uint32_t ph = static_cast<uint32_t>(j >> 1) & 1u;
        if (j + 1 < ntiles) {
          // Its buffer's scores were read before P_(j-1) was announced, and P_(j-1) V_(j-1), which reads the probabilities that took
          // their place, was issued before it: products run in the order of their issue.
          ok = ptx::MbarWait(&ctl->k_full[b ^ 1], static_cast<uint32_t>((j + 1) >> 1) & 1u, abort_flag, 2);
          if (!ok) break;
          scores(b ^ 1);
        }
        ok = ptx::MbarWait(&ctl->v_full[b], ph, abort_flag, 4) && ptx::MbarWait(&ctl->p_full[b], ph, abort_flag, 3);
        if (!ok) break;
        ptx::TcFenceAfter();
        const uint64_t vb = vd + b * (kVBytes / 16);
        const uint32_t pt = tbase + kSCol + b * kKvTile;
#pragma unroll
        for (int k = 0; k < kKvTile / 16; ++k)
          ptx::UmmaF16PairFromTmem(tbase, pt + (k >> 2) * 64 + (k & 3) * 8, vb + ((k >> 2) * kVSlab + (k & 3) * 32) / 16, idesc_o,
                                   (j > 0 || k > 0) ? 1u : 0u);
        ptx::UmmaCommitPairAt(pv_done + b * 8, 3);
      }
      if (ok) ptx::UmmaCommitPairAt(ptx::SmemAddr(&ctl->o_final), 3);
    }
    __syncwarp();
  } else {
    // ---------------- softmax warps: thread = query row = TMEM lane, two warps share a row ----------------
    const int half = warp >> 2, r = (warp & 3) * 32 + lane;
    const int qp = a.pos0 + q0 + r;                               // position of this row's query
    [[maybe_unused]] float q_scale = 1.f;
    const int last_key = limits && r < rows ? max(qp, min(key_limit[q0 + r], kv_limit - 1)) : qp;
    if constexpr (KV4) {
      // Q, which these warps have the time to bring.  (Eight loads of a thread at a time: all 16 at D = 256 took 7300 clocks, these
      // 3900.)  Queries of ordinary size enter as they are: fp16 holds bf16 from 6e-5 on, and is off by 2^-25 below.
      constexpr int kThreadsQ = kSoftmaxWarps * 32, kLanes = D / 8, kAhead = kLanes * kQRows / kThreadsQ < 8 ? kLanes * kQRows / kThreadsQ : 8;
      uint32_t least = 0x3f803f80u, most = 0u;   // of the largest of every four values that a thread has in hand; of all
#pragma unroll 1
      for (int i0 = threadIdx.x; i0 < kQRows * kLanes; i0 += kAhead * kThreadsQ) {
        uint4 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int i = i0 + k * kThreadsQ, row = i / kLanes, c = i % kLanes;       // (rows behind the last one are ones)
          v[k] = row < rows ? __ldg(reinterpret_cast<const uint4*>(a.q + (static_cast<size_t>(q0 + row) * a.Hq + hq) * D + c * 8)) : make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int i = i0 + k * kThreadsQ, row = i / kLanes, c = i % kLanes;
          StoreQuery(Qs + (c >> 3) * (kQRows * 128) + Sw128(row, c & 7), v[k], 1.f);
          const uint32_t top = MaxAbs2(MaxAbs2(v[k].x, v[k].y), MaxAbs2(v[k].z, v[k].w));
          least = MinAbs2(least, top);
          most = MaxAbs2(most, top);
        }
      }
      least &= 0x7fff7fffu;
      most &= 0x7fff7fffu;
      // (2^-12 at least among every four, 2^15 at most)
      if (!__all_sync(0xffffffffu, min(least >> 16, least & 0xffffu) >= 0x3980u && max(most >> 16, most & 0xffffu) <= 0x4700u))
        ScaleQueries<D>(Qs, ctl->q_scale, a.q + (static_cast<size_t>(q0) * a.Hq + hq) * D, static_cast<size_t>(a.Hq) * D, rows, score_scale);
      ptx::FenceProxyAsyncShared();
      join();
      __syncwarp();                              // (the others' arrivals came before the stores: they say nothing of this warp's lanes)
      if (lane == 0) ptx::MbarArriveRemote(ptx::MapToRank(ptx::SmemAddr(&ctl->q_full), 0));
      asm volatile("bar.sync 7, %0;" ::"n"((kSoftmaxWarps + kConvWarps) * 32) : "memory");      // the rows' factors are there, and that of the keys
      q_scale = ctl->q_scale[r] * ctl->k_back;
    }
    const uint32_t t_lane = tbase + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t p_full = ptx::MapToRank(ptx::SmemAddr(&ctl->p_full[0]), 0);
    float m_used = -INFINITY, l_run = 0.f;
    bool ok = true;
    // (both warps of a row reach every one of these, also after a wait that ran out)
    auto exchange = [&](int parity, float mine) -> float {
      ctl->row[parity][half][r] = mine;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory");
      return ctl->row[parity][half ^ 1][r];
    };
    for (int j = 0; j < ntiles; ++j) {
      const int b = j & 1;
      const uint32_t ph = static_cast<uint32_t>(j >> 1) & 1u;
      const uint32_t scol = t_lane + kSCol + b * kKvTile + half * 64;
      if (ok) ok = ptx::WarpMbarWait(&ctl->s_full[b], ph, abort_flag, 6);
      uint32_t s0[32], s1[32];
      float mx = -INFINITY;
      if (ok) {
        ptx::TcFenceAfter();
        ptx::TmemLoad32x32(scol, s0);
        ptx::TmemLoad32x32(scol + 32, s1);
        ptx::TmemLoadWait();
        const int kv0 = (tile0 + j) * kKvTile, k_lo = kv0 + half * 64;
        // tiles that reach past the row's own position (or start before its window) need the mask
        if ((kv0 + kKvTile - 1 > a.pos0 + q0) || (a.window > 0 && kv0 < a.pos0 + q0 + kQRows - a.window) || limits) {
          const int lo = a.window > 0 ? qp - a.window : -1;         // visible: lo < kp <= qp
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const int k0 = k_lo + c, k1 = k_lo + 32 + c;
            if (!(k0 <= last_key && k0 > lo)) s0[c] = 0xff800000u;  // -inf
            if (!(k1 <= last_key && k1 > lo)) s1[c] = 0xff800000u;
          }
        }
        float mx2 = -INFINITY;
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          mx = fmaxf(mx, fmaxf(__uint_as_float(s0[c]), __uint_as_float(s1[c])));
          mx2 = fmaxf(mx2, fmaxf(__uint_as_float(s0[c + 1]), __uint_as_float(s1[c + 1])));
        }
        mx = fmaxf(mx, mx2);
        if constexpr (KV4) mx *= q_scale;
      }
      mx = fmaxf(mx, exchange(b, mx));
      if (!ok) continue;
      // lazy rescale: adopt a new maximum only when some row of the warp has drifted by more than the step
      if (__any_sync(0xffffffffu, mx > m_used + kRescaleStep)) {
        const float m_new = fmaxf(m_used, mx);
        if (j > 0) {
          // every P V issued so far must have landed before O is touched; each warp takes half of the columns
          ok = ptx::WarpMbarWait(&ctl->pv_done[b ^ 1], static_cast<uint32_t>((j - 1) >> 1) & 1u, abort_flag, 7);
          if (!ok) continue;
          ptx::TcFenceAfter();
          const float f = (m_used == -INFINITY) ? 0.f : exp2f(m_used - m_new);
          l_run *= f;
#pragma unroll 1
          for (int c0 = half * (D / 2); c0 < (half + 1) * (D / 2); c0 += 16) {
            uint32_t o[16];
            ptx::TmemLoad32x16(t_lane + c0, o);
            ptx::TmemLoadWait();
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
            ptx::TmemStore32x16(t_lane + c0, o);
          }
          ptx::TmemStoreWait();
        }
        m_used = m_new;
      }
      // P = 2^(S - m), fp16 pairs (k, k+1) per column
      float sum = 0.f, sum2 = 0.f;
      const float mref = (m_used == -INFINITY) ? 0.f : m_used;
      auto probabilities = [&](const uint32_t (&sv)[32], uint32_t col) {
        uint32_t p[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const float x0 = __uint_as_float(sv[2 * c]), x1 = __uint_as_float(sv[2 * c + 1]);
          const float e0 = Exp2Approx(KV4 ? fmaf(x0, q_scale, -mref) : x0 - mref), e1 = Exp2Approx(KV4 ? fmaf(x1, q_scale, -mref) : x1 - mref);
          sum += e0;
          sum2 += e1;
          const __half2 h = __floats2half2_rn(e0, e1);
          p[c] = *reinterpret_cast<const uint32_t*>(&h);
        }
        ptx::TmemStore32x16(col, p);
      };
      probabilities(s0, scol);
      probabilities(s1, scol + 16);
      l_run += sum + sum2;
      ptx::TmemStoreWait();
      ptx::TcFenceBefore();
      __syncwarp();
      if (lane == 0) ptx::MbarArriveRemote(p_full + b * 8);
    }
    // ---------------- epilogue: O / l, output gate, bf16 rows; each warp half of the columns ----------------
    const float l = l_run + exchange(ntiles & 1, l_run);
    if constexpr (KV4) {
      // (a share of keys leaves its maximum and sum, NaN where a wait ran out; the rows follow below)
      if (half == 0) ctl->inv[r] = l == 0.f ? 0.f : 1.f / l;
      if (partial && r < rows && half == 0)
        a.part_ml[(static_cast<size_t>(blockIdx.z) * a.T + q0 + r) * a.Hq + hq] = make_float2(ok ? m_used : 0.f, ok ? l : __uint_as_float(0x7fc00000u));
    } else {
      if (ok && a.gated) ok = ptx::WarpMbarWait(&ctl->gates, 0, abort_flag, 10);
      if (ok) ok = ptx::WarpMbarWait(&ctl->o_final, 0, abort_flag, 9);
    }
    if constexpr (!KV4) if (ok) {
      ptx::TcFenceAfter();
      const float inv = (l > 0.f ? 1.f / l : 0.f) * a.v_descale[hkv];
      // a lane's half row, staged where Q (first half) or V (second) was and sent off as one copy
      constexpr int kHalfRow = D / 2 * 2, kStageRow = kHalfRow + 16;
      static_assert(kQRows * kStageRow <= kQBytes && kQRows * kStageRow <= 2 * kVBytes, "the output tile fits");
      unsigned char* stage = (half == 0 ? Qs : Vs) + r * kStageRow;
#pragma unroll 1
      for (int c0 = 0; c0 < D / 2; c0 += 32) {
        uint32_t o[32];
        ptx::TmemLoad32x32(t_lane + half * (D / 2) + c0, o);
        ptx::TmemLoadWait();
        if (r < rows) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float x[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) x[c] = __uint_as_float(o[8 * v + c]) * inv;
            if (a.gated) {
              const uint4 g = *reinterpret_cast<const uint4*>(Ks + GateChunk<D>(r, (half * (D / 2) + c0) / 8 + v));
              const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                x[2 * c] *= Sigmoid(BfLo(gw[c]));
                x[2 * c + 1] *= Sigmoid(BfHi(gw[c]));
              }
            }
            *reinterpret_cast<uint4*>(stage + (c0 + 8 * v) * 2) =
                make_uint4(PackBf16(x[0], x[1]), PackBf16(x[2], x[3]), PackBf16(x[4], x[5]), PackBf16(x[6], x[7]));
          }
        }
      }
      ptx::FenceProxyAsyncShared();
      if (r < rows) {
        ptx::BulkStore(a.out + (static_cast<size_t>(q0 + r) * a.Hq + hq) * D + half * (D / 2), ptx::SmemAddr(stage), kHalfRow);
        ptx::BulkStoreCommit();
        ptx::BulkStoreWait();
      }
    }
  }

  if constexpr (KV4) {
    // ---------------- epilogue of the 4-bit cache: the sums to shared memory as they are, then whole rows through 1 / l and gate ----------------
    if (warp != kMmaWarp) {
      const int worker = warp < kMmaWarp ? threadIdx.x : threadIdx.x - 32;
      // eight columns of every kStep-th row: `piece` of the row's, `col` of its half's
      constexpr int kRowPieces = D / 8, kWorkers = (kSoftmaxWarps + kConvWarps) * 32, kStep = kWorkers / kRowPieces, kPieces = kQRows / kStep;
      static_assert(kStep % 8 == 0, "a worker's rows lie alike in shared memory");
      const int piece = worker % kRowPieces, row0 = worker / kRowPieces, col = piece % (kRowPieces / 2);
      uint4 gate[kPieces];                       // on their way while the sums are
      if (a.gated && !partial) {
        const __nv_bfloat16* at = a.qg + ((static_cast<size_t>(q0 + row0) * a.Hq + hq) * 2 + 1) * D + piece * 8;
#pragma unroll
        for (int k = 0; k < kPieces; ++k, at += static_cast<size_t>(kStep) * a.Hq * 2 * D)
          gate[k] = row0 + k * kStep < rows ? __ldg(reinterpret_cast<const uint4*>(at)) : make_uint4(0u, 0u, 0u, 0u);
      }
      asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
      ptx::WarpMbarWait(&ctl->o_final, 0, abort_flag, 9);
      ptx::TcFenceAfter();
      // Columns of the first half lie where Q was, of the second where V was (the products have read both): rows of 2 D bytes each, every
      // second four columns in their second half, places permuted so that the lanes of rows and those of columns meet all banks.
      auto place = [&](int row, int four) { return row * 2 * D + ((((four >> 1) + (four & 1) * (D / 16)) ^ (row & 7)) << 4); };
      const int part = worker >> 7, r = (warp & 3) * 32 + lane;              // part: a quarter of the columns
      const uint32_t t_part = tbase + (static_cast<uint32_t>((warp & 3) * 32) << 16) + part * (D / 4);
      constexpr int kCols = D / 4 < 32 ? D / 4 : 32;
#pragma unroll
      for (int c0 = 0; c0 < D / 4; c0 += kCols) {
        uint32_t o[kCols];
        if constexpr (kCols == 32) ptx::TmemLoad32x32(t_part + c0, o);
        else ptx::TmemLoad32x16(t_part + c0, o);
        ptx::TmemLoadWait();
#pragma unroll
        for (int v = 0; v < kCols / 4; ++v)
          *reinterpret_cast<uint4*>((part < 2 ? Qs : Vs) + place(r, ((part & 1) * (D / 4) + c0) / 4 + v)) = make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
      }
      asm volatile("bar.sync 5, %0;" ::"n"(kWorkers) : "memory");
      const bool ran_out = *abort_flag != 0;          // a wait did: the rows are NaN, never what the buffers held
      const unsigned char* from = piece < kRowPieces / 2 ? Qs : Vs;
      const unsigned char *lo_at = from + place(row0, 2 * col), *hi_at = from + place(row0, 2 * col + 1);
      const size_t first = static_cast<size_t>(q0 + row0) * a.Hq + hq, row_step = static_cast<size_t>(kStep) * a.Hq * D;
      __nv_bfloat16* out = a.out + first * D + piece * 8;
      const float back = ctl->v_back[piece >> 3];
      float* sums = partial ? a.part_acc + (static_cast<size_t>(blockIdx.z) * a.T * a.Hq + first) * D + piece * 8 : nullptr;
#pragma unroll
      for (int k = 0; k < kPieces; ++k) {
        const int row = row0 + k * kStep;
        if (row >= rows) break;
        float4 lo = *reinterpret_cast<const float4*>(lo_at + k * kStep * 2 * D), hi = *reinterpret_cast<const float4*>(hi_at + k * kStep * 2 * D);
        if (ran_out || (ctl->nan_groups[row] >> (piece >> 3) & 1) != 0) lo.x = lo.y = lo.z = lo.w = hi.x = hi.y = hi.z = hi.w = __uint_as_float(0x7fc00000u);
        if (partial) {
          *reinterpret_cast<float4*>(sums + k * row_step) = make_float4(lo.x * back, lo.y * back, lo.z * back, lo.w * back);
          *reinterpret_cast<float4*>(sums + k * row_step + 4) = make_float4(hi.x * back, hi.y * back, hi.z * back, hi.w * back);
        } else {
          const float inv = ctl->inv[row];
          float x[8] = {lo.x * inv, lo.y * inv, lo.z * inv, lo.w * inv, hi.x * inv, hi.y * inv, hi.z * inv, hi.w * inv};
#pragma unroll
          for (int c = 0; c < 8; ++c) x[c] *= back;
          if (a.gated) {
            const uint32_t g[4] = {gate[k].x, gate[k].y, gate[k].z, gate[k].w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              x[2 * c] *= SigmoidApprox(BfLo(g[c]));
              x[2 * c + 1] *= SigmoidApprox(BfHi(g[c]));
            }
          }
          *reinterpret_cast<uint4*>(out + k * row_step) = make_uint4(PackBf16(x[0], x[1]), PackBf16(x[2], x[3]), PackBf16(x[4], x[5]), PackBf16(x[6], x[7]));
        }
      }
    }
  }

  // ---------------- teardown ----------------
  ptx::TcFenceBefore();
  __syncthreads();
  if (*abort_flag != 0) {
    if (threadIdx.x == 0 && a.status != nullptr) atomicCAS(a.status, 0, 600 + *abort_flag);
  }
  ptx::ClusterSync();                                 // neither CTA leaves or frees tensor memory while the other still uses it
  if (warp == kMmaWarp) {
    ptx::TcFenceAfter();
    ptx::TmemDeallocPair(tbase, kTmemCols);
  }
}

// The shares of split keys joined: D / 4 threads a row, its gate and its rounding.
template <int D>
__global__ void __launch_bounds__(256) JoinKv4Kernel(Kv4Args a) {
  PdlEnter();
  constexpr int kRow = D / 4;
  const long long row = static_cast<long long>(blockIdx.x) * (256 / kRow) + threadIdx.x / kRow, rows = static_cast<long long>(a.T) * a.Hq;
  if (row >= rows) return;
  const int col = threadIdx.x % kRow * 4;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int z = 0; z < a.splits; ++z) m = fmaxf(m, a.part_ml[z * rows + row].x);
  for (int z = 0; z < a.splits; ++z) {
    const float2 x = a.part_ml[z * rows + row];
    if (x.x == -INFINITY && x.y == 0.f) continue;               // (no key of that share is seen; it may have written nothing else)
    const float f = x.x == -INFINITY ? 1.f : exp2f(x.x - m);    // (-inf with a sum: its scores were NaN, and so is the sum)
    const float4 v = __ldcs(reinterpret_cast<const float4*>(a.part_acc + (z * rows + row) * D + col));
    l = fmaf(f, x.y, l);
    o.x = fmaf(f, v.x, o.x);
    o.y = fmaf(f, v.y, o.y);
    o.z = fmaf(f, v.z, o.z);
    o.w = fmaf(f, v.w, o.w);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  if (a.gated) {
    const uint32_t* gate = reinterpret_cast<const uint32_t*>(a.qg + row * 2 * D + D + col);
    o.x *= Sigmoid(BfLo(gate[0]));
    o.y *= Sigmoid(BfHi(gate[0]));
    o.z *= Sigmoid(BfLo(gate[1]));
    o.w *= Sigmoid(BfHi(gate[1]));
  }
  *reinterpret_cast<uint2*>(a.out + row * D + col) = make_uint2(PackBf16(o.x, o.y), PackBf16(o.z, o.w));
}

template <int D, bool KV4 = false>
int LaunchTc(const Args<KV4>& a, cudaStream_t s) {
  constexpr int NS = D / 64;
  // kClusterAlone: so much of an SM's shared memory that no other CTA shares the SM whose cluster may wait with tensor memory in its
  // hands (sm100_ptx.cuh).  More would cost L1: 8192 rows of 32 heads of 128 columns take 808 us with 131 KB, 821 with 156, 878 with 227.
  constexpr size_t kSmem = NS * kQRows * 128 + 2 * NS * kHalfTile * 128 + 2 * D * 128 + sizeof(std::conditional_t<KV4, Kv4Control, Control>) + 1024;
  constexpr size_t smem = kSmem > ptx::kClusterAlone ? kSmem : ptx::kClusterAlone;
  auto kern = AttnPrefillTcKernel<D, KV4>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return static_cast<int>(e);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = a.by_head ? dim3(a.Hq, (a.T + kQRows - 1) / kQRows) : dim3(2 * a.Hq, (a.T + 2 * kQRows - 1) / (2 * kQRows));
  if constexpr (KV4) cfg.gridDim.z = a.splits;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = KV4 && g_use_pdl ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e != cudaSuccess) return static_cast<int>(e);
  if constexpr (KV4) {
    if (a.splits > 1) {
      constexpr int kPer = 256 / (D / 4);
      const int rc = LaunchPdl(JoinKv4Kernel<D>, dim3(static_cast<unsigned>((static_cast<long long>(a.T) * a.Hq + kPer - 1) / kPer)), dim3(256), 0, s, a);
      if (rc) return rc;
    }
  }
  return FinishLaunch();
}

}  // namespace
}  // namespace r4dxb

using namespace r4dxb;

/* Same contract as r4dxb_attn_prefill (flags bit 0: sigmoid output gate, bits 1..: sliding-window length), for head
   dimensions 128 and 256.  status: device word that receives 600 + role code if a bounded wait ran out. */
extern "C" int r4dxb_attn_prefill_tc(const void* q, const void* qg, const void* cache, const int* block_table,
                                     const float* k_descale, const float* v_descale, void* out, int T, int Hq, int Hkv, int D,
                                     int pos0, int flags, int* status, void* stream) {
  if (T < 1 || Hq % Hkv || (D != 256 && D != 128)) return R4DXB_BAD_ARG;
  TcArgs a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.qg = static_cast<const __nv_bfloat16*>(qg);
  a.cache = static_cast<const uint8_t*>(cache);
  a.block_table = block_table;
  a.k_descale = k_descale;
  a.v_descale = v_descale;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.pos0 = pos0; a.gated = flags & 1; a.window = flags >> 1;
  a.by_head = Hq / Hkv % 2 == 0;
  a.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return D == 256 ? LaunchTc<256>(a, s) : LaunchTc<128>(a, s);
}

/* The same over the 4-bit cache (kv4.cuh), head dimensions 64, 128 and 256; key_limit as for r4dxb_attn_prefill_ex.  splits > 1: the keys of a row
   tile are shared by so many pairs; scratch: splits * T * Hq * (D + 2) floats, 16-byte aligned. */
extern "C" int r4dxb_attn_prefill_kv4(const void* q, const void* qg, const void* cache, const int* block_table, int table_length, int pool, void* out,
                                      int T, int Hq, int Hkv, int D, int pos0, int window, const int* key_limit, int splits, float* scratch, int* status,
                                      void* stream) {
  if (splits < 1 || splits > 64 || (splits > 1 && scratch == nullptr) || reinterpret_cast<uintptr_t>(scratch) & 15) return R4DXB_BAD_ARG;
  if (T < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || (D != 64 && D != 128 && D != 256) || pos0 < 0 || pos0 > 0x7fffffff - T - kKvTile || window < 0 ||
      table_length < 1 || pos0 > static_cast<long long>(table_length) * kv4::kBlock || pool < 1 || q == nullptr || cache == nullptr || block_table == nullptr || out == nullptr)
    return R4DXB_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(qg)) & 15)
    return R4DXB_BAD_ARG;
  if (Hq > 32767 || (T + kQRows - 1) / kQRows > 65535) return R4DXB_TOO_LARGE;
  Kv4Args a = {};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.qg = static_cast<const __nv_bfloat16*>(qg);
  a.cache = static_cast<const uint8_t*>(cache);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.pos0 = pos0; a.gated = qg != nullptr; a.window = window;
  a.by_head = Hq / Hkv % 2 == 0;
  a.status = status;
  a.table = {block_table, table_length, pool};
  a.key_limit = key_limit;
  a.splits = splits;
  a.part_acc = scratch;
  a.part_ml = reinterpret_cast<float2*>(scratch + static_cast<size_t>(splits) * T * Hq * D);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return D == 256 ? LaunchTc<256, true>(a, s) : (D == 128 ? LaunchTc<128, true>(a, s) : LaunchTc<64, true>(a, s));
}
