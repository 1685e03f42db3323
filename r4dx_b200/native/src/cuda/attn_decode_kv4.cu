// Attention of few query rows (decode steps, speculative windows, batches of one row a sequence) over the 4-bit paged cache (kv4.cuh).
//
// Split-KV: a CTA has 8 NT query rows of a kv head (of the G = rows x query heads per kv head) and a share of the sequence's blocks; each
// of its warps walks blocks of its own, which arrive as one bulk copy per block into the warp's ring of shared memory.  Per block
//   scores   S^T[16 tokens x 8 rows] = K Q^T on mma.m16n8k16 (fp16): A = the codes as they lie, since four bits at the bottom of a half are
//            the subnormal n 2^-24 and four bits above them n 2^-20: one AND for two codes, and no conversion at all.  B = the query rows times
//            2^4 (1 under the codes that carry a 16), exact down to 2^-17 and off by 2^-25 below; where some are above 2^11, or eight neighbours
//            below 2^-12, each row times the power of two that brings its largest value to 2^14 .. 2^15.  (That for every call: 0.2 us.)
//            A group gives 2^-24 sum q n; then s (that) in fp32.
//            sum_g lo sum(q): one product of the pairs as they lie (bf16) with the sums in two parts of bf16 (four at D = 64): 2^-17 of them is
//            lost, which only keys of thousands whose products cancel would show.
//   softmax  running maximum per row in the log2 domain, moved only when a score is more than 8 above it (p <= 2^8), so that most blocks
//            need no exchange between lanes; sums in fp32 per lane.
//   values   O^T[D x 8 rows] += n (p s):  A = codes of token pairs, again as subnormals; B = p s times a power of two of the warp and the group of
//            channels, rounded to fp16, turned from scores' to operand order with movmatrix.  The power is made smaller where a product reaches
//            2^7 (to 1), larger again where all rows' maxima rise, so it follows products, not scales: loud tokens without weight
//            leave it alone.  Off by 2^-12 of a product, or by 2^-25 of the largest of the group among the rows of the tile.  sum p lo in fp32.
// The warps' results meet in shared memory; the splits' in the shared memory of a cluster of up to 16 CTAs, or, for long tables, in a second
// kernel.  A sequence short enough for one CTA is finished by it.
// A row with no visible token (position -1) gives zeros; a block that the table or pool does not have gives NaN to the rows that see it.
//
// What bounds it: unpacking.  One token over 131071 keys: 24 heads over 4 of 256 35 us, 32 over 8 of 128 36 us, 4.3 TB/s of a copy's 6.5, with the
// half-rate integer unit 50 / 53 % busy, the issue slots 49 / 55 %, the tensor pipe a quarter.  The first kernel, which made a number of every
// code before the products, took 68 us (32 over 8).  As many warps as the registers allow (8 at D = 256, 12 at 128) each with two blocks in work keep the units
// fed, more of them with fewer registers spill (D = 256, 12 warps: 37 us; D = 128, 14: 40).  Short tables are bound by start and merge: 8192 keys of the
// first 9.6 us, of which about 4 until the first scores and 2 for the second kernel; four rows (three row tiles) 13.
#include <atomic>
#include <type_traits>

#include "kv4.cuh"
#include "sm100_ptx.cuh"

namespace r4dxb {
namespace {

constexpr int kMaxCluster = 16;
constexpr float kRescaleStep = 8.f;
constexpr int kMostPower = 253;            // exponent of the largest power of two that p s is taken by: 2^126
constexpr float kUnit = 1.f / (1 << 24);       // of the scores before the softmax, from the codes
constexpr uint32_t kOrdinary = 131u;           // exponent of the power of two that queries of ordinary size are taken by: 2^4
constexpr float kNone = -3e38f;                // the maximum of a row that has seen nothing: finite, so that 2^(-inf - kNone) is 0

struct DecodeArgs {
  const __nv_bfloat16* q;      // [T, Hq, D]
  const __nv_bfloat16* qg;     // [T, Hq, 2 D], the gate behind (null: none)
  const uint8_t* cache;
  kv4::Table table;
  const int* positions;        // [T]; batched: one row each; null: pos0, pos0 + 1 ..
  const int* row_slot;         // batched: sequence of each row
  float* part_acc;             // [batch][Hkv][G][splits][D]
  float2* part_ml;             // [batch][Hkv][G][splits]
  __nv_bfloat16* out;          // [T, Hq, D]
  int* status;
  int T, Hq, Hkv, splits, slots, window;
  int chunk;                   // blocks of a sequence for which another CTA joins
  int pos0;
  int end;                     // first position behind the table: a row there or further on sees a block that there is not, and no other counts
  uint32_t per_token;          // 2^32 / (query heads per kv head), rounded up; 0: one query head
  // row r of a kv head's G = T Hq / Hkv belongs to token Row(r)
  __device__ __forceinline__ int Position(int t) const { return min(positions != nullptr ? positions[t] : pos0 + t, end); }
  __device__ __forceinline__ int Row(int r) const { return per_token != 0u ? static_cast<int>(__umulhi(static_cast<uint32_t>(r), per_token)) : r; }
};

// Rows of a CTA that takes many: what the registers allow.  Blocks are unpacked once for all of them.
template <int D>
constexpr int kWideTile = D == 256 ? 16 : 32;

// Warps of a CTA, blocks that a warp takes at a time and slots of so many in its ring, by head dimension and row tiles.
template <int D, int NT>
struct Plan {
  static constexpr int kWarps = D == 256 ? 8 : (D == 128 ? (NT == 4 ? 8 : 12) : (NT == 4 ? 12 : 8));
  static constexpr int kCtas = D == 64 && NT == 1 ? 2 : 1;
  static constexpr int kPair = NT == 1 ? 2 : 1;
  static constexpr int kStages = NT == 1 ? 2 : 4;
  static constexpr int kRows = 8 * NT;
  static constexpr int kRing = kWarps * kStages * kPair * kv4::Shape<D>::kRun;
  static constexpr int kStride = D + 4;                          // floats between rows of the merge
  static constexpr int kMerge = kWarps * kRows * kStride * 4;
  static constexpr int kQuery = NT * (D / 32) * 512;             // operand B of the scores
  static constexpr int kBase = kWarps * kRows * (D / 64) * 4;    // sum p lo of each warp, row and group
  static constexpr int kOut = kRows * D * 4;                     // a CTA's rows, for the other CTAs of its cluster
  static constexpr int kBody = kRing > kMerge + kBase + kOut ? kRing : kMerge + kBase + kOut;
  static constexpr int kSums = 2 * NT * (D / 32) * 8 * 4;        // of a row's query over 32 channels: sums, largest magnitudes
  static constexpr size_t kSmem = kBody + kQuery + kSums + kWarps * kStages * 8 + kWarps * kRows * 8 + kRows * 20 + 16;
  static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
};

// The blocks that the rows of a call may see and the number of CTAs that share them: one for every `chunk` blocks.
struct Span {
  int first, blocks, active;
  int position;                // of token `lane`, -1 beyond the last
};
__device__ __forceinline__ Span Visible(const DecodeArgs& a) {
  const int lane = threadIdx.x & 31;
  const int p = lane < a.T ? a.Position(lane) : -1;
  Span s;
  s.position = p;
  const int high = __reduce_max_sync(0xffffffffu, p), low = __reduce_min_sync(0xffffffffu, p < 0 ? 0x7fffffff : p);
  s.first = a.window > 0 && high >= 0 ? max(0, low - a.window + 1) / kv4::kBlock : 0;
  s.blocks = high >= 0 ? high / kv4::kBlock + 1 - s.first : 0;
  s.active = max(1, min(a.splits, static_cast<int>((static_cast<unsigned>(s.blocks) + a.chunk - 1) / a.chunk)));
  return s;
}

struct Frag {
  float x[4];
};
__device__ __forceinline__ Frag MmaF16(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const Frag& c) {
  Frag d;
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d.x[0]), "=f"(d.x[1]), "=f"(d.x[2]), "=f"(d.x[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c.x[0]), "f"(c.x[1]), "f"(c.x[2]), "f"(c.x[3]));
  return d;
}
__device__ __forceinline__ Frag MmaBf16(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const Frag& c) {
  Frag d;
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d.x[0]), "=f"(d.x[1]), "=f"(d.x[2]), "=f"(d.x[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c.x[0]), "f"(c.x[1]), "f"(c.x[2]), "f"(c.x[3]));
  return d;
}
__device__ __forceinline__ uint32_t Transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t Bits(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }
__device__ __forceinline__ uint32_t PackHalf(float lo, float hi) { return Bits(__floats2half2_rn(lo, hi)); }
// codes of the lowest bits of a word's halves (n 2^-24 as fp16), of the next four (n 2^-20)
__device__ __forceinline__ uint32_t Codes(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t Codes16(uint32_t w) { return w & 0x00f000f0u; }

template <int N>
__device__ __forceinline__ void LoadWords(const uint32_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *p;
  }
}

// Four columns of an output row, through its gate.
__device__ __forceinline__ void StoreRow(const DecodeArgs& a, size_t row, int D, int col, float4 o) {
  if (a.qg != nullptr) {
    const uint2 gate = *reinterpret_cast<const uint2*>(a.qg + row * 2 * D + D + col);
    o.x *= Sigmoid(BfLo(gate.x));
    o.y *= Sigmoid(BfHi(gate.x));
    o.z *= Sigmoid(BfLo(gate.y));
    o.w *= Sigmoid(BfHi(gate.y));
  }
  *reinterpret_cast<uint2*>(a.out + row * D + col) = make_uint2(PackBf16(o.x, o.y), PackBf16(o.z, o.w));
}

template <int D, int NT, bool CLUSTER>
__global__ void __launch_bounds__(Plan<D, NT>::kWarps * 32, Plan<D, NT>::kCtas) DecodeKv4Kernel(DecodeArgs a) {
  PdlEnter();
  using S = kv4::Shape<D>;
  using P = Plan<D, NT>;
  constexpr int NG = S::kGroups, NJ = D / 32, kWarps = P::kWarps, kRows = P::kRows, kStages = P::kStages, kPair = P::kPair, kSlot = kPair * S::kRun;
  extern __shared__ __align__(128) unsigned char smem[];
  uint4* query = reinterpret_cast<uint4*>(smem + P::kBody);                     // [row tile][32 channels][lane]
  float* sums = reinterpret_cast<float*>(smem + P::kBody + P::kQuery);          // [row tile][32 channels][row]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + P::kBody + P::kQuery + P::kSums);
  float4* shared_ml = reinterpret_cast<float4*>(bars + kWarps * kStages);       // [rows]: maximum and sum of this CTA
  float2* ml = reinterpret_cast<float2*>(shared_ml + kRows);                    // [warps][rows]
  int* nan_groups = reinterpret_cast<int*>(ml + kWarps * kRows);                // [rows]: groups in which the row sees a NaN among the values
  volatile int* abort_flag = nan_groups + kRows;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x, hkv = blockIdx.y % a.Hkv, row0 = blockIdx.y / a.Hkv * kRows, seq = blockIdx.z;
  bool known = true;           // the sequence has a table
  if (a.row_slot != nullptr) {
    a.q += static_cast<size_t>(seq) * a.Hq * D;
    a.out += static_cast<size_t>(seq) * a.Hq * D;
    if (a.qg != nullptr) a.qg += static_cast<size_t>(seq) * a.Hq * 2 * D;
    a.positions += seq;
    const int slot = a.row_slot[seq];
    known = slot >= 0 && slot < a.slots;
    a.table.entries += static_cast<size_t>(known ? slot : 0) * a.table.length;
  }
  const int gqa = a.Hq / a.Hkv, G = gqa * a.T;
  // A warp lays out 32 channels of a row tile's queries, one or two times; they are on their way while positions and table are.
  constexpr int kTasks = (NT * NJ + kWarps - 1) / kWarps;
  uint4 own_query[kTasks];
#pragma unroll
  for (int i = 0; i < kTasks; ++i) {
    const int task = warp + i * kWarps, r = row0 + task / NJ * 8 + g, t = a.Row(r);
    own_query[i] = task < NT * NJ && r < G ? *reinterpret_cast<const uint4*>(a.q + (static_cast<size_t>(t) * a.Hq + hkv * gqa + r - t * gqa) * D + task % NJ * 32 + 8 * c)
                                           : make_uint4(0u, 0u, 0u, 0u);
  }
  const Span span = Visible(a);
  if (split >= (CLUSTER && span.active > 1 ? a.splits : span.active)) return;       // (a cluster stays together, its CTAs without blocks merge too)
  const int per = (span.blocks + span.active - 1) / span.active;
  // the CTA's blocks b0 .. b1 - 1 go around its warps, kPair at a time where there are more of them than warps
  const int b0 = span.first + split * per, b1 = min(span.first + span.blocks, b0 + per);
  const int take = b1 - b0 > kWarps ? kPair : 1, mine = b0 + warp * take, turn = kWarps * take;
  const int steps = b1 > mine ? (b1 - mine + turn - 1) / turn : 0;

  unsigned char* ring = smem + warp * kStages * kSlot;
  uint64_t* full = bars + warp * kStages;
  const uint32_t ring_at = ptx::SmemAddr(ring), full_at = ptx::SmemAddr(full);
  const uint8_t* head_run = a.cache + static_cast<size_t>(hkv) * S::kRun;
  const size_t block_bytes = static_cast<size_t>(a.Hkv) * S::kRun;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) ptx::MbarInit(full + i, 1);
    ptx::MbarFenceInit();
  }
  if (threadIdx.x == 0) *abort_flag = 0;
  if (threadIdx.x < kRows) nan_groups[threadIdx.x] = 0;
  __syncwarp();

  // ---- copies: the blocks mine + i turn .. of step i into slot i % kStages ----
  uint32_t missing = 0u;                         // a bit per block of the ring: there is none such
  int entry = -1;
  auto issue = [&](int i, int slot) {
    if ((i * kPair & 31) == 0) {
      const int k = i + lane / kPair, b = mine + k * turn + lane % kPair;
      entry = lane % kPair < take && b < b1 && known ? a.table.BlockAt(b) : -1;
    }
    int blk[kPair], copies = 0;
#pragma unroll
    for (int h = 0; h < kPair; ++h) {
      blk[h] = __shfl_sync(0xffffffffu, entry, (i * kPair + h) & 31);
      copies += blk[h] >= 0;
      const uint32_t bit = 1u << (slot * kPair + h);
      missing = blk[h] < 0 ? missing | bit : missing & ~bit;
    }
    if (lane == 0) {
      ptx::MbarArriveExpectTxAt(full_at + slot * 8, copies * S::kRun);
#pragma unroll
      for (int h = 0; h < kPair; ++h)
        if (blk[h] >= 0) ptx::BulkLoadAt(ring_at + slot * kSlot + h * S::kRun, head_run + blk[h] * block_bytes, S::kRun, full_at + slot * 8);
    }
  };
  for (int i = 0; i < min(steps, kStages); ++i) issue(i, i);

  // ---- query rows: operand B (row g; channels 32 j + 8 c .. in the order of the codes) and its sums ----
  auto position = [&](int r) {
    const int p = __shfl_sync(0xffffffffu, span.position, r < G ? a.Row(r) : 0);
    return r < G ? p : -1;
  };
  uint32_t tops[kTasks];                         // the largest magnitude of eight channels, as the bits of bf16
  bool ordinary = true;
#pragma unroll
  for (int i = 0; i < kTasks; ++i) {
    const uint4 v = own_query[i];
    const uint32_t top = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
    tops[i] = max(top >> 16, top & 0xffffu);
    const int task = warp + i * kWarps;
    if (task < NT * NJ && row0 + task / NJ * 8 + g < G) ordinary = ordinary && tops[i] - 0x3980u <= 0x4500u - 0x3980u;      // 2^-12 .. 2^11
  }
  auto lay_out = [&](auto exponent) {            // of a row's power of two, as of a float
#pragma unroll
    for (int i = 0; i < kTasks; ++i) {
      const int task = warp + i * kWarps;
      if (task < NT * NJ) {
        const uint4 v = own_query[i];
        const float power = __uint_as_float(exponent(task / NJ * 8 + g) << 23), power16 = power * 0.0625f;
        // channels i and i + 4 for i = 0 .. 3; every second pair meets codes that carry a factor 16
        const float x[8] = {BfLo(v.x), BfHi(v.x), BfLo(v.y), BfHi(v.y), BfLo(v.z), BfHi(v.z), BfLo(v.w), BfHi(v.w)};
        uint32_t b[4];
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          b[k] = PackHalf(x[k] * (k & 1 ? power16 : power), x[k + 4] * (k & 1 ? power16 : power));
          sum += x[k] + x[k + 4];
        }
        query[task * 32 + lane] = make_uint4(b[0], b[1], b[2], b[3]);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (c == 0) sums[task * 8 + g] = sum * power * kUnit;
      }
    }
  };
  lay_out([](int) { return kOrdinary; });
  const bool by_row = __syncthreads_or(!ordinary) != 0;
  uint32_t* row_tops = reinterpret_cast<uint32_t*>(sums + NT * NJ * 8);         // [row][32 channels]
  auto exponent_of = [&](int row) {
    uint32_t top = 0u;
#pragma unroll
    for (int j = 0; j < NJ; ++j) top = max(top, row_tops[row * NJ + j]);
    const uint32_t e = top >> 7;
    return e == 255u ? 127u : min(max(268u - e, 24u), 253u);      // to 2^14 .. 2^15 (infinite or NaN: as it is)
  };
  if (by_row) {
#pragma unroll
    for (int i = 0; i < kTasks; ++i) {
      const int task = warp + i * kWarps;
      uint32_t top = max(tops[i], __shfl_xor_sync(0xffffffffu, tops[i], 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (c == 0 && task < NT * NJ) row_tops[(task / NJ * 8 + g) * NJ + task % NJ] = top;
    }
    __syncthreads();
    lay_out(exponent_of);
    __syncthreads();
  }
  // operand B of sum_g lo sum(q): pairs (0, sum) in two (D = 256, 128) or four (64) parts of bf16
  uint32_t qpair[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float* of = sums + (nt * NJ + 2 * (c % NG)) * 8 + g;
    float rest = of[0] + of[8];
    float part = 0.f, next = 0.f;
#pragma unroll
    for (int k = 0; k <= 4 / NG; ++k) {
      const float b = __bfloat162float(__float2bfloat16_rn(rest));
      if (k == c / NG) part = b;
      if (k == c / NG + 1) next = b;
      rest -= b;
    }
    qpair[nt][0] = PackBf16(0.f, part);
    qpair[nt][1] = NG == 4 ? PackBf16(0.f, next) : 0u;
  }

  int pos[NT][2], p_min = 0x7fffffff, p_max = -1;
  float scale[NT][2];                            // of the rows' scores, to the log2 domain
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    pos[nt][0] = position(row0 + 8 * nt + 2 * c);
    pos[nt][1] = position(row0 + 8 * nt + 2 * c + 1);
#pragma unroll
    for (int r = 0; r < 2; ++r)
      scale[nt][r] = rsqrtf(static_cast<float>(D)) * 1.4426950408889634f / kUnit * __uint_as_float((254u - (by_row ? exponent_of(8 * nt + 2 * c + r) : kOrdinary)) << 23);
    // among the rows that there are, for blocks that all of them see whole
    const int r = row0 + 8 * nt + g, p = position(r);
    p_min = min(p_min, r < G ? p : 0x7fffffff);
    p_max = max(p_max, p);
  }
  p_min = __reduce_min_sync(0xffffffffu, p_min);
  p_max = __reduce_max_sync(0xffffffffu, p_max);
  auto sees = [&](int at, int kp) { return kp <= at && (a.window == 0 || kp > at - a.window); };

  float m[NT][2], l[NT][2];                      // rows 8 nt + 2 c, + 1: maximum in the log2 domain, sum over this lane's tokens
  Frag acc[NT][NG][4];
  float base[NT][NG][2];                         // sum p lo of this lane's tokens
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = kNone;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      base[nt][j][0] = base[nt][j][1] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[nt][j][e] = {{0.f, 0.f, 0.f, 0.f}};
    }
  }
  float power[NG];                               // what the groups' weights times scales are taken by
#pragma unroll
  for (int j = 0; j < NG; ++j) power[j] = __uint_as_float(static_cast<uint32_t>(kMostPower) << 23);

  // N consecutive blocks from token kp0 on, as they lie in the ring
  auto blocks = [&](auto count, uint32_t* const run, const int kp0) {
    constexpr int N = decltype(count)::value, kWords = S::kRun / 4, kValues = S::kPart / 4;
    const bool whole = kp0 + N * kv4::kBlock - 1 <= p_min && (a.window == 0 || kp0 > p_max - a.window);
    if (!whole) {
      // Value pairs that are no numbers, or of tokens that no row here sees (whose bytes may be anything), are zeros from here on: what
      // a row does not see has the weight 0, and 0 x NaN would reach it.  Rows that do see a NaN are noted.
      bool used = false;
      const int kp = kp0 + lane;
      for (int t = a.Row(row0); t <= a.Row(min(G, row0 + kRows) - 1); ++t) used |= sees(__shfl_sync(0xffffffffu, span.position, t), kp);
      if (lane < N * kv4::kBlock) {
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          uint32_t& pair = run[lane / kv4::kBlock * kWords + kValues + 2 * D + lane % kv4::kBlock * NG + j];
          const bool number = (pair & 0x7f80u) != 0x7f80u && (pair & 0x7f800000u) != 0x7f800000u;
          if (used && !number)
            for (int r = row0; r < min(G, row0 + kRows); ++r)
              if (sees(a.Position(a.Row(r)), kp)) atomicOr(nan_groups + r - row0, 1 << j);
          if (!used || !number) pair = 0u;
        }
      }
      ptx::FenceProxyAsyncShared();              // (the next copy into the slot comes after these stores)
      __syncwarp();
    }

    // ---- scores: tokens g (x[0], x[1]) and g + 8 (x[2], x[3]) of rows 2 c, 2 c + 1 ----
    Frag sc[N][NT];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const uint32_t* kw = run + n * kWords;
      uint32_t pa[NG], pb[NG];
      LoadWords<NG>(kw + 2 * D + g * NG, pa);
      LoadWords<NG>(kw + 2 * D + (g + 8) * NG, pb);
      const uint32_t mine_a = kw[2 * D + g * NG + c % NG], mine_b = kw[2 * D + (g + 8) * NG + c % NG];
      uint32_t ca[NJ], cb[NJ];
      if constexpr (D == 256) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = ((h ^ (g & 1)) * 16) + c * 4;
          const uint4 x = *reinterpret_cast<const uint4*>(kw + g * 32 + at), y = *reinterpret_cast<const uint4*>(kw + (g + 8) * 32 + at);
          ca[4 * h] = x.x; ca[4 * h + 1] = x.y; ca[4 * h + 2] = x.z; ca[4 * h + 3] = x.w;
          cb[4 * h] = y.x; cb[4 * h + 1] = y.y; cb[4 * h + 2] = y.z; cb[4 * h + 3] = y.w;
        }
      } else {
        LoadWords<NJ>(kw + g * (D / 8) + c * NJ, ca);
        LoadWords<NJ>(kw + (g + 8) * (D / 8) + c * NJ, cb);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        sc[n][nt] = MmaBf16(mine_a, mine_b, NG == 4 ? mine_a : 0u, NG == 4 ? mine_b : 0u, qpair[nt][0], qpair[nt][1], Frag{{0.f, 0.f, 0.f, 0.f}});
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        Frag s4[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s4[nt] = {{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t x = ca[2 * j + h], y = cb[2 * j + h], x8 = x >> 8, y8 = y >> 8;
          const uint32_t a0 = Codes(x), a1 = Codes(y), a2 = Codes16(x), a3 = Codes16(y), a4 = Codes(x8), a5 = Codes(y8), a6 = Codes16(x8), a7 = Codes16(y8);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4 b = query[(nt * NJ + 2 * j + h) * 32 + lane];
            s4[nt] = MmaF16(a0, a1, a2, a3, b.x, b.y, s4[nt]);
            s4[nt] = MmaF16(a4, a5, a6, a7, b.z, b.w, s4[nt]);
          }
        }
        const float sa = BfLo(pa[j]), sb = BfLo(pb[j]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          sc[n][nt].x[0] = fmaf(sa, s4[nt].x[0], sc[n][nt].x[0]);
          sc[n][nt].x[1] = fmaf(sa, s4[nt].x[1], sc[n][nt].x[1]);
          sc[n][nt].x[2] = fmaf(sb, s4[nt].x[2], sc[n][nt].x[2]);
          sc[n][nt].x[3] = fmaf(sb, s4[nt].x[3], sc[n][nt].x[3]);
        }
      }
    }
    if (!whole) {
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!sees(pos[nt][e & 1], kp0 + n * kv4::kBlock + g + (e >> 1) * 8)) sc[n][nt].x[e] = -INFINITY;
    }

    // ---- running maximum, powers of two of the groups, probabilities ----
    uint32_t pa[N][NG], pb[N][NG];
    bool move = false;
    float top[NT][2];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      LoadWords<NG>(run + n * kWords + kValues + 2 * D + g * NG, pa[n]);
      LoadWords<NG>(run + n * kWords + kValues + 2 * D + (g + 8) * NG, pb[n]);
    }
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      float largest = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n) largest = fmaxf(largest, fmaxf(BfLo(pa[n][j]), BfLo(pb[n][j])));
      move = move || largest * power[j] >= 128.f;                 // (a probability is 2^8 at most)
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[nt][r] = fmaxf(sc[0][nt].x[r], sc[0][nt].x[2 + r]);
#pragma unroll
        for (int n = 1; n < N; ++n) top[nt][r] = fmaxf(top[nt][r], fmaxf(sc[n][nt].x[r], sc[n][nt].x[2 + r]));
        top[nt][r] *= scale[nt][r];
        move = move || top[nt][r] > m[nt][r] + kRescaleStep;
      }
    if (__any_sync(0xffffffffu, move)) {
      float f[NT][2], keep = 0.f;                // what the rows' sums are taken by; the most of it among rows that have sums
      float pm[N][2];                            // the largest probabilities of tokens g, g + 8 among this lane's rows
#pragma unroll
      for (int n = 0; n < N; ++n) pm[n][0] = pm[n][1] = 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float t = fmaxf(m[nt][r], top[nt][r]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
          f[nt][r] = Exp2(m[nt][r] - t);
          const bool there = pos[nt][r] >= 0;    // (columns behind the last row have queries of zero and count for nothing)
          if (there && m[nt][r] != kNone) keep = fmaxf(keep, f[nt][r]);
          m[nt][r] = t;
          l[nt][r] *= f[nt][r];
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (there) pm[n][h] = fmaxf(pm[n][h], Exp2(fmaf(sc[n][nt].x[2 * h + r], scale[nt][r], -m[nt][r])));
        }
      // where the sums of all rows become small, the products that are added to them need not be
      keep = fmaxf(keep, __shfl_xor_sync(0xffffffffu, keep, 1));
      keep = fmaxf(keep, __shfl_xor_sync(0xffffffffu, keep, 2));
      const int grow = max(126 - static_cast<int>(__float_as_uint(keep) >> 23), 0);
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        float product = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) product = fmaxf(product, fmaxf(pm[n][0] * BfLo(pa[n][j]), pm[n][1] * BfLo(pb[n][j])));
        const int e = static_cast<int>(__reduce_max_sync(0xffffffffu, product < INFINITY ? __float_as_uint(product) : 0u) >> 23);
        const int old = static_cast<int>(__float_as_uint(power[j]) >> 23);
        int now = min(old + grow, kMostPower);
        if (e + now >= 254 + 7) now = max(254 - e, 1);            // a product of 2^7 or more: to 1 .. 2
        power[j] = __uint_as_float(static_cast<uint32_t>(now) << 23);
        const float other = __uint_as_float(static_cast<uint32_t>(min(max(127 + now - old, 0), 254)) << 23);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          base[nt][j][0] *= f[nt][0];
          base[nt][j][1] *= f[nt][1];
#pragma unroll
          for (int e4 = 0; e4 < 4; ++e4)
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[nt][j][e4].x[x] *= f[nt][x & 1] * other;
        }
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const uint32_t* vw = run + n * kWords + kValues;
      float p[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) p[nt][e] = Exp2(fmaf(sc[n][nt].x[e], scale[nt][e & 1], -m[nt][e & 1]));
        l[nt][0] += p[nt][0] + p[nt][2];
        l[nt][1] += p[nt][1] + p[nt][3];
      }

      // ---- values: tokens 2 c, 2 c + 1 and 8 more; of every 64 channels 8 g .. ----
      uint32_t va[NG], vb[NG], vc[NG], vd[NG];
      if constexpr (D == 256) {
        const int at = (g ^ (2 * c)) * 4;
        LoadWords<NG>(vw + (2 * c) * 32 + at, va);
        LoadWords<NG>(vw + (2 * c + 1) * 32 + at, vb);
        LoadWords<NG>(vw + (2 * c + 8) * 32 + at, vc);
        LoadWords<NG>(vw + (2 * c + 9) * 32 + at, vd);
      } else {
        const int unit = 2 * NG, at = D == 128 ? (g ^ (2 * c)) * unit : (g ^ ((c & 2) << 1)) * unit;
        uint32_t x[2 * NG], y[2 * NG];
        LoadWords<2 * NG>(vw + c * (D / 4) + at, x);
        LoadWords<2 * NG>(vw + (c + 4) * (D / 4) + at, y);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          va[j] = x[j]; vb[j] = x[NG + j];
          vc[j] = y[j]; vd[j] = y[NG + j];
        }
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const float sa = BfLo(pa[n][j]) * power[j], sb = BfLo(pb[n][j]) * power[j], la = BfHi(pa[n][j]), lb = BfHi(pb[n][j]);
        uint32_t w0[NT], w1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          w0[nt] = Transpose8x8(PackHalf(p[nt][0] * sa, p[nt][1] * sa));
          w1[nt] = Transpose8x8(PackHalf(p[nt][2] * sb, p[nt][3] * sb));
          base[nt][j][0] = fmaf(p[nt][0], la, fmaf(p[nt][2], lb, base[nt][j][0]));
          base[nt][j][1] = fmaf(p[nt][1], la, fmaf(p[nt][3], lb, base[nt][j][1]));
        }
        uint32_t t[4] = {__byte_perm(va[j], vb[j], 0x5410), __byte_perm(va[j], vb[j], 0x7632), __byte_perm(vc[j], vd[j], 0x5410), __byte_perm(vc[j], vd[j], 0x7632)};
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const uint32_t a0 = Codes(t[0]), a1 = Codes(t[1]), a2 = Codes(t[2]), a3 = Codes(t[3]);
          const uint32_t a4 = Codes16(t[0]), a5 = Codes16(t[1]), a6 = Codes16(t[2]), a7 = Codes16(t[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            acc[nt][j][e] = MmaF16(a0, a1, a2, a3, w0[nt], w1[nt], acc[nt][j][e]);
            acc[nt][j][e + 1] = MmaF16(a4, a5, a6, a7, w0[nt], w1[nt], acc[nt][j][e + 1]);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) t[k] >>= 8;
        }
      }
    }
  };

  bool ok = true;
  int i = 0, slot = 0;
  uint32_t phase = 0u;
#pragma unroll 1
  for (; i < steps; ++i) {
    if (!__all_sync(0xffffffffu, ptx::MbarTestWaitAt(full_at + slot * 8, phase))) {
      ok = ptx::WarpMbarWait(full + slot, phase, abort_flag, 1);
      __syncwarp();                              // (one lane has seen the copy done; a shuffle orders no memory for the others)
    }
    if (!ok) break;
    uint32_t* run = reinterpret_cast<uint32_t*>(ring + slot * kSlot);
    const int b = mine + i * turn, there = min(take, b1 - b);
    const uint32_t gone = missing >> (slot * kPair) & ((1u << there) - 1u);
    if (there == kPair && gone == 0u) {
      blocks(std::integral_constant<int, kPair>{}, run, b * kv4::kBlock);
    } else {
#pragma unroll 1
      for (int h = 0; h < there; ++h) {
        const int kp0 = (b + h) * kv4::kBlock;
        if (gone >> h & 1u) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 2; ++r)
              if (pos[nt][r] >= kp0 && (a.window == 0 || kp0 + kv4::kBlock - 1 > pos[nt][r] - a.window)) l[nt][r] = __int_as_float(0x7fc00000);
        } else if constexpr (kPair > 1) {
          blocks(std::integral_constant<int, 1>{}, run + h * (S::kRun / 4), kp0);
        }
      }
    }
    __syncwarp();                                // every lane has read the slot
    if (i + kStages < steps) issue(i + kStages, slot);
    if (++slot == kStages) {
      slot = 0;
      phase ^= 1u;
    }
  }
  if (!ok) {
    // a copy did not arrive in time: the rows are NaN, the status word says so, and the copies still under way are waited for
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) l[nt][0] = l[nt][1] = __int_as_float(0x7fc00000);
    if (lane == 0) {
      if (a.status != nullptr) atomicCAS(a.status, 0, 800 + *abort_flag);
      const long long t0 = clock64();
      for (int k = i; k < min(steps, i + kStages); ++k)
        while (!ptx::MbarTryWait(full + k % kStages, static_cast<uint32_t>(k / kStages) & 1u) && clock64() - t0 < ptx::kWaitClocks) {}
    }
    __syncwarp();
  }

  // ---- the lanes' sums of rows 2 c, 2 c + 1, then the warps' ----
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[nt][r] += __shfl_xor_sync(0xffffffffu, l[nt][r], o);
  __syncthreads();                               // the ring is read by no one any more
  float* merge = reinterpret_cast<float*>(smem);
  float* sums_lo = reinterpret_cast<float*>(smem + P::kMerge);                  // [warps][rows][groups]
  // warps that had blocks (the first ones)
  const int used = max(1, min(kWarps, (b1 - b0 + take - 1) / take));
  if (warp < used) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // sum p lo over the lanes g: each round halves the values that a lane still adds up, until lane g has the sum of its own one
      float v[2 * NG];
#pragma unroll
      for (int k = 0; k < 2 * NG; ++k) v[k] = base[nt][k >> 1][k & 1];
      int width = 16;
#pragma unroll
      for (int n = NG; n >= 1; n >>= 1, width >>= 1) {
#pragma unroll
        for (int k = 0; k < n; ++k) {
          const bool upper = lane & width;
          const float give = upper ? v[k] : v[k + n];
          v[k] = (upper ? v[k + n] : v[k]) + __shfl_xor_sync(0xffffffffu, give, width);
        }
      }
#pragma unroll
      for (; width >= 4; width >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], width);
      const int k = g / (4 / NG);
      sums_lo[(warp * kRows + 8 * nt + 2 * c + (k & 1)) * NG + (k >> 1)] = v[0];
      // (sixteen bytes of odd row pairs change places, so that the lanes of a store meet all banks)
      float* dst = merge + (warp * kRows + 8 * nt + 2 * c) * P::kStride + 8 * g;
      const int h0 = (c & 1) * 4, h1 = 4 - h0;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const float back = 16777216.f / power[j], back16 = back * 0.0625f;      // codes n 2^-24, n 2^-20
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const Frag(&o)[4] = acc[nt][j];
          float* at = dst + r * P::kStride + 64 * j;
          *reinterpret_cast<float4*>(at + h0) = make_float4(o[0].x[r] * back, o[1].x[r] * back16, o[2].x[r] * back, o[3].x[r] * back16);
          *reinterpret_cast<float4*>(at + h1) = make_float4(o[0].x[2 + r] * back, o[1].x[2 + r] * back16, o[2].x[2 + r] * back, o[3].x[2 + r] * back16);
        }
      }
      if (g == 0) {
#pragma unroll
        for (int r = 0; r < 2; ++r) ml[warp * kRows + 8 * nt + 2 * c + r] = make_float2(m[nt][r] == kNone ? -INFINITY : m[nt][r], l[nt][r]);
      }
    }
  }
  __syncthreads();
  const size_t part_row = ((static_cast<size_t>(seq) * a.Hkv + hkv) * G + row0) * a.splits + split;
  for (int item = threadIdx.x; item < min(kRows, G - row0) * (D / 4); item += kWarps * 32) {
    const int r = item / (D / 4), q4 = item % (D / 4);
    float weight[kWarps], mx = -INFINITY, sum = 0.f;
    float2 x[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      x[w] = w < used ? ml[w * kRows + r] : make_float2(-INFINITY, 0.f);
      mx = fmaxf(mx, x[w].x);
    }
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      weight[w] = x[w].x == -INFINITY ? 0.f : Exp2(x[w].x - mx);
      sum += x[w].x == -INFINITY && x[w].y == 0.f ? 0.f : weight[w] * x[w].y;
    }
    const float none = nan_groups[r] >> (q4 >> 4) & 1 ? __int_as_float(0x7fc00000) : 0.f;
    float4 o = make_float4(none, none, none, none);
    const float* src = merge + r * P::kStride + (q4 ^ ((r >> 1) & 1)) * 4;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < used) {
        const float f = weight[w], b = sums_lo[(w * kRows + r) * NG + (q4 >> 4)];
        const float4 v = *reinterpret_cast<const float4*>(src + w * kRows * P::kStride);
        o.x = fmaf(f, v.x + b, o.x);
        o.y = fmaf(f, v.y + b, o.y);
        o.z = fmaf(f, v.z + b, o.z);
        o.w = fmaf(f, v.w + b, o.w);
      }
    }
    if (span.active == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int t = a.Row(row0 + r);
      StoreRow(a, static_cast<size_t>(t) * a.Hq + hkv * gqa + row0 + r - t * gqa, D, 4 * q4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    } else if constexpr (CLUSTER) {
      *reinterpret_cast<float4*>(smem + P::kMerge + P::kBase + item * 16) = o;
      if (q4 == 0) shared_ml[r] = make_float4(mx, sum, 0.f, 0.f);
    } else {
      const size_t row = part_row + static_cast<size_t>(r) * a.splits;
      *reinterpret_cast<float4*>(a.part_acc + row * D + 4 * q4) = o;
      if (q4 == 0) a.part_ml[row] = make_float2(mx, sum);
    }
  }
  if constexpr (CLUSTER) {
    if (span.active == 1) return;
    ptx::ClusterSync();
    // each CTA finishes its share of the columns from all CTAs' shared memory: statistics first, then the sums, each in flight together
    const uint32_t ml_at = ptx::SmemAddr(shared_ml), o_at = ptx::SmemAddr(smem + P::kMerge + P::kBase);
    for (int item = split * kWarps * 32 + threadIdx.x; item < min(kRows, G - row0) * (D / 4); item += a.splits * kWarps * 32) {
      const int r = item / (D / 4), q4 = item % (D / 4);
      float weight[kMaxCluster], mx = -INFINITY, sum = 0.f;
      float4 part[kMaxCluster], o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kMaxCluster; ++k) part[k] = k < span.active ? ptx::LoadRemote4(ml_at + r * 16, k) : make_float4(-INFINITY, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kMaxCluster; ++k) mx = fmaxf(mx, part[k].x);
#pragma unroll
      for (int k = 0; k < kMaxCluster; ++k) {
        weight[k] = part[k].x == -INFINITY ? 0.f : Exp2(part[k].x - mx);
        sum += part[k].x == -INFINITY && part[k].y == 0.f ? 0.f : weight[k] * part[k].y;
      }
#pragma unroll
      for (int k = 0; k < kMaxCluster; ++k) part[k] = k < span.active ? ptx::LoadRemote4(o_at + item * 16, k) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kMaxCluster; ++k) {
        o.x = fmaf(weight[k], part[k].x, o.x);
        o.y = fmaf(weight[k], part[k].y, o.y);
        o.z = fmaf(weight[k], part[k].z, o.z);
        o.w = fmaf(weight[k], part[k].w, o.w);
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int t = a.Row(row0 + r);
      StoreRow(a, static_cast<size_t>(t) * a.Hq + hkv * gqa + row0 + r - t * gqa, D, 4 * q4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    }
    ptx::ClusterSync();                          // nobody leaves while its results are read
  }
}

// grid (G, Hkv, batch): a CTA per row, D / 4 columns of four times eight groups of splits.  Partial results are fetched before it is known how
// many of them there are (the scratch has room for all), so the statistics, the results and the gate are one round trip to memory.
constexpr int kMaxSplits = 256, kGroups = 8, kAhead = 5;
template <int D>
__global__ void __launch_bounds__(kGroups * D / 4) CombineKv4Kernel(DecodeArgs a) {
  PdlEnter();
  constexpr int kThreads = kGroups * D / 4;
  const int seq = blockIdx.z, hkv = blockIdx.y, r = blockIdx.x, q4 = threadIdx.x % (D / 4), part = threadIdx.x / (D / 4);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (a.row_slot != nullptr) {
    a.out += static_cast<size_t>(seq) * a.Hq * D;
    if (a.qg != nullptr) a.qg += static_cast<size_t>(seq) * a.Hq * 2 * D;
    a.positions += seq;
  }
  __shared__ float weight[kMaxSplits], red[kThreads / 32], lsum[kThreads / 32];
  __shared__ float4 osum[kGroups][D / 4];
  const int gqa = a.Hq / a.Hkv, G = gqa * a.T;
  const size_t at = ((static_cast<size_t>(seq) * a.Hkv + hkv) * G + r) * a.splits;
  const float* src = a.part_acc + at * D + 4 * q4;
  float4 v[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    v[i] = part + kGroups * i < a.splits ? __ldcs(reinterpret_cast<const float4*>(src + static_cast<size_t>(part + kGroups * i) * D)) : make_float4(0.f, 0.f, 0.f, 0.f);
  float2 x[(kMaxSplits + kThreads - 1) / kThreads];
#pragma unroll
  for (int k = 0; k < (kMaxSplits + kThreads - 1) / kThreads; ++k)
    x[k] = static_cast<int>(threadIdx.x) + k * kThreads < a.splits ? a.part_ml[at + threadIdx.x + k * kThreads] : make_float2(0.f, 0.f);
  const int active = Visible(a).active;
  if (active == 1) return;                       // the first kernel has finished the rows
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < (kMaxSplits + kThreads - 1) / kThreads; ++k)
    if (static_cast<int>(threadIdx.x) + k * kThreads < active) m = fmaxf(m, x[k].x);
  m = WarpMax(m);
  if (lane == 0) red[warp] = m;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) m = fmaxf(m, red[w]);
  float l = 0.f;
#pragma unroll
  for (int k = 0; k < (kMaxSplits + kThreads - 1) / kThreads; ++k)
    if (static_cast<int>(threadIdx.x) + k * kThreads < active) {
      const float f = x[k].x == -INFINITY ? 0.f : Exp2(x[k].x - m);
      weight[threadIdx.x + k * kThreads] = f;
      l += x[k].x == -INFINITY && x[k].y == 0.f ? 0.f : f * x[k].y;
    }
  l = WarpSum(l);
  if (lane == 0) lsum[warp] = l;
  __syncthreads();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](int s, const float4& p) {
    if (s < active) {
      const float f = weight[s];
      o.x = fmaf(f, p.x, o.x);
      o.y = fmaf(f, p.y, o.y);
      o.z = fmaf(f, p.z, o.z);
      o.w = fmaf(f, p.w, o.w);
    }
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) add(part + kGroups * i, v[i]);
  for (int s = part + kGroups * kAhead; s < active; s += kGroups) add(s, __ldcs(reinterpret_cast<const float4*>(src + static_cast<size_t>(s) * D)));
  osum[part][q4] = o;
  __syncthreads();
  if (part == 0) {
    l = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) l += lsum[w];
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int k = 1; k < kGroups; ++k) {
      const float4 p = osum[k][q4];
      o.x += p.x; o.y += p.y; o.z += p.z; o.w += p.w;
    }
    const int t = a.Row(r);
    StoreRow(a, static_cast<size_t>(t) * a.Hq + hkv * gqa + r - t * gqa, D, 4 * q4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
  }
}

template <int D, int NT, bool CLUSTER>
int LaunchDecode(DecodeArgs a, int batch, cudaStream_t s) {
  // the kernel's limits of shared memory and cluster size, once per device (a bit each; two threads may both set them)
  static std::atomic<uint64_t> allowed{0};
  const auto kern = DecodeKv4Kernel<D, NT, CLUSTER>;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (device > 63 || !(allowed.load(std::memory_order_acquire) >> device & 1)) {
    e = AllowAllSharedMemory(kern);
    if (e == cudaSuccess && CLUSTER) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (device < 64) allowed.fetch_or(uint64_t{1} << device, std::memory_order_release);
  }
  using P = Plan<D, NT>;
  a.per_token = a.Hq == a.Hkv ? 0u : static_cast<uint32_t>((0x100000000ull + a.Hq / a.Hkv - 1) / (a.Hq / a.Hkv));
  const int G = a.Hq / a.Hkv * a.T, chunks = (G + P::kRows - 1) / P::kRows;
  const dim3 grid(a.splits, a.Hkv * chunks, batch);
  if constexpr (CLUSTER) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(P::kWarps * 32);
    cfg.dynamicSmemBytes = P::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_use_pdl ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, kern, a);
    ++g_launch_count;
    return static_cast<int>(e);
  } else {
    const int rc = LaunchPdl(kern, grid, dim3(P::kWarps * 32), P::kSmem, s, a);
    if (rc || a.splits == 1) return rc;
    return LaunchPdl(CombineKv4Kernel<D>, dim3(G, a.Hkv, batch), dim3(kGroups * D / 4), 0, s, a);
  }
}

// tile: rows of a CTA, 8 or as many as the registers allow.
template <int D, bool CLUSTER>
int LaunchDecodeRows(const DecodeArgs& a, int batch, int tile, cudaStream_t s) {
  return tile == 8 ? LaunchDecode<D, 1, CLUSTER>(a, batch, s) : LaunchDecode<D, kWideTile<D> / 8, CLUSTER>(a, batch, s);
}

template <bool CLUSTER>
int LaunchDecodeDim(const DecodeArgs& a, int batch, int D, int tile, cudaStream_t s) {
  return D == 256 ? LaunchDecodeRows<256, CLUSTER>(a, batch, tile, s)
                  : (D == 128 ? LaunchDecodeRows<128, CLUSTER>(a, batch, tile, s) : LaunchDecodeRows<64, CLUSTER>(a, batch, tile, s));
}

}  // namespace
}  // namespace r4dxb

using namespace r4dxb;

/* tile: query rows of a kv head that a CTA takes, 8, 16 (D = 256) or 32 (D = 64, 128); scratch (splits > 1, no cluster): batch * Hkv * G * splits * (D + 2) floats, 16-byte aligned: the partial sums, then (maximum, sum) pairs */
extern "C" int r4dxb_attn_decode_kv4(const void* q, const void* qg, const void* cache, const int* block_tables, const int* row_slot, int slots,
                                     int table_length, int pool, const int* positions, int pos0, float* scratch, void* out, int T, int batch, int Hq,
                                     int Hkv, int D, int tile, int splits, int chunk, int cluster, int window, int* status, void* stream) {
  if (T < 1 || T > 32 || batch < 1 || batch > 65535 || (row_slot == nullptr && batch != 1) || (row_slot != nullptr && T != 1) || Hkv < 1 || Hq < 1 ||
      Hq % Hkv || (D != 64 && D != 128 && D != 256) || (tile != 8 && tile != (D == 256 ? kWideTile<256> : kWideTile<64>)) ||
      chunk < 1 || splits < 1 || splits > (cluster ? kMaxCluster : kMaxSplits) || slots < 1 || table_length < 1 || pool < 1 || window < 0)
    return R4DXB_BAD_ARG;
  if ((static_cast<long long>(Hq / Hkv) * T + tile - 1) / tile * Hkv > 65535) return R4DXB_TOO_LARGE;
  if (q == nullptr || cache == nullptr || block_tables == nullptr || (positions == nullptr && (row_slot != nullptr || pos0 < 0 || pos0 > 0x7fffffff - T)) || out == nullptr || (splits > 1 && !cluster && scratch == nullptr))
    return R4DXB_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(scratch)) & 15 ||
      (reinterpret_cast<uintptr_t>(qg) | reinterpret_cast<uintptr_t>(out)) & 7)
    return R4DXB_BAD_ARG;
  DecodeArgs a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.qg = static_cast<const __nv_bfloat16*>(qg);
  a.cache = static_cast<const uint8_t*>(cache);
  a.table = {block_tables, table_length, pool};
  a.positions = positions;
  a.row_slot = row_slot;
  a.part_acc = scratch;
  a.part_ml = reinterpret_cast<float2*>(scratch + static_cast<size_t>(batch) * Hq * T * splits * D);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.status = status;
  a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.splits = splits; a.chunk = chunk; a.pos0 = pos0; a.slots = slots; a.window = window;
  a.end = min(table_length, 0x7fffffff / kv4::kBlock) * kv4::kBlock;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return cluster ? LaunchDecodeDim<true>(a, batch, D, tile, s) : LaunchDecodeDim<false>(a, batch, D, tile, s);
}
