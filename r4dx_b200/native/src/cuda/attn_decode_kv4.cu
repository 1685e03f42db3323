// Attention of few query rows (decode steps, speculative windows, batches of one row a sequence) over the 4-bit paged cache (kv4.cuh).
//
// Split-KV: a CTA has eight query rows of a kv head (of the G = rows x query heads per kv head) and a share of the sequence's blocks; each
// of its warps walks blocks of its own, which arrive as one bulk copy per block into the warp's ring of shared memory.  Per block
//   scores   S^T[16 tokens x 8 rows] = K Q^T on mma.m16n8k16 (bf16): A = the codes, widened by a mask and an or to 128 + n, B = the query
//            rows as they are (held in registers).  The sum starts at -136 sum(q), so a group gives sum q (n - 8), exactly up to fp32
//            sums; then s (that) + (lo + 8 s) sum(q) per group, token and row.
//   softmax  running maximum per row in the log2 domain, moved only when a score is more than 8 above it (p <= 2^8), so that most blocks
//            need no exchange between lanes; sums in fp32 per lane.
//   values   O^T[D x 8 rows] += (n - 8) (p s):  A = codes of token pairs, 128 + n less 136, exact in bf16; B = p s rounded to bf16 (2^-9
//            of each product, random in sign: below the rounding of the output), turned from scores' to operand order with movmatrix.
//            sum p (lo + 8 s) per group in fp32.  (Codes left at 128 + n would have the sums at 30 to 40 times their result.)
// The warps' results meet in shared memory, the splits' in a second kernel; a sequence short enough for one CTA is finished by it.
// A row with no visible token (position -1) gives zeros; a block that the table or pool does not have gives NaN to the rows that see it.
#include "kv4.cuh"
#include "sm100_ptx.cuh"

namespace r4dxb {
namespace {

constexpr int kWarps = 8;
constexpr int kRows = 8;               // query rows of a CTA
constexpr float kRescaleStep = 8.f;

struct DecodeArgs {
  const __nv_bfloat16* q;      // [T, Hq, D]
  const __nv_bfloat16* qg;     // [T, Hq, 2 D], the gate behind (null: none)
  const uint8_t* cache;
  kv4::Table table;
  const int* positions;        // [T]; batched: one row each
  const int* row_slot;         // batched: sequence of each row
  float* part_acc;             // [batch][Hkv][G][splits][D]
  float2* part_ml;             // [batch][Hkv][G][splits]
  __nv_bfloat16* out;          // [T, Hq, D]
  int* status;
  int T, Hq, Hkv, splits, slots, window;
};

template <int D>
struct Ring {
  static constexpr int kStages = D == 256 ? 4 : 8;               // blocks in flight per warp
  static constexpr int kBytes = kWarps * kStages * kv4::Shape<D>::kRun;
  static constexpr int kStride = D + 4;                          // floats between rows of the merge
  static constexpr size_t kSmem = kBytes + kWarps * kStages * 8 + kWarps * kRows * 8 + 16;
  static_assert(kWarps * kRows * kStride * 4 <= kBytes, "the warps' results fit where the ring was");
};

// The blocks that the rows of a call may see and the number of CTAs that share them: a block per warp at least.
struct Span {
  int first, blocks, active, low, high;
};
__device__ __forceinline__ Span Visible(const int* positions, int T, int window, int splits) {
  const int lane = threadIdx.x & 31;
  const int p = lane < T ? positions[lane] : -1;
  Span s;
  s.high = __reduce_max_sync(0xffffffffu, p);
  s.low = __reduce_min_sync(0xffffffffu, p < 0 ? 0x7fffffff : p);
  s.first = window > 0 && s.high >= 0 ? max(0, s.low - window + 1) / kv4::kBlock : 0;
  s.blocks = s.high >= 0 ? s.high / kv4::kBlock + 1 - s.first : 0;
  s.active = max(1, min(splits, (s.blocks + kWarps - 1) / kWarps));
  return s;
}

__device__ __forceinline__ void MmaBf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
// codes i and i + 4 of a word as the bf16 pair 128 + n
__device__ __forceinline__ uint32_t CodePair(uint32_t w, int i) { return (w >> (4 * i) & 0x000f000fu) | 0x43004300u; }
__device__ __forceinline__ uint32_t Centred(uint32_t pair) {           // 128 + n -> n - 8
  const uint32_t c = 0x43084308u;
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&pair), *reinterpret_cast<const __nv_bfloat162*>(&c));
  return *reinterpret_cast<const uint32_t*>(&d);
}

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

template <int D>
__global__ void __launch_bounds__(kWarps * 32, 1) DecodeKv4Kernel(DecodeArgs a) {
  PdlEnter();
  using S = kv4::Shape<D>;
  using R = Ring<D>;
  constexpr int NG = S::kGroups, NJ = D / 32;
  extern __shared__ __align__(128) unsigned char smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + R::kBytes);
  float2* ml = reinterpret_cast<float2*>(bars + kWarps * R::kStages);           // [warps][rows]
  volatile int* abort_flag = reinterpret_cast<int*>(ml + kWarps * kRows);
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
  const Span span = Visible(a.positions, a.T, a.window, a.splits);
  if (split >= span.active) return;
  const int per = (span.blocks + span.active - 1) / span.active;
  const int b0 = span.first + split * per + warp, b1 = min(span.first + span.blocks, span.first + (split + 1) * per);
  const int steps = b1 > b0 ? (b1 - b0 + kWarps - 1) / kWarps : 0;

  unsigned char* ring = smem + warp * R::kStages * S::kRun;
  uint64_t* full = bars + warp * R::kStages;
  if (lane == 0) {
    for (int i = 0; i < R::kStages; ++i) ptx::MbarInit(full + i, 1);
    ptx::MbarFenceInit();
  }
  if (threadIdx.x == 0) *abort_flag = 0;
  __syncthreads();

  // ---- copies: block b0 + 8 i into slot i % kStages ----
  uint32_t missing = 0u, phases = 0u;          // by slot: no such block; parity of its next wait
  int entry = -1;
  auto issue = [&](int i) {
    if ((i & 31) == 0) entry = i + lane < steps && known ? a.table.BlockAt(b0 + (i + lane) * kWarps) : -1;
    const int blk = __shfl_sync(0xffffffffu, entry, i & 31), slot = i % R::kStages;
    if (blk < 0) {
      missing |= 1u << slot;
      return;
    }
    missing &= ~(1u << slot);
    if (lane == 0) {
      ptx::MbarArriveExpectTx(full + slot, S::kRun);
      ptx::BulkLoad(ring + slot * S::kRun, a.cache + (static_cast<size_t>(blk) * a.Hkv + hkv) * S::kRun, S::kRun, full + slot);
    }
  };
  for (int i = 0; i < min(steps, R::kStages); ++i) issue(i);

  // ---- query rows: operand B of the scores (row g; channels 32 j + 8 c .. as the pairs of CodePair), and their sums per group ----
  const int my_pos = (lane < a.T) ? a.positions[lane] : -1;
  auto position = [&](int r) {
    const int p = __shfl_sync(0xffffffffu, my_pos, r < G ? r / gqa : 0);
    return r < G ? p : -1;
  };
  uint32_t qb[NJ][4];
  float qsum[NG][2];
  {
    const int r = row0 + g;
    const __nv_bfloat16* src = a.q + (static_cast<size_t>(r / gqa) * a.Hq + hkv * gqa + r % gqa) * D + 8 * c;
    float part[NG];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const uint4 v = r < G ? *reinterpret_cast<const uint4*>(src + 32 * j) : make_uint4(0u, 0u, 0u, 0u);
      qb[j][0] = __byte_perm(v.x, v.z, 0x5410);
      qb[j][1] = __byte_perm(v.x, v.z, 0x7632);
      qb[j][2] = __byte_perm(v.y, v.w, 0x5410);
      qb[j][3] = __byte_perm(v.y, v.w, 0x7632);
      const float sum = ((BfLo(v.x) + BfHi(v.x)) + (BfLo(v.y) + BfHi(v.y))) + ((BfLo(v.z) + BfHi(v.z)) + (BfLo(v.w) + BfHi(v.w)));
      part[j >> 1] = (j & 1) ? part[j >> 1] + sum : sum;
    }
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      float s = part[i];
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      qsum[i][0] = __shfl_sync(0xffffffffu, s, 8 * c);
      qsum[i][1] = __shfl_sync(0xffffffffu, s, 8 * c + 4);
    }
  }
  const float scale = rsqrtf(static_cast<float>(D)) * 1.4426950408889634f;
  const int pos0 = position(row0 + 2 * c), pos1 = position(row0 + 2 * c + 1);
  // positions among the rows that there are, for blocks that all of them see whole
  const int row_pos = position(row0 + g);
  const int p_min = __reduce_min_sync(0xffffffffu, row0 + g < G ? row_pos : 0x7fffffff), p_max = __reduce_max_sync(0xffffffffu, row_pos);

  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;       // rows 2 c, 2 c + 1; l of this lane's tokens
  float acc[NG][4][4], base[NG][2];
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    base[j][0] = base[j][1] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i][0] = acc[j][i][1] = acc[j][i][2] = acc[j][i][3] = 0.f;
  }

  bool ok = true;
  int i = 0;
  for (; i < steps; ++i) {
    const int slot = i % R::kStages, kp0 = (b0 + i * kWarps) * kv4::kBlock;
    if (missing >> slot & 1u) {
      auto sees = [&](int pos) { return pos >= kp0 && (a.window == 0 || kp0 + kv4::kBlock - 1 > pos - a.window); };
      if (sees(pos0)) l0 = __int_as_float(0x7fc00000);
      if (sees(pos1)) l1 = __int_as_float(0x7fc00000);
      if (i + R::kStages < steps) issue(i + R::kStages);
      continue;
    }
    ok = ptx::WarpMbarWait(full + slot, phases >> slot & 1u, abort_flag, 1);
    if (!ok) break;
    phases ^= 1u << slot;
    const uint32_t* kw = reinterpret_cast<const uint32_t*>(ring + slot * S::kRun);
    const uint32_t* vw = kw + S::kPart / 4;

    // ---- scores: tokens g (sc[0], sc[1]) and g + 8 (sc[2], sc[3]) of rows 2 c, 2 c + 1 ----
    float sc[4] = {0.f, 0.f, 0.f, 0.f};
    {
      uint32_t pa[NG], pb[NG];
      LoadWords<NG>(kw + 2 * D + g * NG, pa);
      LoadWords<NG>(kw + 2 * D + (g + 8) * NG, pb);
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
      for (int j = 0; j < NG; ++j) {
        float s4[4] = {-136.f * qsum[j][0], -136.f * qsum[j][1], -136.f * qsum[j][0], -136.f * qsum[j][1]};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t x = ca[2 * j + h], y = cb[2 * j + h];
          MmaBf16(s4, CodePair(x, 0), CodePair(y, 0), CodePair(x, 1), CodePair(y, 1), qb[2 * j + h][0], qb[2 * j + h][1]);
          MmaBf16(s4, CodePair(x, 2), CodePair(y, 2), CodePair(x, 3), CodePair(y, 3), qb[2 * j + h][2], qb[2 * j + h][3]);
        }
        const float sa = BfLo(pa[j]), sb = BfLo(pb[j]), ta = fmaf(8.f, sa, BfHi(pa[j])), tb = fmaf(8.f, sb, BfHi(pb[j]));
        sc[0] = fmaf(sa, s4[0], fmaf(ta, qsum[j][0], sc[0]));
        sc[1] = fmaf(sa, s4[1], fmaf(ta, qsum[j][1], sc[1]));
        sc[2] = fmaf(sb, s4[2], fmaf(tb, qsum[j][0], sc[2]));
        sc[3] = fmaf(sb, s4[3], fmaf(tb, qsum[j][1], sc[3]));
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sc[e] *= scale;
    const bool whole = kp0 + kv4::kBlock - 1 <= p_min && (a.window == 0 || kp0 > p_max - a.window);
    bool seen[4] = {true, true, true, true};
    if (!whole) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int kp = kp0 + g + (e >> 1) * 8, pos = e & 1 ? pos1 : pos0;
        seen[e] = kp <= pos && (a.window == 0 || kp > pos - a.window);
        if (!seen[e]) sc[e] = -INFINITY;
      }
    }

    // ---- running maximum and probabilities ----
    const float mx0 = fmaxf(sc[0], sc[2]), mx1 = fmaxf(sc[1], sc[3]);
    if (__any_sync(0xffffffffu, mx0 > m0 + kRescaleStep || mx1 > m1 + kRescaleStep)) {
      float n0 = fmaxf(m0, mx0), n1 = fmaxf(m1, mx1);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, o));
        n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, o));
      }
      const float f0 = n0 == -INFINITY ? 1.f : Exp2(m0 - n0), f1 = n1 == -INFINITY ? 1.f : Exp2(m1 - n1);
      m0 = n0;
      m1 = n1;
      l0 *= f0;
      l1 *= f1;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        base[j][0] *= f0;
        base[j][1] *= f1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[j][e][0] *= f0; acc[j][e][1] *= f1;
          acc[j][e][2] *= f0; acc[j][e][3] *= f1;
        }
      }
    }
    const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
    const float p[4] = {Exp2(sc[0] - r0), Exp2(sc[1] - r1), Exp2(sc[2] - r0), Exp2(sc[3] - r1)};
    l0 += p[0] + p[2];
    l1 += p[1] + p[3];

    // ---- values: tokens 2 c, 2 c + 1 and 8 more; of every 64 channels 8 g .. ----
    uint32_t va[NG], vb[NG], vc[NG], vd[NG], pa[NG], pb[NG];
    LoadWords<NG>(vw + 2 * D + g * NG, pa);
    LoadWords<NG>(vw + 2 * D + (g + 8) * NG, pb);
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
      const float sa = BfLo(pa[j]), sb = BfLo(pb[j]), ta = fmaf(8.f, sa, BfHi(pa[j])), tb = fmaf(8.f, sb, BfHi(pb[j]));
      // (a token that a row does not see may hold anything: its pair is left out, not multiplied by zero)
      const float w0 = seen[0] ? p[0] * sa : 0.f, w1 = seen[1] ? p[1] * sa : 0.f, w2 = seen[2] ? p[2] * sb : 0.f, w3 = seen[3] ? p[3] * sb : 0.f;
      base[j][0] += (seen[0] ? p[0] * ta : 0.f) + (seen[2] ? p[2] * tb : 0.f);
      base[j][1] += (seen[1] ? p[1] * ta : 0.f) + (seen[3] ? p[3] * tb : 0.f);
      const uint32_t wb0 = Transpose8x8(PackBf16(w0, w1)), wb1 = Transpose8x8(PackBf16(w2, w3));
      const uint32_t ab_lo = __byte_perm(va[j], vb[j], 0x5410), ab_hi = __byte_perm(va[j], vb[j], 0x7632);
      const uint32_t cd_lo = __byte_perm(vc[j], vd[j], 0x5410), cd_hi = __byte_perm(vc[j], vd[j], 0x7632);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        MmaBf16(acc[j][e], Centred(CodePair(ab_lo, e)), Centred(CodePair(ab_hi, e)), Centred(CodePair(cd_lo, e)), Centred(CodePair(cd_hi, e)), wb0, wb1);
    }
    __syncwarp();                                // every lane has read the slot
    if (i + R::kStages < steps) issue(i + R::kStages);
  }
  if (!ok) {
    // a copy did not arrive in time: the rows are NaN, the status word says so, and the copies still under way are waited for
    l0 = l1 = __int_as_float(0x7fc00000);
    if (lane == 0) {
      if (a.status != nullptr) atomicCAS(a.status, 0, 800 + *abort_flag);
      const long long t0 = clock64();
      for (int k = i; k < min(steps, i + R::kStages); ++k) {
        const int slot = k % R::kStages;
        while (!(missing >> slot & 1u) && !ptx::MbarTryWait(full + slot, phases >> slot & 1u) && clock64() - t0 < ptx::kWaitClocks) {}
      }
    }
    __syncwarp();
  }

  // ---- the lanes' sums of rows 2 c, 2 c + 1, then the warps' ----
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, o);
    l1 += __shfl_xor_sync(0xffffffffu, l1, o);
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      base[j][0] += __shfl_xor_sync(0xffffffffu, base[j][0], o);
      base[j][1] += __shfl_xor_sync(0xffffffffu, base[j][1], o);
    }
  }
  __syncthreads();                               // the ring is read by no one any more
  float* merge = reinterpret_cast<float*>(smem);
  {
    float* dst = merge + (warp * kRows + 2 * c) * R::kStride + 8 * g;
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float b = base[j][r];
        *reinterpret_cast<float4*>(dst + r * R::kStride + 64 * j) = make_float4(acc[j][0][r] + b, acc[j][1][r] + b, acc[j][2][r] + b, acc[j][3][r] + b);
        *reinterpret_cast<float4*>(dst + r * R::kStride + 64 * j + 4) =
            make_float4(acc[j][0][2 + r] + b, acc[j][1][2 + r] + b, acc[j][2][2 + r] + b, acc[j][3][2 + r] + b);
      }
    if (g == 0) {
      ml[warp * kRows + 2 * c] = make_float2(m0, l0);
      ml[warp * kRows + 2 * c + 1] = make_float2(m1, l1);
    }
  }
  __syncthreads();
  // a warp per row
  const int r = row0 + warp;
  if (r >= G) return;
  float m = -INFINITY, l = 0.f, weight[kWarps];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[w * kRows + warp].x);
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const float2 x = ml[w * kRows + warp];
    weight[w] = x.x == -INFINITY ? 0.f : Exp2(x.x - m);
    l += x.x == -INFINITY && x.y == 0.f ? 0.f : weight[w] * x.y;
  }
  float o[D / 32];
#pragma unroll
  for (int k = 0; k < D / 32; ++k) {
    o[k] = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) o[k] = fmaf(weight[w], merge[(w * kRows + warp) * R::kStride + 32 * k + lane], o[k]);
  }
  if (span.active == 1) {
    const size_t row = static_cast<size_t>(r / gqa) * a.Hq + hkv * gqa + r % gqa;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      float v = o[k] * inv;
      if (a.qg != nullptr) v *= Sigmoid(__bfloat162float(a.qg[row * 2 * D + D + 32 * k + lane]));
      a.out[row * D + 32 * k + lane] = __float2bfloat16_rn(v);
    }
  } else {
    const size_t at = ((static_cast<size_t>(seq) * a.Hkv + hkv) * G + r) * a.splits + split;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) a.part_acc[at * D + 32 * k + lane] = o[k];
    if (lane == 0) a.part_ml[at] = make_float2(m, l);
  }
}

// grid (G D / 64, Hkv, batch), 256 threads: 64 columns x 4 groups of splits.
constexpr int kMaxSplits = 256;
template <int D>
__global__ void __launch_bounds__(256) CombineKv4Kernel(DecodeArgs a) {
  PdlEnter();
  constexpr int kCols = 64;
  const int seq = blockIdx.z, hkv = blockIdx.y, r = blockIdx.x / (D / kCols), col = blockIdx.x % (D / kCols) * kCols + (threadIdx.x & 63);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = threadIdx.x >> 6;
  if (a.row_slot != nullptr) {
    a.out += static_cast<size_t>(seq) * a.Hq * D;
    if (a.qg != nullptr) a.qg += static_cast<size_t>(seq) * a.Hq * 2 * D;
    a.positions += seq;
  }
  const int gqa = a.Hq / a.Hkv, G = gqa * a.T;
  const int active = Visible(a.positions, a.T, a.window, a.splits).active;
  if (active == 1) return;                       // the first kernel has finished the rows
  __shared__ float wsm[kMaxSplits], red[8], lsum[8], osum[4][kCols];
  const size_t at = ((static_cast<size_t>(seq) * a.Hkv + hkv) * G + r) * a.splits;
  float2 x = make_float2(-INFINITY, 0.f);
  if (static_cast<int>(threadIdx.x) < active) x = a.part_ml[at + threadIdx.x];
  const float mx = WarpMax(x.x);
  if (lane == 0) red[warp] = mx;
  __syncthreads();
  float m = red[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) m = fmaxf(m, red[w]);
  const float weight = x.x == -INFINITY ? 0.f : Exp2(x.x - m);
  wsm[threadIdx.x] = weight;
  const float ls = WarpSum(x.x == -INFINITY && x.y == 0.f ? 0.f : weight * x.y);
  if (lane == 0) lsum[warp] = ls;
  __syncthreads();
  float o = 0.f;
  const float* src = a.part_acc + at * D + col;
  for (int s0 = part; s0 < active; s0 += 32) {   // eight loads in flight
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = s0 + 4 * i < active ? __ldcs(src + static_cast<size_t>(s0 + 4 * i) * D) : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (s0 + 4 * i < active) o = fmaf(wsm[s0 + 4 * i], v[i], o);
  }
  osum[part][threadIdx.x & 63] = o;
  __syncthreads();
  if (part == 0) {
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) l += lsum[w];
    const int k = threadIdx.x;
    float v = ((osum[0][k] + osum[1][k]) + (osum[2][k] + osum[3][k])) * (l == 0.f ? 0.f : 1.f / l);
    const size_t row = static_cast<size_t>(r / gqa) * a.Hq + hkv * gqa + r % gqa;
    if (a.qg != nullptr) v *= Sigmoid(__bfloat162float(a.qg[row * 2 * D + D + col]));
    a.out[row * D + col] = __float2bfloat16_rn(v);
  }
}

template <int D>
int LaunchDecode(const DecodeArgs& a, int batch, cudaStream_t s) {
  const cudaError_t e = AllowAllSharedMemory(DecodeKv4Kernel<D>);
  if (e != cudaSuccess) return static_cast<int>(e);
  const int G = a.Hq / a.Hkv * a.T, chunks = (G + kRows - 1) / kRows;
  const int rc = LaunchPdl(DecodeKv4Kernel<D>, dim3(a.splits, a.Hkv * chunks, batch), dim3(kWarps * 32), Ring<D>::kSmem, s, a);
  if (rc || a.splits == 1) return rc;
  return LaunchPdl(CombineKv4Kernel<D>, dim3(G * (D / 64), a.Hkv, batch), dim3(256), 0, s, a);
}

}  // namespace
}  // namespace r4dxb

using namespace r4dxb;

/* scratch (splits > 1): batch * Hkv * G * splits * (D + 2) floats, 16-byte aligned: the partial sums, then (maximum, sum) pairs */
extern "C" int r4dxb_attn_decode_kv4(const void* q, const void* qg, const void* cache, const int* block_tables, const int* row_slot, int slots,
                                     int table_length, int pool, const int* positions, float* scratch, void* out, int T, int batch, int Hq,
                                     int Hkv, int D, int splits, int window, int* status, void* stream) {
  if (T < 1 || T > 32 || batch < 1 || batch > 65535 || (row_slot == nullptr && batch != 1) || (row_slot != nullptr && T != 1) || Hkv < 1 || Hq < 1 ||
      Hq % Hkv || (D != 64 && D != 128 && D != 256) || splits < 1 || splits > kMaxSplits || slots < 1 || table_length < 1 || pool < 1 || window < 0)
    return R4DXB_BAD_ARG;
  if ((static_cast<long long>(Hq / Hkv) * T + kRows - 1) / kRows * Hkv > 65535) return R4DXB_TOO_LARGE;
  if (q == nullptr || cache == nullptr || block_tables == nullptr || positions == nullptr || out == nullptr || (splits > 1 && scratch == nullptr))
    return R4DXB_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(scratch)) & 15) return R4DXB_BAD_ARG;
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
  a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.splits = splits; a.slots = slots; a.window = window;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return D == 256 ? LaunchDecode<256>(a, batch, s) : (D == 128 ? LaunchDecode<128>(a, batch, s) : LaunchDecode<64>(a, batch, s));
}
