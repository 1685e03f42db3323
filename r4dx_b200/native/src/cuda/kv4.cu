// 4-bit paged KV cache (layout: kv4.cuh): rows written into it, with the norms and the rotation of an attention layer before, and rows
// read back.
//
//   precore   q -> norm, rope -> bf16;  k -> norm, rope -> bf16 -> codes;  v -> codes       (r4dxb_attn_precore_kv4)
//   write     the same without q, norms and rotation                                        (Hq = 0, rotary_dim = 0)
//   read      bf16(n s + lo) of any positions of a sequence                                 (r4dxb_kv4_read)
//
// Codes of a group of 64 channels:  lo = min x,  s = bf16((max x - lo) / 15),  n = clamp(rint((x - lo) / s), 0, 15), with x the row's
// bf16 values brought into +-32768.  The minimum of bf16 values is one of them, so lo loses nothing; the codes are taken against
// the rounded s, so its rounding (2^-9) only clips the top code.  Divisions are IEEE ones: the codes are those of any other
// program that follows the definition.  A group that holds a NaN gets s = NaN and reads back as NaN throughout.
#include "kv4.cuh"

namespace r4dxb {
namespace {

struct PrecoreArgs {
  const __nv_bfloat16* qg;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  const __nv_bfloat16* q_norm;
  const __nv_bfloat16* k_norm;
  const int* positions;
  const int* row_slot;         // row t belongs to the sequence with table row_slot[t] (null: one sequence)
  kv4::Table table;
  __nv_bfloat16* q_out;
  uint32_t* cache;
  int T, Hq, Hkv, slots, rotary_dim, q_stride;
  float theta, eps;
};

// N bf16 values from 2 N bytes at once
template <int N>
__device__ __forceinline__ void LoadRow(const __nv_bfloat16* p, float (&x)[N]) {
  uint32_t w[N / 2];
  if constexpr (N == 8) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (N == 4) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    x[2 * i] = BfLo(w[i]);
    x[2 * i + 1] = BfHi(w[i]);
  }
}

// grid (T, head groups), 8 warps: a warp per head, lane l channels l D / 32 ..  A CTA's angles are one table: for few rows they cost
// each CTA one round of fp64 sincos, for many the table serves all heads of a token.
template <int D>
__global__ void __launch_bounds__(256) PrecoreKv4Kernel(PrecoreArgs a) {
  PdlEnter();
  constexpr int PER = D / 32, LANES = kv4::kGroup / PER;         // channels of a lane, lanes of a group
  extern __shared__ float smem[];
  const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int half = a.rotary_dim / 2, pos = a.positions[t];
  float* cs = smem;                                              // [half] cosines, [half] sines
  float* hrow = smem + a.rotary_dim + warp * D;
  for (int i = threadIdx.x; i < half; i += 256) {
    const double inv = exp2(-log2(static_cast<double>(a.theta)) * (2.0 * i / a.rotary_dim));
    double s, c;
    sincos(static_cast<double>(pos) * inv, &s, &c);
    cs[i] = static_cast<float>(c);
    cs[half + i] = static_cast<float>(s);
  }
  __syncthreads();
  const int slot = a.row_slot != nullptr ? a.row_slot[t] : 0;
  int blk = -1;
  if (pos >= 0 && slot >= 0 && slot < a.slots) {
    kv4::Table table = a.table;
    table.entries += static_cast<size_t>(slot) * table.length;
    blk = table.BlockAt(pos / kv4::kBlock);
  }
  const int tok = pos & (kv4::kBlock - 1);
  for (int hh = blockIdx.y * 8 + warp; hh < a.Hq + 2 * a.Hkv; hh += 8 * gridDim.y) {
    const int kind = hh < a.Hq ? 0 : (hh < a.Hq + a.Hkv ? 1 : 2);       // 0 = q, 1 = k, 2 = v
    const int head = kind == 0 ? hh : (kind == 1 ? hh - a.Hq : hh - a.Hq - a.Hkv);
    if (kind != 0 && blk < 0) continue;
    const __nv_bfloat16* src = kind == 0 ? a.qg + (static_cast<size_t>(t) * a.Hq + head) * a.q_stride
                                         : (kind == 1 ? a.k : a.v) + (static_cast<size_t>(t) * a.Hkv + head) * D;
    float x[PER];
    LoadRow<PER>(src + lane * PER, x);
    if (kind != 2) {
      const __nv_bfloat16* nw = kind == 0 ? a.q_norm : a.k_norm;
      if (nw != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) ss += x[i] * x[i];
        const float r = rsqrtf(WarpSum(ss) / D + a.eps);
        float w[PER];
        LoadRow<PER>(nw + lane * PER, w);
#pragma unroll
        for (int i = 0; i < PER; ++i) x[i] = x[i] * r * (1.0f + w[i]);
      }
      if (half > 0) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < PER; ++i) hrow[lane * PER + i] = x[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int d = lane * PER + i;
          if (d < a.rotary_dim) {
            const int j = d < half ? d : d - half;
            const float fc = cs[j], fs = cs[half + j];
            x[i] = d < half ? hrow[d] * fc - hrow[d + half] * fs : hrow[d] * fc + hrow[d - half] * fs;
          }
        }
      }
    }
    uint32_t packed[PER / 2];
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) packed[i] = PackBf16(x[2 * i], x[2 * i + 1]);
    if (kind == 0) {
      __nv_bfloat16* dst = a.q_out + (static_cast<size_t>(t) * a.Hq + head) * D + lane * PER;
      if constexpr (PER == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
      else if constexpr (PER == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[1]);
      else *reinterpret_cast<uint32_t*>(dst) = packed[0];
      continue;
    }
    bool nan = false;
    float lo = kv4::kLimit, hi = -kv4::kLimit;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      x[i] = (i & 1) ? BfHi(packed[i / 2]) : BfLo(packed[i / 2]);
      nan |= x[i] != x[i];
      x[i] = fminf(fmaxf(x[i], -kv4::kLimit), kv4::kLimit);
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const uint32_t nans = __ballot_sync(0xffffffffu, nan);
    constexpr uint32_t kOne = LANES == 32 ? 0xffffffffu : (1u << (LANES & 31)) - 1u;
    const bool bad = (nans >> (lane / LANES * LANES) & kOne) != 0u;
    const __nv_bfloat16 sb = __float2bfloat16_rn(bad ? __int_as_float(0x7fc00000) : __fdiv_rn(hi - lo, 15.f));
    const float s = __bfloat162float(sb);
    uint32_t codes = 0u;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float n = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(x[i] - lo, s)), 0.f), 15.f) : 0.f;
      codes |= static_cast<uint32_t>(n) << (4 * i);
    }
    // the lanes of a word: D = 256 one, 128 two, 64 four
#pragma unroll
    for (int o = 1; o < 8 / PER; o <<= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, codes, o);
      codes = lane & o ? other | codes << (4 * PER * o) : codes | other << (4 * PER * o);
    }
    uint32_t* part = a.cache + ((static_cast<size_t>(blk) * a.Hkv + head) * 2 + (kind - 1)) * (kv4::Shape<D>::kPart / 4);
    const int w = lane * PER / 8;
    if (lane % (8 / PER) == 0) part[kind == 1 ? kv4::Word<D, false>(tok, w) : kv4::Word<D, true>(tok, w)] = codes;
    if (lane % LANES == 0)
      part[2 * D + tok * kv4::Shape<D>::kGroups + lane / LANES] =
          static_cast<uint32_t>(__bfloat16_as_ushort(sb)) | static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(lo))) << 16;
  }
}

// A thread per word of eight channels: [row][head][keys, values][word].
template <int D>
__global__ void __launch_bounds__(256) ReadKv4Kernel(const uint32_t* __restrict__ cache, kv4::Table table, const int* __restrict__ positions,
                                                     const int* __restrict__ row_slot, int slots, __nv_bfloat16* __restrict__ k,
                                                     __nv_bfloat16* __restrict__ v, long long words, int Hkv) {
  PdlEnter();
  using S = kv4::Shape<D>;
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= words) return;
  const int w = static_cast<int>(i % S::kWords), part = static_cast<int>(i / S::kWords) & 1;
  const long long rh = i / (2 * S::kWords);                     // row * Hkv + head
  const int head = static_cast<int>(rh % Hkv), t = static_cast<int>(rh / Hkv);
  const int pos = positions[t], slot = row_slot != nullptr ? row_slot[t] : 0;
  int blk = -1;
  if (pos >= 0 && slot >= 0 && slot < slots) {
    table.entries += static_cast<size_t>(slot) * table.length;
    blk = table.BlockAt(pos / kv4::kBlock);
  }
  uint4 o = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
  if (blk >= 0) {
    const int tok = pos & (kv4::kBlock - 1);
    const uint32_t* at = cache + ((static_cast<size_t>(blk) * Hkv + head) * 2 + part) * (S::kPart / 4);
    const uint32_t codes = __ldg(at + (part == 0 ? kv4::Word<D, false>(tok, w) : kv4::Word<D, true>(tok, w)));
    const uint32_t pair = __ldg(at + 2 * D + tok * S::kGroups + w / 8);
    const float s = BfLo(pair), lo = BfHi(pair);
    uint32_t p[4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
      p[c] = PackBf16(fmaf(static_cast<float>(codes >> (8 * c) & 15u), s, lo), fmaf(static_cast<float>(codes >> (8 * c + 4) & 15u), s, lo));
    o = make_uint4(p[0], p[1], p[2], p[3]);
  }
  *reinterpret_cast<uint4*>((part == 0 ? k : v) + rh * D + 8 * w) = o;
}

template <int D>
int LaunchPrecore(const PrecoreArgs& a, cudaStream_t s) {
  // enough CTAs for eight to an SM where there are few rows, one CTA (and one table of angles) a row where there are many
  const int groups = (a.Hq + 2 * a.Hkv + 7) / 8, most = (8 * 148 + a.T - 1) / a.T;
  const size_t smem = (a.rotary_dim + 8 * D) * sizeof(float);
  return LaunchPdl(PrecoreKv4Kernel<D>, dim3(a.T, groups < most ? groups : most), dim3(256), smem, s, a);
}

template <int D>
int LaunchRead(const void* cache, const kv4::Table& table, const int* positions, const int* row_slot, int slots, void* k, void* v, int T, int Hkv,
               cudaStream_t s) {
  const long long words = static_cast<long long>(T) * Hkv * 2 * kv4::Shape<D>::kWords;
  if ((words + 255) / 256 > 0x7fffffffll) return R4DXB_TOO_LARGE;
  return LaunchPdl(ReadKv4Kernel<D>, dim3(static_cast<unsigned>((words + 255) / 256)), dim3(256), 0, s, static_cast<const uint32_t*>(cache), table,
                   positions, row_slot, slots, static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v), words, Hkv);
}

bool Misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace
}  // namespace r4dxb

using namespace r4dxb;

extern "C" {

int r4dxb_attn_precore_kv4(const void* qg, const void* k, const void* v, const void* q_norm, const void* k_norm, const int* positions,
                           const int* block_tables, const int* row_slot, int slots, int table_length, int pool, void* q_out, void* cache, int T,
                           int Hq, int Hkv, int D, int rotary_dim, float theta, float eps, int q_stride, void* stream) {
  if (T < 1 || Hq < 0 || Hkv < 1 || (D != 64 && D != 128 && D != 256) || rotary_dim < 0 || rotary_dim > D || rotary_dim % 2 || slots < 1 ||
      table_length < 1 || pool < 1 || q_stride < D || q_stride % 8 || k == nullptr || v == nullptr || positions == nullptr ||
      block_tables == nullptr || cache == nullptr || (Hq > 0 && (qg == nullptr || q_out == nullptr)))
    return R4DXB_BAD_ARG;
  if (Misaligned(qg) || Misaligned(k) || Misaligned(v) || Misaligned(q_norm) || Misaligned(k_norm) || Misaligned(q_out) || Misaligned(cache))
    return R4DXB_BAD_ARG;
  PrecoreArgs a;
  a.qg = static_cast<const __nv_bfloat16*>(qg);
  a.k = static_cast<const __nv_bfloat16*>(k);
  a.v = static_cast<const __nv_bfloat16*>(v);
  a.q_norm = static_cast<const __nv_bfloat16*>(q_norm);
  a.k_norm = static_cast<const __nv_bfloat16*>(k_norm);
  a.positions = positions;
  a.row_slot = row_slot;
  a.table = {block_tables, table_length, pool};
  a.q_out = static_cast<__nv_bfloat16*>(q_out);
  a.cache = static_cast<uint32_t*>(cache);
  a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.slots = slots; a.rotary_dim = rotary_dim; a.q_stride = q_stride; a.theta = theta; a.eps = eps;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return D == 256 ? LaunchPrecore<256>(a, s) : (D == 128 ? LaunchPrecore<128>(a, s) : LaunchPrecore<64>(a, s));
}

int r4dxb_kv4_read(const void* cache, const int* block_tables, const int* row_slot, int slots, int table_length, int pool, const int* positions,
                   void* k, void* v, int T, int Hkv, int D, void* stream) {
  if (T < 1 || Hkv < 1 || (D != 64 && D != 128 && D != 256) || slots < 1 || table_length < 1 || pool < 1 || cache == nullptr ||
      block_tables == nullptr || positions == nullptr || k == nullptr || v == nullptr || Misaligned(cache) || Misaligned(k) || Misaligned(v))
    return R4DXB_BAD_ARG;
  const kv4::Table table = {block_tables, table_length, pool};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (D == 256) return LaunchRead<256>(cache, table, positions, row_slot, slots, k, v, T, Hkv, s);
  if (D == 128) return LaunchRead<128>(cache, table, positions, row_slot, slots, k, v, T, Hkv, s);
  return LaunchRead<64>(cache, table, positions, row_slot, slots, k, v, T, Hkv, s);
}

}  // extern "C"
