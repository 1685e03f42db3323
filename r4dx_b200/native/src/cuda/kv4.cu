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
#include <cmath>

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
  int steps, groups;           // rounds of heads that a warp takes, warps to a token
  float eps;
  double turn_exponent, turn_step;      // angle of channel pair i, in turns per position: 2^(turn_exponent + i turn_step)
};

__device__ __forceinline__ void Unpack8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = BfLo(w[i]);
    x[2 * i + 1] = BfHi(w[i]);
  }
}
__device__ __forceinline__ uint4 Load8(const __nv_bfloat16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
// A warp has one token and some of its heads (q, then k, then v): eight channels a lane, D / 8 lanes a head, so 1, 2 or 4 heads at a time, the
// next ones' rows on their way meanwhile.  A channel pair's angle is position x frequency in turns, in 64 bits; what its whole turns
// leave fits 32 bits for the sine and cosine (64-bit ones took as long as all the rest).  Rotated channels change lanes by shuffle
// where their distance is a power of two of lanes, else through shared memory.
template <int D>
__global__ void __launch_bounds__(256) PrecoreKv4Kernel(PrecoreArgs a) {
  PdlEnter();
  constexpr int LPH = D / 8, HPW = 32 / LPH;
  extern __shared__ float smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, li = lane % LPH;
  const int task = blockIdx.x * 8 + warp, t = task / a.groups;
  if (t >= a.T) return;
  const int half = a.rotary_dim / 2, pos = a.positions[t], heads = a.Hq + 2 * a.Hkv;
  float* cs = smem + warp * (a.rotary_dim + 32 * 8);             // [half] cosines, [half] sines
  float* rows = cs + a.rotary_dim;                               // [32 lanes][8]
  const int first = (task % a.groups) * a.steps * HPW + lane / LPH, last = min(heads, first - lane / LPH + a.steps * HPW);

  auto source = [&](int hh) {
    return hh < a.Hq ? a.qg + (static_cast<size_t>(t) * a.Hq + hh) * a.q_stride
                     : (hh < a.Hq + a.Hkv ? a.k + (static_cast<size_t>(t) * a.Hkv + hh - a.Hq) * D : a.v + (static_cast<size_t>(t) * a.Hkv + hh - a.Hq - a.Hkv) * D);
  };
  uint4 next = first < last ? Load8(source(first) + 8 * li) : make_uint4(0u, 0u, 0u, 0u);
  const int slot = a.row_slot != nullptr ? a.row_slot[t] : 0;
  int blk = -1;
  if (pos >= 0 && slot >= 0 && slot < a.slots) {
    kv4::Table table = a.table;
    table.entries += static_cast<size_t>(slot) * table.length;
    blk = table.BlockAt(pos / kv4::kBlock);
  }
  const int tok = pos & (kv4::kBlock - 1);
  for (int i = lane; i < half; i += 32) {
    const double turns = static_cast<double>(pos) * exp2(a.turn_exponent + i * a.turn_step);
    float s, c;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
    cs[i] = c;
    cs[half + i] = s;
  }
  __syncwarp();
  // this lane's rotated channels: d < half with the one half further on, or the other way round
  const int hop = half / 8;                      // lanes
  const bool shuffle = half % 8 == 0 && (hop & (hop - 1)) == 0;
  float fc[8], fs[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = 8 * li + i, j = d < half ? d : d - half;
    fc[i] = d < a.rotary_dim ? cs[j] : 1.f;
    fs[i] = d < a.rotary_dim ? (d < half ? -cs[half + j] : cs[half + j]) : 0.f;
  }
  uint4 norm = make_uint4(0u, 0u, 0u, 0u);       // the weights of the kind at hand
  int norm_kind = -1;

  for (int step = 0; step < a.steps; ++step) {
    const int hh = first + step * HPW;
    const uint4 raw = next;
    if (step + 1 < a.steps && hh + HPW < last) next = Load8(source(hh + HPW) + 8 * li);
    if (hh - lane / LPH >= last) break;          // (the warp's heads are done)
    const int kind = hh >= last ? 3 : (hh < a.Hq ? 0 : (hh < a.Hq + a.Hkv ? 1 : 2));       // 0 = q, 1 = k, 2 = v, 3 = none
    const int head = kind == 0 ? hh : (kind == 1 ? hh - a.Hq : hh - a.Hq - a.Hkv);
    float x[8];
    Unpack8(raw, x);
    const __nv_bfloat16* nw = kind == 0 ? a.q_norm : (kind == 1 ? a.k_norm : nullptr);
    if (nw != nullptr && kind != norm_kind) {
      norm = Load8(nw + 8 * li);
      norm_kind = kind;
    }
    if (a.q_norm != nullptr || a.k_norm != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
      for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (nw != nullptr) {
        const float r = rsqrtf(ss / D + a.eps);
        float w[8];
        Unpack8(norm, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * r * (1.0f + w[i]);
      }
    }
    if (half > 0) {
      float y[8];
      if (shuffle) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __shfl_xor_sync(0xffffffffu, x[i], hop);
      } else {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) rows[lane * 8 + i] = x[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = 8 * li + i;
          y[i] = d < a.rotary_dim ? rows[(lane - li) * 8 + (d < half ? d + half : d - half)] : 0.f;
        }
      }
      if (kind < 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (8 * li + i < a.rotary_dim) x[i] = x[i] * fc[i] + y[i] * fs[i];
      }
    }
    const uint4 packed = make_uint4(PackBf16(x[0], x[1]), PackBf16(x[2], x[3]), PackBf16(x[4], x[5]), PackBf16(x[6], x[7]));
    if (kind == 0) *reinterpret_cast<uint4*>(a.q_out + (static_cast<size_t>(t) * a.Hq + head) * D + 8 * li) = packed;
    if (__all_sync(0xffffffffu, kind == 0)) continue;
    Unpack8(packed, x);
    bool nan = false;
    float lo = kv4::kLimit, hi = -kv4::kLimit;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      nan |= x[i] != x[i];
      x[i] = fminf(fmaxf(x[i], -kv4::kLimit), kv4::kLimit);
      lo = fminf(lo, x[i]);
      hi = fmaxf(hi, x[i]);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {            // the eight lanes of a group
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const bool bad = (__ballot_sync(0xffffffffu, nan) >> (lane & ~7) & 0xffu) != 0u;
    const __nv_bfloat16 sb = __float2bfloat16_rn(bad ? __int_as_float(0x7fc00000) : __fdiv_rn(hi - lo, 15.f));
    const float s = __bfloat162float(sb);
    uint32_t codes = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float n = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(x[i] - lo, s)), 0.f), 15.f) : 0.f;
      codes |= static_cast<uint32_t>(n) << (4 * i);
    }
    if (kind >= 1 && kind <= 2 && blk >= 0) {
      uint32_t* part = a.cache + ((static_cast<size_t>(blk) * a.Hkv + head) * 2 + (kind - 1)) * (kv4::Shape<D>::kPart / 4);
      part[kind == 1 ? kv4::Word<D, false>(tok, li) : kv4::Word<D, true>(tok, li)] = codes;
      if (li % 8 == 0)
        part[2 * D + tok * kv4::Shape<D>::kGroups + li / 8] =
            static_cast<uint32_t>(__bfloat16_as_ushort(sb)) | static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(lo))) << 16;
    }
  }
}

// Rows read back: a thread has one word (eight channels) of a row and up to ITEMS of its 2 Hkv heads' keys and values, whose codes and pairs it
// asks for at once.  (A thread per value word, each with the row's position and table entry to find first, took 62 us for 32517 rows of
// 8 heads of 128 where the bytes take 26.)
template <int D, int ITEMS>
__global__ void __launch_bounds__(256) ReadKv4Kernel(const uint32_t* __restrict__ cache, kv4::Table table, const int* __restrict__ positions,
                                                     const int* __restrict__ row_slot, int slots, __nv_bfloat16* __restrict__ k,
                                                     __nv_bfloat16* __restrict__ v, int T, int Hkv) {
  PdlEnter();
  using S = kv4::Shape<D>;
  const int w = threadIdx.x % S::kWords, t = blockIdx.x * (256 / S::kWords) + threadIdx.x / S::kWords;
  if (t >= T) return;
  const int pos = positions[t], slot = row_slot != nullptr ? row_slot[t] : 0;
  int blk = -1;
  if (pos >= 0 && slot >= 0 && slot < slots) {
    table.entries += static_cast<size_t>(slot) * table.length;
    blk = table.BlockAt(pos / kv4::kBlock);
  }
  const int tok = pos & (kv4::kBlock - 1), first = blockIdx.y * ITEMS;
  const int at_k = kv4::Word<D, false>(tok, w), at_v = kv4::Word<D, true>(tok, w), at_pair = 2 * D + tok * S::kGroups + w / 8;
  uint32_t codes[ITEMS], pair[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {              // item: head, then keys or values - the order of the pool
    codes[i] = 0u;
    pair[i] = 0x7fc07fc0u;
    if (blk >= 0 && first + i < 2 * Hkv) {
      const uint32_t* part = cache + (static_cast<size_t>(blk) * 2 * Hkv + first + i) * (S::kPart / 4);
      codes[i] = __ldg(part + ((first + i) & 1 ? at_v : at_k));
      pair[i] = __ldg(part + at_pair);
    }
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    if (first + i >= 2 * Hkv) break;
    const float s = BfLo(pair[i]), lo = BfHi(pair[i]);
    uint32_t p[4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
      p[c] = PackBf16(fmaf(static_cast<float>(codes[i] >> (8 * c) & 15u), s, lo), fmaf(static_cast<float>(codes[i] >> (8 * c + 4) & 15u), s, lo));
    *reinterpret_cast<uint4*>(((first + i) & 1 ? v : k) + (static_cast<size_t>(t) * Hkv + (first + i) / 2) * D + 8 * w) = make_uint4(p[0], p[1], p[2], p[3]);
  }
}

template <int D>
int LaunchPrecore(PrecoreArgs a, cudaStream_t s) {
  // warps for every SM four times over where there are rows enough; up to eight rounds of heads to a warp, which share its angles
  const int per_round = 256 / D, rounds = (a.Hq + 2 * a.Hkv + per_round - 1) / per_round;
  const long long most = static_cast<long long>(a.T) * rounds / (4 * 148 * 32);
  a.steps = static_cast<int>(most < 1 ? 1 : (most > 8 ? 8 : most));
  a.groups = (rounds + a.steps - 1) / a.steps;
  const long long tasks = static_cast<long long>(a.T) * a.groups;
  if (tasks > 0x7fffffffll - 8) return R4DXB_TOO_LARGE;
  const size_t smem = 8 * (a.rotary_dim + 32 * 8) * sizeof(float);
  return LaunchPdl(PrecoreKv4Kernel<D>, dim3(static_cast<unsigned>((tasks + 7) / 8)), dim3(256), smem, s, a);
}

template <int D>
int LaunchRead(const void* cache, const kv4::Table& table, const int* positions, const int* row_slot, int slots, void* k, void* v, int T, int Hkv,
               cudaStream_t s) {
  constexpr int kRows = 256 / kv4::Shape<D>::kWords;
  if (Hkv > 32767) return R4DXB_TOO_LARGE;
  const unsigned rows = (static_cast<unsigned>(T) + kRows - 1) / kRows, items = 2 * Hkv;
  auto launch = [&](auto kern, unsigned per) {
    return LaunchPdl(kern, dim3(rows, (items + per - 1) / per), dim3(256), 0, s, static_cast<const uint32_t*>(cache), table, positions, row_slot, slots,
                     static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v), T, Hkv);
  };
  return static_cast<unsigned long long>(rows) * items >= 8 * 8 * 148 ? launch(ReadKv4Kernel<D, 8>, 8) : launch(ReadKv4Kernel<D, 1>, 1);
}

bool Misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

}  // namespace
}  // namespace r4dxb

using namespace r4dxb;

extern "C" {

int r4dxb_attn_precore_kv4(const void* qg, const void* k, const void* v, const void* q_norm, const void* k_norm, const int* positions,
                           const int* block_tables, const int* row_slot, int slots, int table_length, int pool, void* q_out, void* cache, int T,
                           int Hq, int Hkv, int D, int rotary_dim, float theta, float eps, int q_stride, void* stream) {
  if (T < 1 || Hq < 0 || Hkv < 1 || (D != 64 && D != 128 && D != 256) || rotary_dim < 0 || rotary_dim > D || rotary_dim % 2 || (rotary_dim > 0 && !(theta > 0.f)) || slots < 1 ||
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
  a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.slots = slots; a.rotary_dim = rotary_dim; a.q_stride = q_stride; a.eps = eps;
  a.turn_step = rotary_dim > 0 ? -2.0 / rotary_dim * std::log2(static_cast<double>(theta)) : 0.0;
  a.turn_exponent = -2.651496129472319;          // -log2(2 pi)
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
