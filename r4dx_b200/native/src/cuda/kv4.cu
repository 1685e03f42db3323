// 4-bit paged KV cache (layout: kv4.cuh): rows written into it, with the norms and the rotation of an attention layer before, and rows
// read back.
//
//   precore   q -> norm, rope -> bf16;  k -> norm, rope -> bf16 -> codes;  v -> codes       (r4dxb_attn_precore_kv4)
//   write     the same without q, norms and rotation                                        (Hq = 0, rotary_dim = 0)
//   read      bf16(n s + lo) of any positions of a sequence                                 (r4dxb_kv4_read)
//
// Codes of a group of 64 channels:  lo = min x,  s = bf16((max x - lo) / 15),  n = clamp(rint((x - lo) / s), 0, 15), with x the row's
// bf16 values brought into +-32768.  The minimum of bf16 values is one of them, so lo loses nothing; the codes are taken against
// the rounded s, so its rounding (2^-8) only clips the top code.  Quotients are those of IEEE divisions: the codes are those of any other
// program that follows the definition.  A group that holds a NaN gets s = NaN and reads back as NaN throughout.
#include <cmath>

#include "kv4.cuh"
#include "sm100_ptx.cuh"

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
  int steps, groups;           // rounds of heads that a warp takes at most, warps to a token
  float eps;
  double turn_exponent, turn_step;      // angle of channel pair i, in turns per position: 2^(turn_exponent + i turn_step)
};

// eight bf16 values as pairs, and back
__device__ __forceinline__ void Unpack8(const uint4& v, float2 (&x)[4]) {
  x[0] = make_float2(BfLo(v.x), BfHi(v.x));
  x[1] = make_float2(BfLo(v.y), BfHi(v.y));
  x[2] = make_float2(BfLo(v.z), BfHi(v.z));
  x[3] = make_float2(BfLo(v.w), BfHi(v.w));
}
__device__ __forceinline__ uint4 Pack8(const float2 (&x)[4]) {
  return make_uint4(PackBf16(x[0].x, x[0].y), PackBf16(x[1].x, x[1].y), PackBf16(x[2].x, x[2].y), PackBf16(x[3].x, x[3].y));
}
__device__ __forceinline__ uint4 Load8(const __nv_bfloat16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
__device__ __forceinline__ float2 Mul2(float2 a, float2 b) {
  float2 d;
  asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mul.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z; }"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// What a warp knows of its token.
struct Token {
  int t, tok, blk, lane, li;
  const float4* turns;         // [4][32 lanes] of shared memory: of two channels each, own value x (x, y) + the partner channel's x (z, w)
  float* rows;                 // [32 lanes][8] of shared memory
};

// Rounds of heads `first` .. (one, two or four at a time, lane / (D / 8)) of one kind: q (KIND 0), k (1) or v (2); AHEAD rounds in flight.
template <int D, int AHEAD, int KIND>
__device__ __forceinline__ void Heads(const PrecoreArgs& a, const Token& tk, int first, int rounds) {
  constexpr int LPH = D / 8, HPW = 32 / LPH;
  const int heads = KIND == 0 ? a.Hq : a.Hkv, li = tk.li, lane = tk.lane;
  const __nv_bfloat16* src = KIND == 0 ? a.qg + static_cast<size_t>(tk.t) * a.Hq * a.q_stride : (KIND == 1 ? a.k : a.v) + static_cast<size_t>(tk.t) * a.Hkv * D;
  const int step = KIND == 0 ? a.q_stride : D;
  const __nv_bfloat16* norm = KIND == 0 ? a.q_norm : (KIND == 1 ? a.k_norm : nullptr);
  float2 w[4];
  if (norm != nullptr) {
    Unpack8(Load8(norm + 8 * li), w);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = make_float2(1.0f + w[i].x, 1.0f + w[i].y);
  }
  // partner channels: by shuffle where they are a power of two of lanes away
  const int half = a.rotary_dim / 2, hop = half / 8;
  const bool shuffle = half % 8 == 0 && (hop & (hop - 1)) == 0;

  auto load = [&](int round) {
    const int head = first + round * HPW;
    return round < rounds && head < heads ? Load8(src + static_cast<size_t>(head) * step + 8 * li) : make_uint4(0u, 0u, 0u, 0u);
  };
  uint4 next[AHEAD];
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) next[u] = load(u);
#pragma unroll 1
  for (int round = 0; round < rounds; round += AHEAD) {
    float2 x[AHEAD][4];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      Unpack8(next[u], x[u]);
      next[u] = load(round + AHEAD + u);
    }
    if (KIND < 2 && norm != nullptr) {
      float ss[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        float2 p = Mul2(x[u][0], x[u][0]);
#pragma unroll
        for (int i = 1; i < 4; ++i) p = ptx::Fma2(x[u][i], x[u][i], p);
        ss[u] = p.x + p.y;
      }
#pragma unroll
      for (int o = 1; o < LPH; o <<= 1)
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) ss[u] += __shfl_xor_sync(0xffffffffu, ss[u], o);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const float r = rsqrtf(ss[u] * (1.0f / D) + a.eps);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[u][i] = Mul2(Mul2(x[u][i], make_float2(r, r)), w[i]);
      }
    }
    if (KIND < 2 && half > 0) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        float2 y[4];
        if (shuffle) {
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = make_float2(__shfl_xor_sync(0xffffffffu, x[u][i].x, hop), __shfl_xor_sync(0xffffffffu, x[u][i].y, hop));
          if (8 * li < a.rotary_dim) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float4 f = tk.turns[i * 32 + lane];
              x[u][i] = ptx::Fma2(x[u][i], make_float2(f.x, f.y), Mul2(y[i], make_float2(f.z, f.w)));
            }
          }
        } else {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<float2*>(tk.rows + lane * 8 + 2 * i) = x[u][i];
          __syncwarp();
          auto turn = [&](float& v, int d, float c, float s) {
            if (d < a.rotary_dim) v = fmaf(v, c, tk.rows[(lane - li) * 8 + (d < half ? d + half : d - half)] * s);
          };
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 f = tk.turns[i * 32 + lane];
            turn(x[u][i].x, 8 * li + 2 * i, f.x, f.z);
            turn(x[u][i].y, 8 * li + 2 * i + 1, f.y, f.w);
          }
        }
      }
    }
    if constexpr (KIND == 0) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int head = first + (round + u) * HPW;
        if (round + u < rounds && head < heads) *reinterpret_cast<uint4*>(a.q_out + (static_cast<size_t>(tk.t) * a.Hq + head) * D + 8 * li) = Pack8(x[u]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const uint4 bits = Pack8(x[u]);
        Unpack8(bits, x[u]);
        // the largest magnitudes of the two halves of the words: beyond the limit or no number at all?
        const uint32_t mag = __vmaxu2(__vmaxu2(bits.x & 0x7fff7fffu, bits.y & 0x7fff7fffu), __vmaxu2(bits.z & 0x7fff7fffu, bits.w & 0x7fff7fffu));
        const uint32_t top = max(mag >> 16, mag & 0xffffu);
        if (__any_sync(0xffffffffu, top > 0x4700u)) {           // 32768
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[u][i].x = fminf(fmaxf(x[u][i].x, -kv4::kLimit), kv4::kLimit);
            x[u][i].y = fminf(fmaxf(x[u][i].y, -kv4::kLimit), kv4::kLimit);
          }
        }
        float lo = fminf(fminf(fminf(x[u][0].x, x[u][0].y), fminf(x[u][1].x, x[u][1].y)), fminf(fminf(x[u][2].x, x[u][2].y), fminf(x[u][3].x, x[u][3].y)));
        float hi = fmaxf(fmaxf(fmaxf(x[u][0].x, x[u][0].y), fmaxf(x[u][1].x, x[u][1].y)), fmaxf(fmaxf(x[u][2].x, x[u][2].y), fmaxf(x[u][3].x, x[u][3].y)));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {        // the eight lanes of a group
          lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
          hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        const bool bad = (__ballot_sync(0xffffffffu, top > 0x7f80u) >> (lane & ~7) & 0xffu) != 0u;
        const __nv_bfloat16 sb = __float2bfloat16_rn(bad ? __int_as_float(0x7fc00000) : __fdiv_rn(hi - lo, 15.f));
        const float s = __bfloat162float(sb);
        // (x - lo) / s as the IEEE division gives it, without its branches: from the rounded reciprocal two steps of remainder and correction
        // (Markstein); scales near the bottom of the range are lifted first, which changes no quotient
        const float lift = s < 1e-18f ? 18446744073709551616.f : 1.f, sl = s * lift, inv = s > 0.f ? __frcp_rn(sl) : 0.f;
        uint32_t codes = 0u;
        auto code = [&](float v, int at) {
          const float d = (v - lo) * lift;
          float n = d * inv;
          n = fmaf(fmaf(-n, sl, d), inv, n);
          n = fmaf(fmaf(-n, sl, d), inv, n);
          n = fminf(fmaxf(n, 0.f), 15.f) + 12582912.f;          // 1.5 x 2^23: the integer, rounded to even at halves, in the lowest bits
          codes |= (__float_as_uint(n) & 15u) << (4 * at);
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          code(x[u][i].x, 2 * i);
          code(x[u][i].y, 2 * i + 1);
        }
        const int head = first + (round + u) * HPW;
        if (round + u < rounds && head < heads) {
          uint32_t* part = a.cache + ((static_cast<size_t>(tk.blk) * a.Hkv + head) * 2 + (KIND - 1)) * (kv4::Shape<D>::kPart / 4);
          part[kv4::Word<D, KIND == 2>(tk.tok, li)] = codes;
          if (li % 8 == 0)
            part[2 * D + tk.tok * kv4::Shape<D>::kGroups + li / 8] =
                static_cast<uint32_t>(__bfloat16_as_ushort(sb)) | static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(lo))) << 16;
        }
      }
    }
  }
}

// A warp has one token and some of its q, its k or its v heads: eight channels a lane, D / 8 lanes a head.  A channel pair's angle is position x
// frequency in turns, in 64 bits; what its whole turns leave fits 32 bits for the sine and cosine.
// What bounds many rows is the time between dependent instructions, so warps count: factors of the rotation in shared memory and 64 registers (32
// warps to an SM) took 8192 rows of 24 + 4 + 4 heads of 256 from 105 to 78 us, one round in flight instead of two is 83; one row 3.0 / 2.3 us.
template <int D, int AHEAD>
__global__ void __launch_bounds__(256, D == 256 || AHEAD == 1 ? 4 : 3) PrecoreKv4Kernel(PrecoreArgs a) {
  PdlEnter();
  constexpr int LPH = D / 8, HPW = 32 / LPH;
  extern __shared__ float smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, li = lane % LPH;
  const int task = blockIdx.x * 8 + warp, t = task / a.groups;
  if (t >= a.T) return;
  int part = task % a.groups;
  const int rounds_q = (a.Hq + HPW - 1) / HPW, rounds_kv = (a.Hkv + HPW - 1) / HPW;
  const int parts_q = (rounds_q + a.steps - 1) / a.steps, parts_kv = (rounds_kv + a.steps - 1) / a.steps;
  const int kind = part < parts_q ? 0 : (part < parts_q + parts_kv ? 1 : 2);
  part -= kind == 0 ? 0 : (kind == 1 ? parts_q : parts_q + parts_kv);
  const int pos = a.positions[t], half = a.rotary_dim / 2;
  Token tk;
  tk.t = t;
  tk.lane = lane;
  tk.li = li;
  tk.tok = pos & (kv4::kBlock - 1);
  tk.blk = -1;
  if (kind != 0) {
    const int slot = a.row_slot != nullptr ? a.row_slot[t] : 0;
    if (pos >= 0 && slot >= 0 && slot < a.slots) {
      kv4::Table table = a.table;
      table.entries += static_cast<size_t>(slot) * table.length;
      tk.blk = table.BlockAt(pos / kv4::kBlock);
    }
    if (tk.blk < 0) return;
  }
  // of a warp: [4][32] float4 of factors, [32 lanes][8] for channels that change lanes - before that the cosines and sines of the pairs
  float* own = smem + warp * (4 * 32 * 4 + 32 * 8);
  float4* turns = reinterpret_cast<float4*>(own);
  float* cs = own + 4 * 32 * 4;
  tk.turns = turns;
  tk.rows = cs;
  if (kind != 2) {
    for (int i = lane; i < half; i += 32) {
      const double turns = static_cast<double>(pos) * exp2(a.turn_exponent + i * a.turn_step);
      float s, c;
      sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
      cs[i] = c;
      cs[half + i] = s;
    }
    __syncwarp();
    auto turn = [&](int d, float& c, float& s) {
      const int j = d < half ? d : d - half;
      c = d < a.rotary_dim ? cs[j] : 1.f;
      s = d < a.rotary_dim ? (d < half ? -cs[half + j] : cs[half + j]) : 0.f;
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float4 f;
      turn(8 * li + 2 * i, f.x, f.z);
      turn(8 * li + 2 * i + 1, f.y, f.w);
      turns[i * 32 + lane] = f;
    }
    __syncwarp();                                // (the cosines are read: what follows may take their place)
  }
  const int first = part * a.steps * HPW + lane / LPH, rounds = min(a.steps, (kind == 0 ? rounds_q : rounds_kv) - part * a.steps);
  if (kind == 0) Heads<D, AHEAD, 0>(a, tk, first, rounds);
  else if (kind == 1) Heads<D, AHEAD, 1>(a, tk, first, rounds);
  else Heads<D, AHEAD, 2>(a, tk, first, rounds);
}

// Rows read back: a thread has one word (eight channels) of a row and up to ITEMS of its 2 Hkv heads' keys and values, whose codes and pairs it
// asks for at once.  (A thread per value word, each with the row's position and table entry to find first, took 62 us for 32517 rows of
// 8 heads of 128, this one 31; their bytes take 26.)
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
  const int per_round = 256 / D, rounds_q = (a.Hq + per_round - 1) / per_round, rounds_kv = (a.Hkv + per_round - 1) / per_round;
  const long long most = static_cast<long long>(a.T) * (rounds_q + 2 * rounds_kv) / (4 * 148 * 32);
  a.steps = static_cast<int>(most < 1 ? 1 : (most > 8 ? 8 : most));
  a.groups = (rounds_q + a.steps - 1) / a.steps + 2 * ((rounds_kv + a.steps - 1) / a.steps);
  const long long tasks = static_cast<long long>(a.T) * a.groups;
  if (tasks > 0x7fffffffll - 8) return R4DXB_TOO_LARGE;
  const size_t smem = 8 * (4 * 32 * 4 + 32 * 8) * sizeof(float);      // (D of the 256 floats hold a token's cosines and sines)
  const dim3 grid(static_cast<unsigned>((tasks + 7) / 8));
  return a.steps == 1 ? LaunchPdl(PrecoreKv4Kernel<D, 1>, grid, dim3(256), smem, s, a) : LaunchPdl(PrecoreKv4Kernel<D, 2>, grid, dim3(256), smem, s, a);
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
