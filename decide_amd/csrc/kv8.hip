// Rotary positions, the append to the 8-bit paged cache and the copying of its pages, for gfx950.
//
//   rope    y = rope(norm(x), pos): one workgroup a row, its heads dealt to groups of 16, 32 or 64 lanes (4 elements a
//           lane). The angle position * inv_freq is a product of a whole number and an fp32 one: exact in 64 bits up
//           to positions of 2^29, where in 32 bits it is off by half a turn's fraction already at 10^5. It is formed
//           and reduced to half turns in 64 bits, once per row and pair, and shared by the heads through LDS.
//   append  codes K and V rows into pages, a workgroup a block (16 tokens of one head, K or V).
//   copy    moves whole pages, 16 bytes a lane.
//
// Each value is read once and written once. Rotations of many rows and copies run at 90 % of a large copy's rate; the append
// does not: 2,307 rows of 4 heads of 256 take 14.4 us where their bytes take 4.4. Its workgroups read the row range, the
// position, the page and the started block one after another, each head's form the same angles in 64 bits, and V is read one
// element a lane; how much each of these costs was not measured apart.
#include <algorithm>
#include <cmath>

#include "kv8_device.h"

namespace dh {

namespace {
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef uint16_t us4 __attribute__((ext_vector_type(4)));

// N (1, 2 or 4) elements of dtype T (float, Half, Bf16), as they lie in memory and as floats. Loads come before the
// branches that use them, so that a wave's are all in flight at once.
struct Half {};
struct Bf16 {};
template <typename T, int N>
struct Raw {
  typedef std::conditional_t<std::is_same_v<T, float>, float, uint16_t> E;
  struct alignas(N * sizeof(E)) Pack {
    E e[N];
  } v;
  __device__ __forceinline__ void load(const void* base, size_t at) { v = *(const Pack*)((const E*)base + at); }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (std::is_same_v<T, float>)
      return v.e[i];
    else if constexpr (std::is_same_v<T, Half>)
      return (float)__builtin_bit_cast(_Float16, v.e[i]);
    else
      return __uint_as_float((uint32_t)v.e[i] << 16);
  }
};

__device__ __forceinline__ uint16_t to_bf16(float x) {
  const uint32_t u = __float_as_uint(x);
  if (x != x) return (uint16_t)(u >> 16 | 0x40);  // stays a NaN
  return (uint16_t)((u + 0x7fff + (u >> 16 & 1)) >> 16);
}

template <typename T>
__device__ __forceinline__ void store4(void* base, size_t at, const float* x) {
  if constexpr (std::is_same_v<T, float>)
    *(f4*)((float*)base + at) = f4{x[0], x[1], x[2], x[3]};
  else if constexpr (std::is_same_v<T, Half>)
    *(h4*)((_Float16*)base + at) = h4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
  else
    *(us4*)((uint16_t*)base + at) = us4{to_bf16(x[0]), to_bf16(x[1]), to_bf16(x[2]), to_bf16(x[3])};
}

// The angle pos * f in half turns, reduced to [-1, 1]; 1 / pi in two parts, so that far positions lose nothing.
__device__ __forceinline__ double half_turns(double pos, float f) {
  const double a = pos * (double)f;
  const double t = a * 0x1.45f306dc9c883p-2, low = fma(a, 0x1.45f306dc9c883p-2, -t) + a * -0x1.6b01ec5417056p-56;
  return t - 2.0 * rint(0.5 * t) + low;
}

// The value of the lane `ror` further on within its row of 16.
template <int ROR>
__device__ __forceinline__ uint32_t row_rotate(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + ROR, 0xf, 0xf, false);
}
template <int ROR, typename R>
__device__ __forceinline__ R rotated(R x) {
  if constexpr (sizeof(R) == 4) {
    return __builtin_bit_cast(R, row_rotate<ROR>(__builtin_bit_cast(uint32_t, x)));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    return __builtin_bit_cast(R, (uint64_t)row_rotate<ROR>((uint32_t)u) | (uint64_t)row_rotate<ROR>((uint32_t)(u >> 32)) << 32);
  }
}
// x of the lanes that differ in bit 4 (H = 16) or 5 (32), combined by f
template <int H, typename R, typename F>
__device__ __forceinline__ R across(R x, F f) {
  auto swap = [](uint32_t v) {
    if constexpr (H == 16)
      return __builtin_amdgcn_permlane16_swap(v, v, false, false);
    else
      return __builtin_amdgcn_permlane32_swap(v, v, false, false);
  };
  if constexpr (sizeof(R) == 4) {
    const auto p = swap(__builtin_bit_cast(uint32_t, x));
    return f(__builtin_bit_cast(R, (uint32_t)p[0]), __builtin_bit_cast(R, (uint32_t)p[1]));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const auto lo = swap((uint32_t)u), hi = swap((uint32_t)(u >> 32));
    return f(__builtin_bit_cast(R, (uint64_t)lo[0] | (uint64_t)hi[0] << 32),
             __builtin_bit_cast(R, (uint64_t)lo[1] | (uint64_t)hi[1] << 32));
  }
}
// f over the W (16, 32 or 64) lanes of a group, in every lane: register moves, no LDS
template <int W, typename R, typename F>
__device__ __forceinline__ R reduce(R x, F f) {
  x = f(x, rotated<8>(x));
  x = f(x, rotated<4>(x));
  x = f(x, rotated<2>(x));
  x = f(x, rotated<1>(x));
  if constexpr (W >= 32) x = across<16>(x, f);
  if constexpr (W >= 64) x = across<32>(x, f);
  return x;
}

// How a lane's elements d .. d + 3 of a head are normed and turned: their weights and where their pairs are. `quick`:
// all four turn or none does, and their pairs lie in one other lane or in this one.
template <typename R>
struct Turn {
  R w[4], wo[4];     // weights of the four and of what they pair with (1 without a norm)
  uint32_t d, pair;  // pair: the first's number
  uint32_t partner;  // the lane that holds what they pair with
  bool quick, turns, first;
  __device__ __forceinline__ void init(const RopeArgs& p, uint32_t lane, uint32_t width, R add) {
    d = 4 * lane;
    quick = p.interleaved ? p.rot % 4 == 0 : p.rot % 8 == 0;
    turns = d < p.rot;
    first = d < p.rot / 2;
    pair = p.interleaved ? d / 2 : first ? d : d - p.rot / 2;
    partner = p.interleaved || !turns ? lane : first ? lane + p.rot / 8 : lane - p.rot / 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = p.norm_w && d < width ? (R)p.norm_w[d + i] + add : (R)1;
      wo[i] = p.norm_w && d < width ? (R)p.norm_w[4 * partner % width + i] + add : (R)1;
    }
  }
};

// Normed and turned: x the lane's own values, at base[at + d] in memory, inv the head's norm factor, cs (cos, sin) of
// each pair. Every lane of the head's group calls it. The products and sums are spelled out, so that the same row gets
// the same bits wherever it stands.
template <typename T, int W, typename R>
__device__ __forceinline__ void turn4(const float* x, const void* base, size_t at, const RopeArgs& p, const Turn<R>& t,
                                      R inv, R (*cs)[2], R* y) {
  auto low = [](R a, R c, R b, R s) { return fma(a, c, -(b * s)); };
  auto high = [](R a, R c, R b, R s) { return fma(a, c, b * s); };
  R z[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = z[i] = (R)x[i] * (inv * t.w[i]);
  if (t.quick) {
    if (p.interleaved) {
      if (t.turns) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const R c = cs[t.pair + i / 2][0], s = cs[t.pair + i / 2][1];
          y[i] = low(z[i], c, z[i + 1], s);
          y[i + 1] = high(z[i + 1], c, z[i], s);
        }
      }
    } else {
      R o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = (R)__shfl(x[i], (int)t.partner, W) * (inv * t.wo[i]);
      if (t.turns) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const R c = cs[t.pair + i][0], s = cs[t.pair + i][1];
          y[i] = t.first ? low(z[i], c, o[i], s) : high(z[i], c, o[i], s);
        }
      }
    }
    return;
  }
  const uint32_t half = p.rot / 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t e = t.d + i;
    if (e >= p.rot) continue;
    const uint32_t with = p.interleaved ? e ^ 1 : e < half ? e + half : e - half;
    const bool first = p.interleaved ? !(e & 1) : e < half;
    const uint32_t pair = p.interleaved ? e / 2 : first ? e : e - half;
    Raw<T, 1> r;
    r.load(base, at + with);  // in the lines that this wave has just read
    const R o = (R)r[0] * (inv * (p.norm_w ? (R)p.norm_w[with] + (R)(p.add_one ? 1 : 0) : (R)1));
    const R c = cs[pair][0], s = cs[pair][1];
    y[i] = first ? low(z[i], c, o, s) : high(z[i], c, o, s);
  }
}

// 1 / sqrt(mean of squares + eps) over a head held 4 elements a lane by W lanes
template <int W, typename R>
__device__ __forceinline__ R norm_factor(const float* x, uint32_t head_dim, float eps) {
  R ss = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) ss = fma((R)x[i], (R)x[i], ss);
  ss = reduce<W>(ss, [](R a, R b) { return a + b; });
  if constexpr (std::is_same_v<R, double>)
    return rsqrt(ss / (double)head_dim + (double)eps);
  else
    return 1.0f / sqrtf(ss / (float)head_dim + eps);
}

// ---- rope ----------------------------------------------------------------------------------------------------------
template <typename TX, typename TY, int W>
__global__ __launch_bounds__(256) void rope_kernel(const void* x, uint32_t ldx, void* y, uint32_t ldy,
                                                   const uint32_t* __restrict__ pos, uint32_t heads, RopeArgs p) {
  constexpr uint32_t kAtOnce = 4;  // heads that a group of lanes has in flight
  __shared__ float cs[128][2];
  const uint32_t r = blockIdx.x, tid = threadIdx.x, lane = tid % W;
  const bool mine = 4 * lane < p.head_dim;
  const uint32_t d = mine ? 4 * lane : 0;
  Raw<TX, 4> raw[kAtOnce];
  auto load = [&](uint32_t h0) {
#pragma unroll
    for (uint32_t j = 0; j < kAtOnce; ++j) {
      const uint32_t h = min(h0 + j * (256 / W), heads - 1);
      raw[j].load(x, (size_t)r * ldx + (size_t)h * p.head_dim + d);
    }
  };
  load(tid / W);
  Turn<float> turn;
  turn.init(p, lane, p.head_dim, p.add_one ? 1.f : 0.f);
  if (tid < p.rot / 2) {
    const double t = half_turns((double)pos[r], p.inv_freq[tid]);
    float s, c;
    sincospif((float)t, &s, &c);
    cs[tid][0] = c * p.amp;
    cs[tid][1] = s * p.amp;
  }
  __syncthreads();
  for (uint32_t h0 = tid / W; h0 < heads; h0 += kAtOnce * (256 / W)) {
    if (h0 != tid / W) load(h0);
    float o[kAtOnce][4];
#pragma unroll
    for (uint32_t j = 0; j < kAtOnce; ++j) {
      const uint32_t h = min(h0 + j * (256 / W), heads - 1);
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = mine ? raw[j][i] : 0.f;
      const float inv = p.norm_w ? norm_factor<W, float>(v, p.head_dim, p.eps) : 1.0f;
      turn4<TX, W, float>(v, x, (size_t)r * ldx + (size_t)h * p.head_dim, p, turn, inv, cs, o[j]);
    }
    __builtin_amdgcn_wave_barrier();  // y may be x: every lane has read its pairs before one stores
#pragma unroll
    for (uint32_t j = 0; j < kAtOnce; ++j) {
      const uint32_t h = h0 + j * (256 / W);
      if (mine && h < heads) store4<TY>(y, (size_t)r * ldy + (size_t)h * p.head_dim + d, o[j]);
    }
  }
}

// ---- append --------------------------------------------------------------------------------------------------------
constexpr float kMinScale = 0x1p-100f;

// The scale of a block whose largest magnitude is amax.
template <bool INT8>
__device__ __forceinline__ float block_scale(float amax) {
  if constexpr (INT8) {
    return fmaxf(amax * (1.0f / 127.0f), kMinScale);
  } else {
    // amax = m 2^e, m in [1/2, 1): at most 448 2^x = 0.875 2^(9 + x) from x = e - 9 on, or e - 8 where m > 0.875
    if (!(amax > 0.0f)) return kMinScale;
    int e;
    const float m = frexpf(amax, &e);
    return fmaxf(ldexpf(1.0f, e - 9 + (m > 0.875f)), kMinScale);
  }
}

// x / scale, correctly rounded, with inv = 1 / scale correctly rounded: a power of two has an exact reciprocal; otherwise
// the product's remainder, exact in a fused multiply-add, corrects it (Markstein's division).
template <bool INT8>
__device__ __forceinline__ float scaled(float x, float scale, float inv) {
  const float q = x * inv;
  return INT8 ? fmaf(fmaf(-q, scale, x), inv, q) : q;
}

// Four values, divided by their scale, as code bytes (round to nearest even; e4m3 to e4m3 in the hardware's conversion).
template <bool INT8>
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d) {
  if constexpr (INT8) {
    auto one = [](float v) { return (uint32_t)(int)(rintf(v) + 128.0f); };
    return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
  } else {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
  }
}

// The numbers that four code bytes stand for, without their scale.
template <bool INT8>
__device__ __forceinline__ void values4(uint32_t u, float* v) {
  if constexpr (INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)(u >> 8 * i & 255) - 128.0f;
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)u, true);
    v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
  }
}

template <bool INT8>
__device__ __forceinline__ uint32_t recode4(uint32_t u, float ratio) {
  float v[4];
  values4<INT8>(u, v);
  return code4<INT8>(v[0] * ratio, v[1] * ratio, v[2] * ratio, v[3] * ratio);
}

// What a wave's values say to its block: their largest magnitude, NaN where one is not finite.
template <int N>
__device__ __forceinline__ float wave_amax(const float* x) {
  float amax = 0.f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    amax = fmaxf(amax, fabsf(x[i]));
    finite = finite && fabsf(x[i]) < INFINITY;
  }
  amax = reduce<64>(amax, [](float a, float b) { return fmaxf(a, b); });
  return __all(finite) ? amax : NAN;
}

// A workgroup is one block (16 tokens of one head, K or V). K: a wave takes four tokens, 4 dims a lane. V: a thread takes
// one dim of 16, 8 or 4 tokens (D = 256, 128, 64), which are consecutive bytes. The waves meet once, over the largest
// magnitude. With a wave per block, and so four times fewer waves with four times the work each, 2,307 rows of 4 heads
// of 256 took 18.7 us against 14.0, one row of each of 64 sequences 12.4 against 7.4.
template <typename T, int D, bool INT8>
__global__ __launch_bounds__(256) void kv8_append_kernel(KvArgs a, const void* __restrict__ k, uint32_t ldk,
                                                         const void* __restrict__ v, uint32_t ldv, RopeArgs rope,
                                                         uint32_t at_once) {
  extern __shared__ __attribute__((aligned(16))) double angles[];  // (cos, sin) [4 waves][4 tokens][rot / 2]
  __shared__ float amax[2][4];
  const uint32_t groups = (a.kv_heads + at_once - 1) / at_once;
  const bool is_v = blockIdx.y >= groups;
  const uint32_t head0 = blockIdx.y % groups * at_once, head1 = min(head0 + at_once, a.kv_heads);
  uint32_t r0, r1;
  const uint32_t s = kv_find_seq(a.row0, a.seqs, a.rows, blockIdx.x, 1, kKvBlock, 2, r0, r1);
  if (s >= a.seqs || r1 <= r0) return;
  const uint64_t p0 = a.qpos[r0], p1 = p0 + (r1 - r0);  // the tokens p0 .. p1 - 1 are new
  const uint64_t t0 = (p0 / kKvBlock + (blockIdx.x - (r0 / kKvBlock + 2 * s))) * kKvBlock;  // the block's first token
  const uint64_t page = t0 / kKvPage;
  if (p0 == 0xffffffffu || page >= a.ld_table || t0 >= p1) return;
  const uint32_t id = a.table[(size_t)s * a.ld_table + page];
  if (id >= a.pages) return;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, block = (uint32_t)(t0 % kKvPage) / kKvBlock;
  uint8_t* const rec = a.pool + id * a.page_bytes;
  auto scale_of = [&](uint32_t head) {
    return (float*)(rec + kv_scale_at<D>(head, a.kv_heads)) + (is_v ? 4 : 0) + block;
  };
  const uint32_t kept = p0 > t0 ? (uint32_t)(p0 - t0) : 0;                    // earlier tokens of the block
  const uint32_t end = p1 < t0 + kKvBlock ? (uint32_t)(p1 - t0) : kKvBlock;  // its new tokens are kept .. end - 1
  const size_t row = r0 + (size_t)(t0 - p0);  // the row of the block's token 0 (wraps below zero before row r0)
  auto row_of = [&](uint32_t t) { return row + min(max(t, kept), end - 1); };  // one of the call's in place of others

  // the block's scale, once the waves have left what they say
  auto block_scale_now = [&](uint32_t head, float before, float mine) {
    float* const said = amax[head % 2];  // what the head before left is read by now, not what this one's will
    if (lane == 0) said[wave] = mine;
    __syncthreads();
    const float a0 = said[0], a1 = said[1], a2 = said[2], a3 = said[3];
    const float sum = a0 + a1 + a2 + a3;  // NaN where one is
    const float fresh = block_scale<INT8>(fmaxf(fmaxf(a0, a1), fmaxf(a2, a3)));
    const float sc = sum != sum || (kept && before != before) ? NAN : kept ? fmaxf(fresh, before) : fresh;
    if (tid == 0) *scale_of(head) = sc;
    return sc;
  };

  if (is_v) {
    constexpr int N = kKvBlock * D / 256;  // tokens of a thread
    const uint32_t d = tid % D, tok = tid / D * N;
    struct alignas(N) Words {
      uint32_t w[N / 4];
    };
    Raw<T, 1> raw[N];
    auto load = [&](uint32_t head) {
#pragma unroll
      for (int t = 0; t < N; ++t) raw[t].load(v, row_of(tok + t) * ldv + head * D + d);
    };
    load(head0);
    for (uint32_t head = head0; head < head1; ++head) {
      Words* const at = (Words*)(rec + kv_v_at<D>(head, a.kv_heads) + (size_t)d * kKvPage + block * kKvBlock + tok);
      Words old{};
      float before = 0.f;
      if (kept) old = *at, before = *scale_of(head);
      float x[N];
#pragma unroll
      for (int t = 0; t < N; ++t) x[t] = tok + t >= kept && tok + t < end ? raw[t][0] : 0.f;
      load(min(head + 1, head1 - 1));
      const float sc = block_scale_now(head, before, wave_amax<N>(x));
      const float inv = 1.0f / sc, ratio = before / sc;
      Words out;
#pragma unroll
      for (int w = 0; w < N / 4; ++w) {
        float q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = sc == sc ? scaled<INT8>(x[4 * w + i], sc, inv) : 0.f;
        const int stay = (int)kept - (int)tok - 4 * w;  // bytes of tokens that stay
        const uint32_t m = stay >= 4 ? ~0u : stay <= 0 ? 0u : (1u << 8 * stay) - 1u;
        uint32_t o = old.w[w];
        if (kept && sc > before) o = recode4<INT8>(o, ratio);
        out.w[w] = (o & m) | (code4<INT8>(q[0], q[1], q[2], q[3]) & ~m);
      }
      *at = out;
    }
    return;
  }

  constexpr int W = D / 4;   // lanes of a key
  constexpr int TP = 64 / W;  // keys a wave reads at once
  constexpr int P = 4 / TP;   // passes over its four: pass n holds token 4 wave + n TP + lane / W
  const uint32_t d = 4 * (lane % W);
  auto token = [&](int n) { return 4 * wave + n * TP + lane / W; };
  Raw<T, 4> raw[P];
  auto load = [&](uint32_t head) {
#pragma unroll
    for (int n = 0; n < P; ++n) raw[n].load(k, row_of(token(n)) * ldk + head * D + d);
  };
  load(head0);
  const bool turning = rope.inv_freq && 4 * wave < end && 4 * wave + 4 > kept;
  const uint32_t pairs = rope.rot / 2;
  double(*const cs)[2] = (double(*)[2])angles + (size_t)wave * 4 * pairs;
  Turn<double> turn;
  if (turning) {
    turn.init(rope, lane % W, D, rope.add_one ? 1.0 : 0.0);
    for (uint32_t i = lane; i < 4 * pairs; i += 64) {
      const uint32_t pair = i % pairs, t = 4 * wave + i / pairs;
      if (t < kept || t >= end) continue;
      double sn, c;
      sincospi(half_turns((double)(t0 + t), rope.inv_freq[pair]), &sn, &c);
      cs[i][0] = c * (double)rope.amp;
      cs[i][1] = sn * (double)rope.amp;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // this wave's own reads follow
    __builtin_amdgcn_wave_barrier();
  }
  const bool stays = tid * 16 / D < kept;  // the thread's 16 bytes of the block as it was, which are one token's
  for (uint32_t head = head0; head < head1; ++head) {
    uint8_t* const base = rec + kv_k_at<D>(head) + (size_t)block * kKvBlock * D;
    u4 old = u4{0, 0, 0, 0};
    float before = 0.f;
    if (stays) old = *(const u4*)(base + tid * 16);
    if (kept) before = *scale_of(head);
    float x[P][4];
#pragma unroll
    for (int n = 0; n < P; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[n][i] = raw[n][i];
    load(min(head + 1, head1 - 1));
    if (turning) {
#pragma unroll
      for (int n = 0; n < P; ++n) {
        if (4 * wave + n * TP >= end || 4 * wave + n * TP + TP <= kept) continue;
        const double inv = rope.norm_w ? norm_factor<W, double>(x[n], D, rope.eps) : 1.0;
        double y[4];
        turn4<T, W, double>(x[n], k, row_of(token(n)) * ldk + head * D, rope, turn, inv, cs + token(n) % 4 * pairs, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[n][i] = (float)y[i];
      }
    }
#pragma unroll
    for (int n = 0; n < P; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[n][i] = token(n) >= kept && token(n) < end ? x[n][i] : 0.f;
    const float sc = block_scale_now(head, before, wave_amax<P * 4>(&x[0][0]));
    const float inv = 1.0f / sc;
    if (stays && sc > before) {
      const float ratio = before / sc;
      u4 now;
#pragma unroll
      for (int w = 0; w < 4; ++w) now[w] = recode4<INT8>(old[w], ratio);
      *(u4*)(base + tid * 16) = now;
    }
#pragma unroll
    for (int n = 0; n < P; ++n) {
      float q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = sc == sc ? scaled<INT8>(x[n][i], sc, inv) : 0.f;
      if (token(n) >= kept) *(uint32_t*)(base + token(n) * D + d) = code4<INT8>(q[0], q[1], q[2], q[3]);
    }
  }
}

// ---- copy ----------------------------------------------------------------------------------------------------------
constexpr uint32_t kCopyBytes = 16384;  // of a workgroup

__global__ __launch_bounds__(256) void kv8_copy_pages_kernel(uint8_t* pool, uint64_t page_bytes, uint32_t pages,
                                                             const uint32_t* __restrict__ src,
                                                             const uint32_t* __restrict__ dst, uint32_t n,
                                                             uint32_t chunks) {
  const uint32_t chunk = blockIdx.x % chunks, pair = blockIdx.x / chunks % n, layer = blockIdx.x / chunks / n;
  const uint32_t from = src[pair], to = dst[pair];
  if (from >= pages || to >= pages) return;
  uint8_t* const base = pool + (uint64_t)layer * pages * page_bytes;
  const u4* in = (const u4*)(base + from * page_bytes);
  u4* out = (u4*)(base + to * page_bytes);
  const uint32_t words = (uint32_t)(page_bytes / 16), at = chunk * (kCopyBytes / 16) + threadIdx.x;
  u4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + 256 * i < words) v[i] = in[at + 256 * i];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + 256 * i < words) out[at + 256 * i] = v[i];
}
}  // namespace

hipError_t launch_rope(const void* x, uint32_t ldx, uint32_t x_dtype, void* y, uint32_t ldy, uint32_t y_dtype,
                       const uint32_t* pos, uint32_t rows, uint32_t heads, const RopeArgs& p, hipStream_t s) {
  if (rows == 0 || heads == 0) return hipSuccess;
  auto go = [&](auto tx, auto ty) {
    using TX = decltype(tx);
    using TY = decltype(ty);
    if (p.head_dim <= 64)
      hipLaunchKernelGGL((rope_kernel<TX, TY, 16>), dim3(rows), dim3(256), 0, s, x, ldx, y, ldy, pos, heads, p);
    else if (p.head_dim <= 128)
      hipLaunchKernelGGL((rope_kernel<TX, TY, 32>), dim3(rows), dim3(256), 0, s, x, ldx, y, ldy, pos, heads, p);
    else
      hipLaunchKernelGGL((rope_kernel<TX, TY, 64>), dim3(rows), dim3(256), 0, s, x, ldx, y, ldy, pos, heads, p);
  };
  auto to = [&](auto tx) {
    if (y_dtype == 0)
      go(tx, Half{});
    else if (y_dtype == 1)
      go(tx, Bf16{});
    else
      go(tx, float{});
  };
  if (x_dtype == 0)
    to(Half{});
  else if (x_dtype == 1)
    to(Bf16{});
  else
    to(float{});
  return hipGetLastError();
}

namespace {
template <typename T, bool INT8>
void append_dim(const KvArgs& a, uint32_t head_dim, const void* k, uint32_t ldk, const void* v, uint32_t ldv,
                const RopeArgs& p, uint32_t cus, hipStream_t s) {
  // A workgroup takes one head after another where there would be more of them than run at once (four a CU):
  // 385 blocks of 8 heads 21.4 us with one head each, 17.0 with four, 15.9 with eight; 146 blocks of 4 heads 14.0 with one,
  // 15.9 with two.
  const uint64_t single = ((uint64_t)a.rows / kKvBlock + a.seqs) * 2 * a.kv_heads;
  const uint32_t at_once = (uint32_t)std::min<uint64_t>(a.kv_heads, std::max<uint64_t>(1, single / (4ull * cus)));
  const dim3 grid(a.rows / kKvBlock + 2 * a.seqs, 2 * ((a.kv_heads + at_once - 1) / at_once));
  const size_t lds = p.inv_freq ? (size_t)4 * 4 * (p.rot / 2) * 2 * sizeof(double) : 0;
  if (head_dim == 64)
    hipLaunchKernelGGL((kv8_append_kernel<T, 64, INT8>), grid, dim3(256), lds, s, a, k, ldk, v, ldv, p,
                       at_once);
  else if (head_dim == 128)
    hipLaunchKernelGGL((kv8_append_kernel<T, 128, INT8>), grid, dim3(256), lds, s, a, k, ldk, v, ldv, p,
                       at_once);
  else
    hipLaunchKernelGGL((kv8_append_kernel<T, 256, INT8>), grid, dim3(256), lds, s, a, k, ldk, v, ldv, p,
                       at_once);
}
template <typename T>
void append_format(const KvArgs& a, uint32_t head_dim, bool int8, const void* k, uint32_t ldk, const void* v,
                   uint32_t ldv, const RopeArgs& p, uint32_t cus, hipStream_t s) {
  if (int8)
    append_dim<T, true>(a, head_dim, k, ldk, v, ldv, p, cus, s);
  else
    append_dim<T, false>(a, head_dim, k, ldk, v, ldv, p, cus, s);
}
}  // namespace

hipError_t launch_kv8_append(const KvArgs& a, uint32_t head_dim, bool int8, const void* k, uint32_t ldk, const void* v,
                             uint32_t ldv, uint32_t dtype, const RopeArgs& p, uint32_t cus, hipStream_t s) {
  if (a.rows == 0 || a.seqs == 0) return hipSuccess;
  if (dtype == 0)
    append_format<Half>(a, head_dim, int8, k, ldk, v, ldv, p, cus, s);
  else if (dtype == 1)
    append_format<Bf16>(a, head_dim, int8, k, ldk, v, ldv, p, cus, s);
  else
    append_format<float>(a, head_dim, int8, k, ldk, v, ldv, p, cus, s);
  return hipGetLastError();
}

hipError_t launch_kv8_copy_pages(uint8_t* pool, uint64_t page_bytes, uint32_t pages, uint32_t layers,
                                 const uint32_t* src, const uint32_t* dst, uint32_t n, hipStream_t s) {
  if (n == 0 || layers == 0) return hipSuccess;
  const uint32_t chunks = (uint32_t)((page_bytes + kCopyBytes - 1) / kCopyBytes);
  hipLaunchKernelGGL(kv8_copy_pages_kernel, dim3(chunks * n * layers), dim3(256), 0, s, pool, page_bytes, pages, src,
                     dst, n, chunks);
  return hipGetLastError();
}

}  // namespace dh
