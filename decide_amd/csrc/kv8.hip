// Rotary positions, the append to the 8-bit paged cache and the copying of its pages, for gfx950.
//
//   rope    y = rope(norm(x), pos): one workgroup a row, its heads dealt to groups of 16, 32 or 64 lanes (4 elements a
//           lane). The angle position * inv_freq is a product of a whole number and an fp32 one: exact in 64 bits up
//           to positions of 2^29, where in 32 bits it is off by half a turn's fraction already at 10^5. It is formed
//           and reduced to half turns in 64 bits, once per row and pair, and shared by the heads through LDS.
//   append  codes K and V rows into pages. A wave takes one block (16 tokens of one head, K or V), so the largest
//           magnitude, the scale, the earlier tokens' new codes and the stores need no other wave.
//   copy    moves whole pages, 16 bytes a lane.
//
// All three are bound by memory: each value is read once and written once.
#include <cmath>

#include "kv8_device.h"

namespace dh {

namespace {
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef uint16_t us4 __attribute__((ext_vector_type(4)));

// N (1, 2 or 4) elements of dtype T as floats
struct Half {};
struct Bf16 {};

template <typename T, int N>
__device__ __forceinline__ void load_n(const void* base, size_t at, float* out) {
  typedef std::conditional_t<std::is_same_v<T, float>, float, uint16_t> E;
  struct alignas(N * sizeof(E)) Pack {
    E e[N];
  };
  const Pack x = *(const Pack*)((const E*)base + at);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (std::is_same_v<T, float>)
      out[i] = x.e[i];
    else if constexpr (std::is_same_v<T, Half>)
      out[i] = (float)__builtin_bit_cast(_Float16, x.e[i]);
    else
      out[i] = __uint_as_float((uint32_t)x.e[i] << 16);
  }
}

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

// R(1) / sqrt(mean of squares + eps) over a head held 4 elements a lane by W lanes
template <int W, typename R>
__device__ __forceinline__ R norm_factor(const float* x, uint32_t head_dim, float eps) {
  R ss = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) ss += (R)x[i] * (R)x[i];
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, W);
  if constexpr (std::is_same_v<R, double>)
    return 1.0 / sqrt(ss / (double)head_dim + (double)eps);
  else
    return 1.0f / sqrtf(ss / (float)head_dim + eps);
}

// The lane's elements d .. d + 3 of a head, normed and turned. x: the lane's own values; base[at ..]: the head (the
// values that x pairs with are read there again: they lie in the lines that this wave has just read); cs: (cos, sin) of
// each pair.
template <typename T, typename R>
__device__ __forceinline__ void rope4(const float* x, const void* base, size_t at, uint32_t d, const RopeArgs& p, R inv,
                                      R (*cs)[2], R* y) {
  const uint32_t half = p.rot / 2;
  auto weight = [&](uint32_t e) { return p.norm_w ? inv * ((R)p.norm_w[e] + (R)(p.add_one ? 1 : 0)) : (R)1; };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t e = d + i;
    y[i] = (R)x[i] * weight(e);
    if (e < p.rot) {
      R other;
      uint32_t pair;
      bool first;
      if (p.interleaved) {
        pair = e / 2;
        first = !(e & 1);
        other = (R)x[i ^ 1] * weight(e ^ 1);
      } else {
        first = e < half;
        pair = first ? e : e - half;
        const uint32_t o = first ? e + half : e - half;
        float ox;
        load_n<T, 1>(base, at + o, &ox);
        other = (R)ox * weight(o);
      }
      const R c = cs[pair][0], s = cs[pair][1];
      y[i] = first ? y[i] * c - other * s : y[i] * c + other * s;
    }
  }
}

// ---- rope ----------------------------------------------------------------------------------------------------------
template <typename TX, typename TY, int W>
__global__ __launch_bounds__(256) void rope_kernel(const void* x, uint32_t ldx, void* y, uint32_t ldy,
                                                   const uint32_t* __restrict__ pos, uint32_t heads, RopeArgs p) {
  __shared__ float cs[128][2];
  const uint32_t r = blockIdx.x, tid = threadIdx.x;
  if (tid < p.rot / 2) {
    const double t = half_turns(pos[r], p.inv_freq[tid]);
    float s, c;
    sincospif((float)t, &s, &c);
    cs[tid][0] = c * p.amp;
    cs[tid][1] = s * p.amp;
  }
  __syncthreads();
  const uint32_t d = 4 * (tid % W);
  for (uint32_t h = tid / W; h < heads; h += 256 / W) {
    const size_t at = (size_t)r * ldx + (size_t)h * p.head_dim;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (d < p.head_dim) load_n<TX, 4>(x, at + d, v);
    const float inv = p.norm_w ? norm_factor<W, float>(v, p.head_dim, p.eps) : 1.0f;
    float o[4];
    if (d < p.head_dim) rope4<TX, float>(v, x, at, d, p, inv, cs, o);
    __builtin_amdgcn_wave_barrier();  // y may be x: every lane has read its pairs before one stores
    if (d < p.head_dim) store4<TY>(y, (size_t)r * ldy + (size_t)h * p.head_dim + d, o);
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

// x / scale; a scale that is a power of two has an exact reciprocal.
template <bool INT8>
__device__ __forceinline__ float scaled(float x, float scale, float inv) {
  return INT8 ? x / scale : x * inv;
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

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
  return x;
}

// Largest magnitude of a wave's values and whether all are finite, then the block's scale: `keep` tokens stay with theirs.
template <bool INT8, int N>
__device__ __forceinline__ float new_scale(const float* x, bool keep, float before) {
  float amax = 0.f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    amax = fmaxf(amax, fabsf(x[i]));
    finite = finite && fabsf(x[i]) < INFINITY;
  }
  const float s = block_scale<INT8>(wave_max(amax));
  if (!__all(finite) || (keep && before != before)) return NAN;
  return keep ? fmaxf(s, before) : s;
}

// A workgroup is one page of one sequence x one head x K or V, a wave one block of the page.
template <typename T, int D, bool INT8>
__global__ __launch_bounds__(256) void kv8_append_kernel(KvArgs a, const void* __restrict__ k, uint32_t ldk,
                                                         const void* __restrict__ v, uint32_t ldv, RopeArgs rope) {
  constexpr int W = D / 4;        // lanes of a key
  constexpr int TP = 64 / W;      // keys a wave reads at once
  constexpr int P = kKvBlock / TP;  // passes over a block's keys
  __shared__ double cs[4][4][128][2];
  const uint32_t head = blockIdx.y % a.kv_heads;
  const bool is_v = blockIdx.y >= a.kv_heads;
  const uint32_t s = kv_find_seq(a.row0, a.seqs, a.rows, blockIdx.x, 1, kKvPage, 2);
  if (s >= a.seqs) return;
  const uint32_t r0 = min(a.row0[s], a.rows), r1 = min(a.row0[s + 1], a.rows);
  if (r1 <= r0) return;
  const uint64_t p0 = a.qpos[r0], p1 = p0 + (r1 - r0);  // the tokens p0 .. p1 - 1 are new
  const uint64_t page = p0 / kKvPage + (blockIdx.x - (r0 / kKvPage + 2 * s));
  const uint32_t lane = threadIdx.x & 63, block = threadIdx.x >> 6;
  const uint64_t t0 = page * kKvPage + block * kKvBlock;  // the block's first token
  if (p0 == 0xffffffffu || page >= a.ld_table || t0 >= p1 || t0 + kKvBlock <= p0) return;
  const uint32_t id = a.table[(size_t)s * a.ld_table + page];
  if (id >= a.pages) return;
  uint8_t* const rec = a.pool + id * a.page_bytes;
  float* const scale = (float*)(rec + kv_scale_at<D>(head, a.kv_heads)) + (is_v ? 4 : 0) + block;
  const uint32_t kept = p0 > t0 ? (uint32_t)(p0 - t0) : 0;                      // earlier tokens of the block
  const uint32_t end = p1 < t0 + kKvBlock ? (uint32_t)(p1 - t0) : kKvBlock;  // its new tokens are kept .. end - 1
  const float before = kept ? *scale : 0.f;
  const size_t row = r0 + (size_t)(t0 - p0);  // the row of the block's token 0 (wraps below zero before row r0)
  constexpr uint32_t kZero = INT8 ? 0x80808080u : 0u;

  if (is_v) {
    constexpr int C = D / 64;  // dims of a lane, all 16 tokens
    const uint32_t d = lane * C;
    float x[kKvBlock][C];
#pragma unroll
    for (uint32_t t = 0; t < kKvBlock; ++t) {
#pragma unroll
      for (int c = 0; c < C; ++c) x[t][c] = 0.f;
      if (t >= kept && t < end) load_n<T, C>(v, (row + t) * ldv + head * D + d, x[t]);
    }
    const float sc = new_scale<INT8, kKvBlock * C>(&x[0][0], kept != 0, before);
    const float ratio = before / sc, inv = 1.0f / sc;
    if (lane == 0) *scale = sc;
    uint8_t* const at = rec + kv_v_at<D>(head, a.kv_heads) + (size_t)d * kKvPage + block * kKvBlock;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      u4 out, old = u4{0, 0, 0, 0};
      if (kept) old = *(const u4*)(at + c * kKvPage);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = sc == sc ? scaled<INT8>(x[4 * w + i][c], sc, inv) : 0.f;
        const uint32_t fresh = code4<INT8>(q[0], q[1], q[2], q[3]);
        const uint32_t stay = sc == before || sc != sc ? old[w] : recode4<INT8>(old[w], ratio);
        uint32_t m = 0;  // bytes of tokens that stay
#pragma unroll
        for (int i = 0; i < 4; ++i) m |= 4 * w + i < (int)kept ? 255u << 8 * i : 0u;
        out[w] = (stay & m) | (fresh & ~m);
      }
      *(u4*)(at + c * kKvPage) = out;
    }
    return;
  }

  const uint32_t d = 4 * (lane % W);
  float x[P][4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {  // four tokens share a table of angles
    if (rope.inv_freq && 4u * g < end && 4u * g + 4 > kept) {
      for (uint32_t i = lane; i < 2 * rope.rot; i += 64) {
        const uint32_t pair = i % (rope.rot / 2), t = i / (rope.rot / 2);
        double sn, c;
        sincospi(half_turns((double)(t0 + 4 * g + t), rope.inv_freq[pair]), &sn, &c);
        cs[block][t][pair][0] = c * (double)rope.amp;
        cs[block][t][pair][1] = sn * (double)rope.amp;
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // this wave's own reads follow
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int j = 0; j < P / 4; ++j) {
      const int n = g * (P / 4) + j;
      const uint32_t t = n * TP + lane / W;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[n][i] = 0.f;
      const bool fresh = t >= kept && t < end;
      const size_t at = (row + t) * ldk + head * D;
      if (fresh) load_n<T, 4>(k, at + d, x[n]);
      if (rope.inv_freq) {
        const double inv = rope.norm_w ? norm_factor<W, double>(x[n], D, rope.eps) : 1.0;
        if (fresh) {
          double y[4];
          rope4<T, double>(x[n], k, at, d, rope, inv, cs[block][t % 4], y);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[n][i] = (float)y[i];
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  const float sc = new_scale<INT8, P * 4>(&x[0][0], kept != 0, before);
  const float ratio = before / sc, inv = 1.0f / sc;
  if (lane == 0) *scale = sc;
  uint8_t* const base = rec + kv_k_at<D>(head) + (size_t)block * kKvBlock * D + d;
#pragma unroll
  for (int n = 0; n < P; ++n) {
    const uint32_t t = n * TP + lane / W;
    uint32_t* const at = (uint32_t*)(base + t * D);
    if (t < kept) {
      if (sc > before) *at = recode4<INT8>(*at, ratio);
    } else if (t < end && sc == sc) {
      *at = code4<INT8>(scaled<INT8>(x[n][0], sc, inv), scaled<INT8>(x[n][1], sc, inv), scaled<INT8>(x[n][2], sc, inv),
                        scaled<INT8>(x[n][3], sc, inv));
    } else {
      *at = kZero;
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
                const RopeArgs& p, hipStream_t s) {
  const dim3 grid(a.rows / kKvPage + 2 * a.seqs, 2 * a.kv_heads);
  if (head_dim == 64)
    hipLaunchKernelGGL((kv8_append_kernel<T, 64, INT8>), grid, dim3(256), 0, s, a, k, ldk, v, ldv, p);
  else if (head_dim == 128)
    hipLaunchKernelGGL((kv8_append_kernel<T, 128, INT8>), grid, dim3(256), 0, s, a, k, ldk, v, ldv, p);
  else
    hipLaunchKernelGGL((kv8_append_kernel<T, 256, INT8>), grid, dim3(256), 0, s, a, k, ldk, v, ldv, p);
}
template <typename T>
void append_format(const KvArgs& a, uint32_t head_dim, bool int8, const void* k, uint32_t ldk, const void* v,
                   uint32_t ldv, const RopeArgs& p, hipStream_t s) {
  if (int8)
    append_dim<T, true>(a, head_dim, k, ldk, v, ldv, p, s);
  else
    append_dim<T, false>(a, head_dim, k, ldk, v, ldv, p, s);
}
}  // namespace

hipError_t launch_kv8_append(const KvArgs& a, uint32_t head_dim, bool int8, const void* k, uint32_t ldk, const void* v,
                             uint32_t ldv, uint32_t dtype, const RopeArgs& p, hipStream_t s) {
  if (a.rows == 0 || a.seqs == 0) return hipSuccess;
  if (dtype == 0)
    append_format<Half>(a, head_dim, int8, k, ldk, v, ldv, p, s);
  else if (dtype == 1)
    append_format<Bf16>(a, head_dim, int8, k, ldk, v, ldv, p, s);
  else
    append_format<float>(a, head_dim, int8, k, ldk, v, ldv, p, s);
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
