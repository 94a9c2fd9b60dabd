// AdamW over many tensors at once (sm_100a): the global gradient norm with its
// clip factor, the step with 32-bit moments, the step with 8-bit moments, and
// the values of 8-bit moments.
//
// Every entry takes a host array of tensors.  Pointers, sizes, types and the
// groups' hyper-parameters travel in the kernel's parameters (up to 32 KB), so
// a call uploads nothing, keeps nothing, and can be captured in a CUDA graph;
// one launch covers all tensors of a call up to the table's capacity.  A CTA
// finds the tensor of its chunk by a binary search over the chunk prefix.
//
// The step moves 28 B an element (float32) or 22 B (16-bit parameters) and is
// bound by HBM: 268 M float32 elements take 1.08 ms (6.97 TB/s), bfloat16 ones
// 0.85 ms.  With 8-bit moments it moves 16 B or 10 B.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <type_traits>

#include "cs_common.cuh"

namespace cs {

constexpr int kChunkThreads = 128;
constexpr int kPerThread = 8;
constexpr int kBlock8 = CS_ADAMW8_BLOCK;                  // elements of a scale block: one warp's
constexpr int kChunk = kChunkThreads * kPerThread;        // elements of a CTA's chunk
static_assert(kBlock8 == 32 * kPerThread, "a warp holds one scale block");
constexpr int64_t kMaxNumel = int64_t(1) << 38;           // its scale blocks fit 32 bits
constexpr int64_t kMaxEntry = int64_t(1) << 30;           // longer tensors take several entries
constexpr int kMaxTensors = 1 << 22;                      // places that fit an entry's word

// ---------------------------------------------------------------------------
// Tables in kernel parameters

struct AdamGroup {
  float b1, omb1, b2, omb2, eps, lr, wd, ibc1, rbc2;  // ibc1 = 1/(1-b1^t), rbc2 = 1/sqrt(1-b2^t)
  uint32_t key;                                       // of the stochastic rounding
  const float* lr_dev;                                // replaces lr where given
};

struct AdamEntry {
  void* p;
  const void* g;
  void* m;
  void* v;
  int64_t numel;
  uint32_t word;  // see entry_word
  uint32_t pad;
};

struct AdamEntry8 {
  void* p;
  const void* g;
  uint8_t* m;   // codes
  uint8_t* v;
  uint8_t* ms;  // scale bytes
  uint8_t* vs;
  int64_t numel;
  uint32_t word;
  uint32_t block0;  // number of its first block in its tensor
};

// Bits 0-1 type, 2 everything aligned, 3-6 group, 7 moments aligned, 8-31 place
// in the call's array.
constexpr uint32_t kAligned = 4, kMomentsAligned = 128;
constexpr uint32_t entry_word(int dtype, bool all, bool moments, int group, int place) {
  return (uint32_t)dtype | (all ? kAligned : 0u) | ((uint32_t)group << 3) |
         (moments ? kMomentsAligned : 0u) | ((uint32_t)place << 8);
}
static_assert(CS_ADAMW_MAX_GROUPS <= 16, "four bits of group");

template <class Entry, int N>
struct Table {
  int count;
  int shift;  // a CTA takes 2^shift kChunks
  float one;  // 1 (see sum2)
  uint32_t place_key;  // of the place that the call's first tensor has
  const float* grad_scale;
  const float* coef;  // {ibc1, rbc2, key bits, -} of each group, or of each tensor; or NULL
  int each;           // of each tensor
  AdamGroup groups[CS_ADAMW_MAX_GROUPS];
  int first[N];  // first chunk of each entry
  Entry e[N];
};

// The entry of a chunk.  (Eight ways at a time, with seven independent reads a
// step, measured no faster.)
__device__ __forceinline__ int find_entry(const int* first, int count, int chunk) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= chunk)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// ---------------------------------------------------------------------------
// Eight elements of a thread as float32: contiguous ones with wide accesses
// (the pointer aligned to eight elements), or every 32nd of the warp's 256.

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

template <class T>
struct alignas(16) Pack8 {
  T x[8];
};

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const Pack8<T> q = *reinterpret_cast<const Pack8<T>*>(p);
#pragma unroll
  for (int u = 0; u < 8; ++u) x[u] = to_f32(q.x[u]);
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  Pack8<T> q;
#pragma unroll
  for (int u = 0; u < 8; ++u) q.x[u] = from_f32<T>(x[u]);
  *reinterpret_cast<Pack8<T>*>(p) = q;
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float2 (&x)[4]) {
  Pack8<T> q;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    q.x[2 * u] = from_f32<T>(x[u].x);
    q.x[2 * u + 1] = from_f32<T>(x[u].y);
  }
  *reinterpret_cast<Pack8<T>*>(p) = q;
}

// One 32-byte store of a lane (aligned to 32 bytes): whole sectors at once.
__device__ __forceinline__ void store_wide(float* p, const float2 (&x)[4]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0].x),
               "f"(x[0].y), "f"(x[1].x), "f"(x[1].y), "f"(x[2].x), "f"(x[2].y), "f"(x[3].x),
               "f"(x[3].y)
               : "memory");
}

// Two elements of a word or two, as float32.
template <class T>
__device__ __forceinline__ float2 unpack2(const uint32_t* w);
template <>
__device__ __forceinline__ float2 unpack2<float>(const uint32_t* w) {
  return make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(const uint32_t* w) {
  return make_float2(__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(const uint32_t* w) {
  return __half22float2(*reinterpret_cast<const __half2*>(w));
}

struct StepCoef {
  float b1, omb1, b2, omb2, eps, step_size, decay, rbc2, scale;
  uint32_t key;
};

template <class Entry, int N>
__device__ __forceinline__ StepCoef load_coef(const Table<Entry, N>& t, uint32_t word) {
  const uint32_t group = (word >> 3) & 15;
  const AdamGroup& g = t.groups[group];
  StepCoef c;
  c.b1 = g.b1;
  c.omb1 = g.omb1;
  c.b2 = g.b2;
  c.omb2 = g.omb2;
  c.eps = g.eps;
  const float lr = g.lr_dev ? __ldg(g.lr_dev) : g.lr;
  float ibc1 = g.ibc1;
  c.rbc2 = g.rbc2;
  c.key = g.key;
  if (t.coef) {
    const float* coef = t.coef + 4 * (t.each ? word >> 8 : group);
    ibc1 = __ldg(coef);
    c.rbc2 = __ldg(coef + 1);
    c.key = __float_as_uint(__ldg(coef + 2));
  }
  c.step_size = lr * ibc1;
  c.decay = __fmaf_rn(-lr, g.wd, 1.0f);
  c.scale = t.grad_scale ? __ldg(t.grad_scale) : 1.0f;
  return c;
}

// One element, in float32 with one rounding an operation in the order written
// (step_lane8 does the same to m and v, whose bytes are defined by it).
__device__ __forceinline__ void adamw_element(const StepCoef& c, float& p, float g, float& m,
                                              float& v) {
  g = g * c.scale;
  m = m * c.b1 + g * c.omb1;
  v = v * c.b2 + (g * g) * c.omb2;
  p = p * c.decay - c.step_size * (m / (sqrtf(v) * c.rbc2 + c.eps));
}

// ---------------------------------------------------------------------------
// 32-bit moments

template <class T>
__device__ __forceinline__ void step_chunk(const AdamEntry& e, const StepCoef& c, int64_t at) {
  T* p = static_cast<T*>(e.p) + at;
  const T* g = static_cast<const T*>(e.g) + at;
  float* m = static_cast<float*>(e.m) + at;
  float* v = static_cast<float*>(e.v) + at;
  const int lane = threadIdx.x & 31, base = (threadIdx.x >> 5) * kBlock8;
  const int64_t left = e.numel - at - base;
  if (left <= 0) return;
  float P[8], G[8], M[8], V[8];
  if ((e.word & kAligned) && left >= kBlock8) {
    const int i = base + lane * 8;
    load8(p + i, P);
    load8(g + i, G);
    load8(m + i, M);
    load8(v + i, V);
#pragma unroll
    for (int u = 0; u < 8; ++u) adamw_element(c, P[u], G[u], M[u], V[u]);
    store8(p + i, P);
    store8(m + i, M);
    store8(v + i, V);
  } else {
    // by single elements 64 M float32 elements take as long as aligned ones (275
    // us), bfloat16 ones 256 us (216)
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = base + lane + 32 * u;
      if (lane + 32 * u < left) {
        P[u] = to_f32(p[i]);
        G[u] = to_f32(g[i]);
        M[u] = m[i];
        V[u] = v[i];
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = base + lane + 32 * u;
      if (lane + 32 * u < left) {
        adamw_element(c, P[u], G[u], M[u], V[u]);
        p[i] = from_f32<T>(P[u]);
        m[i] = M[u];
        v[i] = V[u];
      }
    }
  }
}

template <int N>
__global__ void __launch_bounds__(kChunkThreads)
    adamw_kernel(const __grid_constant__ Table<AdamEntry, N> t) {
  const int k = find_entry(t.first, t.count, blockIdx.x);
  const AdamEntry& e = t.e[k];
  const StepCoef c = load_coef(t, e.word);
  const int64_t at = (int64_t)((int)blockIdx.x - t.first[k]) * kChunk;
  switch (e.word & 3) {
    case CS_F32: step_chunk<float>(e, c, at); break;
    case CS_BF16: step_chunk<__nv_bfloat16>(e, c, at); break;
    default: step_chunk<__half>(e, c, at); break;
  }
}

// ---------------------------------------------------------------------------
// 8-bit moments
//
// A block of 256 elements (one warp, eight a lane) shares one scale byte E that
// stands for 2^(E-127): the smallest power of two, E >= 40, with
// max|x| <= 1.875 * 2^(E-127).  x / 2^(E-127) is multiplied by 2^-112 (m) or
// 2^-96 (v), which puts the largest value at the exponent field 15 (m) or 31
// (v) of a float32, and the code is that float's bits 20..26 with the sign (m:
// sign, 4 exponent, 3 fraction bits) or 20..27 (v: 5 and 3), the float's own
// gradual underflow included.  Decoding is the same shift and two
// multiplications, by a power of two and by the average's beta over another.  The 20 low bits
// go by stochastic rounding: a moment that moves by 1 - beta2 = 0.1% a step
// would never leave its code (6 to 12% wide) by rounding to nearest.  A v above
// zero keeps at least its smallest code, so that m / sqrt(v) stays bounded.
// E = 255 marks a block whose largest magnitude is NaN or needs E >= 254; all
// of its elements then stand for NaN.

constexpr int kMinScale = 40;
constexpr float kLeastEps = 8.673617379884035e-19f;  // 2^-60, the root of the smallest v

constexpr float kLargest = 3.4028234663852886e38f;           // of the finite float32 values

constexpr float kTwoM112 = 1.925929944387236e-34f, kTwo112 = 5.192296858534828e33f;
constexpr float kTwoM96 = 1.262177448353619e-29f, kTwo96 = 7.922816251426434e28f;

__host__ __device__ constexpr uint32_t mix32(uint32_t h) {
  h = (h ^ (h >> 16)) * 0x6A09E667u;
  h = (h ^ (h >> 15)) * 0xBB67AE85u;
  return h ^ (h >> 16);
}
// Key of a step, of a block of a tensor, and the 32 random bits of an element:
// multiply-xorshift mixing with fractional digits of square roots and the
// golden ratio as multipliers (an element's bits in step_lane8).
__host__ __device__ constexpr uint32_t step_key(uint32_t seed, uint32_t step) {
  return mix32(seed + step * 0x9E3779B1u);
}
__host__ __device__ constexpr uint32_t place_key(uint32_t place) { return place * 0x3C6EF373u; }
__device__ __forceinline__ uint32_t block_key(uint32_t key, uint32_t place, uint32_t block) {
  return mix32(key + place_key(place) + block * 0xA54FF53Bu);
}
__device__ __forceinline__ float scale_unit(uint32_t e) {
  const float x = __uint_as_float(e << 23);  // infinity for 255
  return __fmaf_rn(x, 0.0f, x);              // which this turns into NaN
}
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest_bits) {
  const uint32_t e = max((largest_bits + 0xFFFFFu) >> 23, (uint32_t)kMinScale);  // NaN: 256
  return e >= 254 ? 255u : e;
}
__device__ __forceinline__ float scale_inverse(uint32_t e) {  // codes of a marked block: any
  return __uint_as_float((254u - e) << 23);
}
__device__ __forceinline__ float decode_m(uint32_t code) {  // times 2^(E-127)
  return __uint_as_float(((code & 127u) << 20) | ((code & 128u) << 24)) * kTwo112;
}
__device__ __forceinline__ float decode_v(uint32_t code) {
  return __uint_as_float(code << 20) * kTwo96;
}

// x + y of pairs, one rounding each.  A packed sum of a packed product is fused
// by the assembler whatever rounding both are written with, which would round
// once instead of twice; as x * one + y with a `one` that only the host knows it
// is the same sum and cannot be.
__device__ __forceinline__ float2 sum2(float2 x, float2 one, float2 y) {
  return __ffma2_rn(x, one, y);
}
__device__ __forceinline__ float2 pair(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 bits2(uint32_t a, uint32_t b) {
  return make_float2(__uint_as_float(a), __uint_as_float(b));
}
// max(|a|, |b|, |c|), NaN if any is
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float sqrt_approx(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Codes u and u+1 of a word of four, as the float2 whose bits they are.
template <int U>
__device__ __forceinline__ float2 bits_m(uint32_t w) {
  // the code in the top byte: its sign is the float's, its magnitude 4 down
  const int a = (int)(w << (24 - 8 * U)), b = (int)(w << (16 - 8 * U));
  return bits2((uint32_t)(a >> 4) & 0x87F00000u, (uint32_t)(b >> 4) & 0x87F00000u);
}
template <int U>
__device__ __forceinline__ float2 bits_v(uint32_t w) {
  return bits2((w << (20 - 8 * U)) & 0x0FF00000u,
               (U == 0 ? w << 12 : w >> 4) & 0x0FF00000u);
}
__device__ __forceinline__ uint32_t top_bytes(const uint32_t (&t)[4]) {
  return __byte_perm(__byte_perm(t[0], t[1], 0x0073), __byte_perm(t[2], t[3], 0x0073), 0x5410);
}

struct StepCoef8 {
  float b1, b2, omb1, omb2, scale, one, decay, root, off;
  uint32_t key;
};
// off / root hold eps (at least the root of the smallest v that the format
// holds) and the correction of v, both over the negative step size.  A step size
// near or at zero makes off infinite, which moves nothing; root stays finite, so
// that neither its product with v = 0 nor an infinite v with it is NaN.
template <int N>
__device__ __forceinline__ StepCoef8 load_coef8(const Table<AdamEntry8, N>& t, uint32_t word) {
  const StepCoef s = load_coef(t, word);
  StepCoef8 c;
  c.b1 = s.b1;
  c.b2 = s.b2;
  c.omb1 = s.omb1;
  c.omb2 = s.omb2;
  c.scale = s.scale;
  c.one = t.one;
  c.decay = s.decay;
  c.root = fminf(fmaxf(__fdividef(-s.rbc2, s.step_size), -kLargest), kLargest);
  c.off = __fdividef(-fmaxf(s.eps, kLeastEps), s.step_size);
  c.key = s.key + t.place_key;
  return c;
}

// Gives positive v whose code is 0 the code 1.  Rare, and not inlined: inline it
// would be executed under predicates every time.
__device__ __noinline__ uint32_t raised_zeros(uint32_t w, float a, float b, float c, float d) {
  if (!(w & 0xFFu) && a > 0.0f) w |= 1u;
  if (!(w & 0xFF00u) && b > 0.0f) w |= 1u << 8;
  if (!(w & 0xFF0000u) && c > 0.0f) w |= 1u << 16;
  if (!(w & 0xFF000000u) && d > 0.0f) w |= 1u << 24;
  return w;
}
// A lane's eight elements of one block: P and the codes in mw, vw in, the same
// out, and the block's new scale bytes; mk, vk are the betas times the old
// scales' units.  Arithmetic on m and v is in float32 pairs (two independent
// IEEE operations an instruction) in the written order; decoding's power of two
// is folded into beta, which changes no bit.  The parameter's update,
// -step m / (sqrt(v) rbc2 + eps) = m / (sqrt(v) c.root + c.off), uses the
// hardware's square root and reciprocal, each within 2^-22: the bytes do not
// depend on it.  `first` is the element of the lane's first value in the block,
// kStride the distance of the next.
//
// With 16-bit parameters the instructions bound it, not the memory: some 47 an
// element, 20 of them integer.  268 M bfloat16 elements take 444 us (6.05 TB/s,
// 93% of the copy rate; 618 us before the codes were built word by word, the
// per-block values prepared a block a lane and the next block prefetched),
// float32 643 us (6.68 TB/s, the copy rate).  Seven CTAs of 128 threads an SM
// leave 72 registers a thread, which just hold it; three of 256 took 459 us.
template <int kStride>
__device__ __forceinline__ void step_lane8(const StepCoef8& c, float2 (&P)[4],
                                           const float2 (&G)[4], uint32_t (&mw)[2],
                                           uint32_t (&vw)[2], float mk, float vk,
                                           uint32_t key, uint32_t first, uint32_t& me,
                                           uint32_t& ve) {
  float2 M[4], V[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    M[u] = (u & 1) ? bits_m<2>(mw[u >> 1]) : bits_m<0>(mw[u >> 1]);
    V[u] = (u & 1) ? bits_v<2>(vw[u >> 1]) : bits_v<0>(vw[u >> 1]);
  }
  float mmax = 0.0f, vmax = 0.0f;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const float2 g = __fmul2_rn(G[u], pair(c.scale));
    M[u] = sum2(__fmul2_rn(__fmul2_rn(M[u], pair(kTwo112)), pair(mk)), pair(c.one), __fmul2_rn(g, pair(c.omb1)));
    V[u] = sum2(__fmul2_rn(__fmul2_rn(V[u], pair(kTwo96)), pair(vk)), pair(c.one),
                __fmul2_rn(__fmul2_rn(g, g), pair(c.omb2)));
    mmax = max3_abs(mmax, M[u].x, M[u].y);
    vmax = max3_abs(vmax, V[u].x, V[u].y);
    const float2 root = make_float2(sqrt_approx(V[u].x), sqrt_approx(V[u].y));
    const float2 d = __ffma2_rn(root, pair(c.root), pair(c.off));
    P[u] = __ffma2_rn(M[u], make_float2(rcp_approx(d.x), rcp_approx(d.y)),
                      __fmul2_rn(P[u], pair(c.decay)));
  }
  me = scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(mmax)));
  ve = scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(vmax)));
  const float2 mi = pair(scale_inverse(me)), vi = pair(scale_inverse(ve));
  const uint32_t start = key + first * 0x9E3779B1u;
  uint32_t zero = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t t[4], w[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int u = 2 * h + j;
      const float2 ym = __fmul2_rn(__fmul2_rn(M[u], mi), pair(kTwoM112));
      const float2 yv = __fmul2_rn(__fmul2_rn(V[u], vi), pair(kTwoM96));
      uint32_t r0 = start + (uint32_t)(2 * u * kStride) * 0x9E3779B1u;
      uint32_t r1 = start + (uint32_t)((2 * u + 1) * kStride) * 0x9E3779B1u;
      r0 = (r0 ^ (r0 >> 16)) * 0x6A09E667u;
      r1 = (r1 ^ (r1 >> 16)) * 0x6A09E667u;
      r0 ^= r0 >> 15;
      r1 ^= r1 >> 15;
      // (bits + (random << 4)) << 4: the code comes to lie in the top byte
      const uint32_t mx = __float_as_uint(ym.x), my = __float_as_uint(ym.y);
      t[2 * j] = (mx * 16u + __byte_perm(r0, 0, 0x4104)) | (mx & 0x80000000u);
      t[2 * j + 1] = (my * 16u + __byte_perm(r1, 0, 0x4104)) | (my & 0x80000000u);
      w[2 * j] = __float_as_uint(yv.x) * 16u + __byte_perm(r0, 0, 0x4324);
      w[2 * j + 1] = __float_as_uint(yv.y) * 16u + __byte_perm(r1, 0, 0x4324);
    }
    mw[h] = top_bytes(t);
    vw[h] = top_bytes(w);
    zero |= (vw[h] - 0x01010101u) & ~vw[h] & 0x80808080u;
  }
  if (zero) {  // some code of v is 0: only for v = 0
    vw[0] = raised_zeros(vw[0], V[0].x, V[0].y, V[1].x, V[1].y);
    vw[1] = raised_zeros(vw[1], V[2].x, V[2].y, V[3].x, V[3].y);
  }
}

// One lane's share of an aligned, full block as it lies in memory, and where.
template <class T>
struct Raw8 {
  static constexpr int kWords = 2 * sizeof(T);
  uint32_t p[kWords], g[kWords];
  uint2 m, v;
};
template <int kWords>
__device__ __forceinline__ void load_words(const char* at, uint32_t (&w)[kWords]) {
#pragma unroll
  for (int i = 0; i < kWords; i += 4) {
    const uint4 q = *reinterpret_cast<const uint4*>(at + 4 * i);
    w[i] = q.x;
    w[i + 1] = q.y;
    w[i + 2] = q.z;
    w[i + 3] = q.w;
  }
}
template <class T>
struct Lane8 {  // offsets are 32 bits: an entry holds at most 2^30 elements
  char *p, *m, *v;
  const char* g;
  uint32_t lane;
  __device__ __forceinline__ Lane8(const AdamEntry8& e, uint32_t lane)
      : p(static_cast<char*>(e.p)),
        m(reinterpret_cast<char*>(e.m)),
        v(reinterpret_cast<char*>(e.v)),
        g(static_cast<const char*>(e.g)),
        lane(lane) {}
  __device__ __forceinline__ void load(uint32_t block, Raw8<T>& r) const {
    const uint32_t at = block * kBlock8 + lane * 8;
    load_words(p + at * (uint32_t)sizeof(T), r.p);
    load_words(g + at * (uint32_t)sizeof(T), r.g);
    r.m = *reinterpret_cast<const uint2*>(m + at);
    r.v = *reinterpret_cast<const uint2*>(v + at);
  }
  // The step of a loaded block; new scale bytes in me, ve.
  __device__ __forceinline__ void step(const StepCoef8& c, uint32_t block, const Raw8<T>& r,
                                       float mk, float vk, uint32_t key, uint32_t& me,
                                       uint32_t& ve) const {
    float2 P[4], G[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      P[u] = unpack2<T>(r.p + u * (sizeof(T) / 2));
      G[u] = unpack2<T>(r.g + u * (sizeof(T) / 2));
    }
    uint32_t mw[2] = {r.m.x, r.m.y}, vw[2] = {r.v.x, r.v.y};
    step_lane8<1>(c, P, G, mw, vw, mk, vk, key, lane * 8, me, ve);
    const uint32_t at = block * kBlock8 + lane * 8;
    store8(reinterpret_cast<T*>(p + at * (uint32_t)sizeof(T)), P);
    *reinterpret_cast<uint2*>(m + at) = make_uint2(mw[0], mw[1]);
    *reinterpret_cast<uint2*>(v + at) = make_uint2(vw[0], vw[1]);
  }
};

// A block that is cut short or not aligned: every 32nd element, one at a time.
template <class T>
__device__ __forceinline__ void step_part8(const AdamEntry8& e, const StepCoef8& c, uint32_t block,
                                           int lane) {
  const int64_t at = (int64_t)block * kBlock8;
  const int left = (int)min((int64_t)kBlock8, e.numel - at);
  T* p = static_cast<T*>(e.p) + at;
  const T* g = static_cast<const T*>(e.g) + at;
  uint8_t* mc = e.m + at;
  uint8_t* vc = e.v + at;
  float2 P[4], G[4];
  uint32_t mw[2] = {0, 0}, vw[2] = {0, 0}, me, ve;
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int i = lane + 32 * u;
    const bool in = i < left;
    (u & 1 ? P[u >> 1].y : P[u >> 1].x) = in ? to_f32(p[i]) : 0.0f;
    (u & 1 ? G[u >> 1].y : G[u >> 1].x) = in ? to_f32(g[i]) : 0.0f;
    mw[u >> 2] |= (in ? (uint32_t)mc[i] : 0u) << (8 * (u & 3));
    vw[u >> 2] |= (in ? (uint32_t)vc[i] : 0u) << (8 * (u & 3));
  }
  const uint32_t em = e.ms[block], ev = e.vs[block];
  step_lane8<32>(c, P, G, mw, vw, c.b1 * scale_unit(em), c.b2 * scale_unit(ev),
                 block_key(c.key, e.word >> 8, e.block0 + block), lane, me, ve);
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int i = lane + 32 * u;
    if (i < left) {
      p[i] = from_f32<T>(u & 1 ? P[u >> 1].y : P[u >> 1].x);
      mc[i] = (uint8_t)(mw[u >> 2] >> (8 * (u & 3)));
      vc[i] = (uint8_t)(vw[u >> 2] >> (8 * (u & 3)));
    }
  }
  if (lane == 0) {
    e.ms[block] = (uint8_t)me;
    e.vs[block] = (uint8_t)ve;
  }
}

// A warp's 256 elements of an unaligned tensor, moved between memory (every 32nd
// element a lane, so that an access is one stretch) and eight consecutive
// elements a lane by way of the warp's kilobyte of shared memory.
constexpr int kExchange = 64;  // uint4 a warp
template <class T>
__device__ __forceinline__ void load8_loose(const T* p, uint4* buf, int lane, float2 (&x)[4]) {
  T* b = reinterpret_cast<T*>(buf);
  T q[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) q[u] = p[lane + 32 * u];
  __syncwarp();  // the last use of the buffer
#pragma unroll
  for (int u = 0; u < 8; ++u) b[lane + 32 * u] = q[u];
  __syncwarp();
  uint32_t w[2 * sizeof(T)];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    const uint4 r = buf[lane * (sizeof(T) / 2) + i];
    w[4 * i] = r.x;
    w[4 * i + 1] = r.y;
    w[4 * i + 2] = r.z;
    w[4 * i + 3] = r.w;
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) x[u] = unpack2<T>(w + u * (sizeof(T) / 2));
}
template <class T>
__device__ __forceinline__ void store8_loose(T* p, uint4* buf, int lane, const float2 (&x)[4]) {
  T* b = reinterpret_cast<T*>(buf);
  __syncwarp();
  store8(b + lane * 8, x);
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 8; ++u) p[lane + 32 * u] = b[lane + 32 * u];
}

// A full block whose codes are aligned and whose parameters or gradients are not:
// 64 M float32 elements take 195 us, 300 by single elements throughout, 165
// aligned; bfloat16 ones 245, 276 and 119 (their 16-bit accesses are what is
// left).
template <class T>
__device__ __forceinline__ void step_loose8(const AdamEntry8& e, const StepCoef8& c,
                                            uint32_t block, int lane, uint4* buf) {
  const int64_t at = (int64_t)block * kBlock8;
  T* p = static_cast<T*>(e.p) + at;
  uint2* mc = reinterpret_cast<uint2*>(e.m + at) + lane;
  uint2* vc = reinterpret_cast<uint2*>(e.v + at) + lane;
  const uint2 a = *mc, b = *vc;
  const uint32_t em = e.ms[block], ev = e.vs[block];
  float2 P[4], G[4];
  load8_loose(p, buf, lane, P);
  load8_loose(static_cast<const T*>(e.g) + at, buf, lane, G);
  uint32_t mw[2] = {a.x, a.y}, vw[2] = {b.x, b.y}, me, ve;
  step_lane8<1>(c, P, G, mw, vw, c.b1 * scale_unit(em), c.b2 * scale_unit(ev),
                block_key(c.key, e.word >> 8, e.block0 + block), lane * 8, me, ve);
  store8_loose(p, buf, lane, P);
  *mc = make_uint2(mw[0], mw[1]);
  *vc = make_uint2(vw[0], vw[1]);
  if (lane == 0) {
    e.ms[block] = (uint8_t)me;
    e.vs[block] = (uint8_t)ve;
  }
}

// A warp's blocks: one of each kChunk that its CTA takes, which lie as far
// apart as the tensor has CTAs, so that all CTAs together walk through memory
// (neighbouring chunks for each CTA were 2.4 times slower: everything in flight
// was a slice of 8 KB in every 64).  What a block has one of (scales, key) is
// prepared and stored for all of the warp's blocks at once, a block a lane (32
// blocks a warp at most; with eight at most 268 M bfloat16 elements took 5%
// longer, with two 27%).
// With 16-bit parameters the next block's loads are issued before the present
// one's arithmetic (they need 12 registers; float32's 20 spill at seven CTAs an
// SM, 698 us for 268 M elements instead of 643, and gain nothing at five).
template <class T>
__device__ __forceinline__ void step_warp8(const AdamEntry8& e, const StepCoef8& c, uint32_t chunk,
                                           int shift, uint4* buf) {
  constexpr uint32_t kWarps = kChunkThreads / 32;
  const int lane = threadIdx.x & 31;
  const uint32_t chunks = (uint32_t)((e.numel + kChunk - 1) / kChunk);
  const uint32_t stride = (chunks + (1u << shift) - 1) >> shift << 2;
  static_assert(kWarps == 4, "2 bits");
  const uint32_t first = chunk * kWarps + (threadIdx.x >> 5);
  const uint32_t end = (uint32_t)((e.numel + kBlock8 - 1) / kBlock8);
  const uint32_t whole = (uint32_t)(e.numel / kBlock8);
  const uint32_t full = (e.word & kAligned) ? whole : 0;
  int n = 0;  // full blocks of this warp
  if (first < full) n = shift ? (int)min(1u << shift, (full - first + stride - 1) / stride) : 1;
  if (n > 0) {
    const Lane8<T> at(e, lane);
    Raw8<T> a, b;
    at.load(first, a);
    const uint32_t mine = first + lane * stride;
    uint32_t em = 1, ev = 1;
    if (lane < n) {
      em = e.ms[mine];
      ev = e.vs[mine];
    }
    const float mk = c.b1 * scale_unit(em), vk = c.b2 * scale_unit(ev);
    const uint32_t key = block_key(c.key, e.word >> 8, e.block0 + mine);
    const auto step = [&](int i, const Raw8<T>& r) {
      uint32_t me, ve;
      at.step(c, first + i * stride, r, __shfl_sync(0xffffffffu, mk, i),
              __shfl_sync(0xffffffffu, vk, i),
              __shfl_sync(0xffffffffu, key, i), me, ve);
      if (lane == i) {
        em = me;
        ev = ve;
      }
    };
    if (sizeof(T) == 2) {
      for (int i = 0;;) {
        if (i + 1 < n) at.load(first + (i + 1) * stride, b);
        step(i, a);
        if (++i == n) break;
        if (i + 1 < n) at.load(first + (i + 1) * stride, a);
        step(i, b);
        if (++i == n) break;
      }
    } else {
      for (int i = 0;;) {
        step(i, a);
        if (++i == n) break;
        at.load(first + i * stride, a);
      }
    }
    if (lane < n) {
      e.ms[mine] = (uint8_t)em;
      e.vs[mine] = (uint8_t)ev;
    }
  }
  for (uint32_t block = first + n * stride, i = n; i >> shift == 0 && block < end;
       ++i, block += stride) {
    if ((e.word & kMomentsAligned) && block < whole)
      step_loose8<T>(e, c, block, lane, buf);
    else
      step_part8<T>(e, c, block, lane);
  }
}

template <int N>
__global__ void __launch_bounds__(kChunkThreads, 7)
    adamw8_kernel(const __grid_constant__ Table<AdamEntry8, N> t) {
  __shared__ uint4 exchange[kChunkThreads / 32][kExchange];
  uint4* buf = exchange[threadIdx.x >> 5];
  const int k = find_entry(t.first, t.count, blockIdx.x);
  const AdamEntry8& e = t.e[k];
  const StepCoef8 c = load_coef8(t, e.word);
  const int chunk = (int)blockIdx.x - t.first[k];
  switch (e.word & 3) {
    case CS_F32: step_warp8<float>(e, c, chunk, t.shift, buf); break;
    case CS_BF16: step_warp8<__nv_bfloat16>(e, c, chunk, t.shift, buf); break;
    default: step_warp8<__half>(e, c, chunk, t.shift, buf); break;
  }
}

// Values of 8-bit moments: entries hold the float outputs in p (m) and g (v).
template <int N>
__global__ void __launch_bounds__(kChunkThreads)
    adamw8_moments_kernel(const __grid_constant__ Table<AdamEntry8, N> t) {
  const int k = find_entry(t.first, t.count, blockIdx.x);
  const AdamEntry8& e = t.e[k];
  const int lane = threadIdx.x & 31;
  const int64_t block =
      (int64_t)((int)blockIdx.x - t.first[k]) * (kChunk / kBlock8) + (threadIdx.x >> 5);
  const int64_t left = e.numel - block * kBlock8;
  if (left <= 0) return;
  float* om = static_cast<float*>(e.p) + block * kBlock8;
  float* ov = static_cast<float*>(const_cast<void*>(e.g)) + block * kBlock8;
  const uint8_t* mc = e.m + block * kBlock8;
  const uint8_t* vc = e.v + block * kBlock8;
  const float mb = scale_unit(e.ms[block]), vb = scale_unit(e.vs[block]);
  if ((e.word & kAligned) && left >= kBlock8) {
    const uint2 a = *reinterpret_cast<const uint2*>(mc + lane * 8);
    const uint2 b = *reinterpret_cast<const uint2*>(vc + lane * 8);
    const float2 mk = pair(mb), vk = pair(vb), up112 = pair(kTwo112), up96 = pair(kTwo96);
    float2 M[4] = {bits_m<0>(a.x), bits_m<2>(a.x), bits_m<0>(a.y), bits_m<2>(a.y)};
    float2 V[4] = {bits_v<0>(b.x), bits_v<2>(b.x), bits_v<0>(b.y), bits_v<2>(b.y)};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      M[u] = __fmul2_rn(__fmul2_rn(M[u], up112), mk);
      V[u] = __fmul2_rn(__fmul2_rn(V[u], up96), vk);
    }
    store_wide(om + lane * 8, M);
    store_wide(ov + lane * 8, V);
  } else {
    for (int i = lane; i < kBlock8 && i < left; i += 32) {
      om[i] = decode_m(mc[i]) * mb;
      ov[i] = decode_v(vc[i]) * vb;
    }
  }
}

// ---------------------------------------------------------------------------
// Bias corrections and rounding keys from device step counters: thread i
// advances counter i and writes {1/(1-b1^t), 1/sqrt(1-b2^t), key} of its group.
template <int N>
struct CountTable {
  int count;
  uint32_t seed;
  float* coef;
  double b1[CS_ADAMW_MAX_GROUPS], b2[CS_ADAMW_MAX_GROUPS];
  int64_t* step[N];
  uint8_t group[N];
};
constexpr int kCountThreads = 64;

template <int N>
__global__ void __launch_bounds__(kCountThreads)
    adamw_advance_kernel(const __grid_constant__ CountTable<N> a) {
  const int i = blockIdx.x * kCountThreads + threadIdx.x;
  if (i >= a.count) return;
  const int g = a.group[i];
  const int64_t t = *a.step[i] + 1;
  *a.step[i] = t;
  a.coef[4 * i] = (float)(1.0 / (1.0 - pow(a.b1[g], (double)t)));
  a.coef[4 * i + 1] = (float)(1.0 / sqrt(1.0 - pow(a.b2[g], (double)t)));
  a.coef[4 * i + 2] = __uint_as_float(step_key(a.seed, (uint32_t)t));
}

// ---------------------------------------------------------------------------
// Global gradient norm: per-CTA sums in double in a fixed order, then one CTA.
// Squares are formed in double, so neither 1e30 nor 1e-30 is lost.  403 M
// bfloat16 elements take 120 us (6.7 TB/s, the copy rate; 150 us with the
// conversion instruction and chunks of 16 KB), float32 228 us (7.0 TB/s).  Run
// for a tenth of a second on end it meets the power limit.

struct NormEntry {
  const void* g;
  int64_t numel;
};

template <int N>
struct NormTable {
  int count, chunks;
  double* partials;
  int first[N];
  uint8_t word[N];
  NormEntry e[N];
};

constexpr int kNormThreads = 256;
// A chunk is 32 KB: eight 16-byte loads a thread in flight.
constexpr int norm_chunk_of(int dtype) { return kNormThreads * (dtype == CS_F32 ? 32 : 64); }
constexpr int kNormBlocks = 148 * 5;  // as many as are resident

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ double block_sum_d(double v) {  // valid in thread 0
  __shared__ double sh[32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  v = warp_sum_d(v);
  if (lane == 0) sh[wid] = v;
  __syncthreads();
  double r = 0.0;
  if (wid == 0) {
    r = lane < (int)(blockDim.x >> 5) ? sh[lane] : 0.0;
    r = warp_sum_d(r);
  }
  return r;
}

// Sum of squares in double.  float32 is converted by the instruction for it.
// That one runs at a quarter of the integer rate and bound the 16-bit types, so
// theirs goes by integer operations, two elements a word: the exponent and
// fraction bits moved to their places in a double's upper word are |x| times a
// power of two (2^-896 for bfloat16, 2^-1008 for float16), subnormal numbers and
// zero included, and one exact product makes that |x|.  Infinities and NaN come
// out finite there, so the largest magnitude is kept and looked at in the end.
template <class T>
struct SquareSum;

template <>
struct SquareSum<float> {
  using Bits = float;
  double acc = 0.0;
  __device__ __forceinline__ void add(float x) { acc = fma((double)x, (double)x, acc); }
  __device__ __forceinline__ void add_words(const uint32_t (&w)[8]) {
#pragma unroll
    for (int u = 0; u < 8; ++u) add(__uint_as_float(w[u]));
  }
  __device__ __forceinline__ double sum() const { return acc; }
};

template <class Pair, int kLeft, int kRight, uint32_t kMask>
struct SquareSum16 {
  using Bits = uint16_t;
  static constexpr double kFactor = kLeft == 13 ? 0x1p896 : 0x1p1008;
  double lo = 0.0, hi = 0.0;
  Pair most = {};
  __device__ __forceinline__ void add_word(uint32_t w) {
    most = __hmax2_nan(most, __habs2(*reinterpret_cast<Pair*>(&w)));
    const double x = __hiloint2double((int)((w << kLeft) & kMask), 0) * kFactor;
    const double y = __hiloint2double((int)((w >> kRight) & kMask), 0) * kFactor;
    lo = fma(x, x, lo);
    hi = fma(y, y, hi);
  }
  __device__ __forceinline__ void add(uint16_t x) { add_word(x); }
  __device__ __forceinline__ void add_words(const uint32_t (&w)[4]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) add_word(w[u]);
  }
  __device__ __forceinline__ double sum() const {
    const float m = to_f32(__hmax_nan(most.x, most.y));
    return m < __int_as_float(0x7f800000) ? lo + hi : (double)m;
  }
};
template <>
struct SquareSum<__nv_bfloat16> : SquareSum16<__nv_bfloat162, 13, 3, 0x0FFFE000u> {};
template <>
struct SquareSum<__half> : SquareSum16<__half2, 10, 6, 0x01FFFC00u> {};

// A short or unaligned chunk: the elements before the first 16-byte border and
// after the last one by themselves, the rest with half as many loads at once.
template <class T>
__device__ __noinline__ double norm_part(const T* g, int n) {
  constexpr int kLoads = 16 / sizeof(T), kWords = 2 * sizeof(T);
  const int thread = threadIdx.x % kNormThreads;
  SquareSum<T> s;
  using Bits = typename SquareSum<T>::Bits;
  const int head = min(n, (int)((-reinterpret_cast<uintptr_t>(g) & 15u) / sizeof(T)));
  const Bits* bits = reinterpret_cast<const Bits*>(g);
  if (thread < head) s.add(bits[thread]);
  g += head;
  bits += head;
  n -= head;
  const int last = (n & ~7) + thread;
  if (last < n) s.add(bits[last]);
#pragma unroll 1
  for (int from = thread * 8; from + 8 <= n; from += kLoads / 2 * kNormThreads * 8) {
    uint32_t w[kLoads / 2][kWords];
#pragma unroll
    for (int u = 0; u < kLoads / 2; ++u) {
      const int i = from + u * kNormThreads * 8;
#pragma unroll
      for (int j = 0; j < kWords; ++j) w[u][j] = 0;
      if (i + 8 <= n) load_words(reinterpret_cast<const char*>(g + i), w[u]);
    }
#pragma unroll
    for (int u = 0; u < kLoads / 2; ++u) s.add_words(w[u]);
  }
  return s.sum();
}

// A square p as float32 times 2^-896: its bits three places down in a double
// (kLow: with more than 20 fraction bits, which the upper word does not hold).
template <bool kLow>
__device__ __forceinline__ double square_bits(float p) {
  const uint32_t b = __float_as_uint(p);
  return __hiloint2double((int)(b >> 3), kLow ? (int)(b << 29) : 0);
}

template <class T>
__device__ __forceinline__ double norm_chunk(const void* data, int chunk, int64_t numel,
                                             bool vec) {
  const int thread = threadIdx.x % kNormThreads;
  constexpr int kLoads = 16 / sizeof(T), kElems = kNormThreads * kLoads * 8;
  static_assert(kElems == norm_chunk_of(sizeof(T) == 4 ? CS_F32 : CS_BF16), "one chunk size");
  const int64_t at = (int64_t)chunk * kElems;
  const T* g = static_cast<const T*>(data) + at;
  const int64_t left = numel - at;
  const int n = left < kElems ? (int)left : kElems;
  if (!vec || n < kElems) return norm_part(g, n);
  uint32_t w[kLoads][2 * sizeof(T)];
#pragma unroll
  for (int u = 0; u < kLoads; ++u)
    load_words(reinterpret_cast<const char*>(g + (u * kNormThreads + thread) * 8), w[u]);
  if (sizeof(T) == 4) {
    SquareSum<T> s;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) s.add_words(w[u]);
    return s.sum();
  }
  // Squares of 16-bit types are exact in float32 (16 and 22 significant bits)
  // where they stay in its range, which leaves one addition in double: fewer
  // operations, and less power (403 M bfloat16 elements on end: 121 us, 136 with
  // the squares in double).  A sum that is not well inside the range is formed
  // again by norm_part, which takes every value, unless all elements are zero.
  constexpr bool kHalf = std::is_same<T, __half>::value;
  double lo = 0.0, hi = 0.0;
  uint32_t any = 0;
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      any |= w[u][j];
      const float2 x = unpack2<T>(&w[u][j]);
      const float2 p = __fmul2_rn(x, x);
      lo += square_bits<kHalf>(p.x);
      hi += square_bits<kHalf>(p.y);
    }
  }
  const double sum = (lo + hi) * 0x1p896;
  const bool fine = (sum >= 0x1p-90 && sum < 0x1p120) || !(any & 0x7FFF7FFFu);
  return __any_sync(0xffffffffu, !fine) ? norm_part(g, n) : sum;
}

// The CTA's chunks, one for each 256 of its threads at a time.
template <int N>
__device__ __forceinline__ double norm_chunks(const NormTable<N>& t) {
  const int groups = blockDim.x / kNormThreads;
  double acc = 0.0;
  int k = 0, end = 0;  // the entry of the chunk before, and the chunk after its last
#pragma unroll 1
  for (int c = blockIdx.x + gridDim.x * (threadIdx.x / kNormThreads); c < t.chunks;
       c += gridDim.x * groups) {
    if (c >= end) {
      k = find_entry(t.first, t.count, c);
      end = k + 1 < t.count ? t.first[k + 1] : t.chunks;
    }
    const NormEntry& e = t.e[k];
    const int chunk = c - t.first[k];
    const bool vec = (t.word[k] & 4) != 0;
    switch (t.word[k] & 3) {
      case CS_F32: acc += norm_chunk<float>(e.g, chunk, e.numel, vec); break;
      case CS_BF16: acc += norm_chunk<__nv_bfloat16>(e.g, chunk, e.numel, vec); break;
      default: acc += norm_chunk<__half>(e.g, chunk, e.numel, vec); break;
    }
  }
  return block_sum_d(acc);
}

template <int N>
__global__ void __launch_bounds__(kNormThreads)
    grad_norm_kernel(const __grid_constant__ NormTable<N> t) {
  const double acc = norm_chunks(t);
  if (threadIdx.x == 0) t.partials[blockIdx.x] = acc;
}

struct NormOut {
  double max_norm, eps;
  float *norm, *scale;
  __device__ __forceinline__ void write(double sum) const {
    const double r = sqrt(sum);
    *norm = (float)r;
    if (scale) {
      const double q = max_norm / (r + eps);
      *scale = max_norm > 0.0 ? (q > 1.0 ? 1.0f : (float)q) : 1.0f;  // NaN stays NaN
    }
  }
};

// The whole norm in one cluster of 16 full CTAs (2 MB of loads in flight), which
// leave their sums in the first one's shared memory.
constexpr int kNormCluster = 16, kNormGroups = 4;

template <int N>
__global__ void __launch_bounds__(kNormThreads * kNormGroups)
    grad_norm_small_kernel(const __grid_constant__ NormTable<N> t, NormOut out) {
  __shared__ double sums[kNormCluster];
  // the first CTA has to have started before another one writes to it
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  const double acc = norm_chunks(t);
  asm volatile("barrier.cluster.wait;" ::: "memory");
  if (threadIdx.x == 0) {
    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(sums + blockIdx.x);
    uint32_t first;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(first) : "r"(mine));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(first), "d"(acc) : "memory");
  }
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::
                   : "memory");
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    double sum = 0.0;
    for (int i = 0; i < kNormCluster; ++i) sum += sums[i];
    out.write(sum);
  }
}

__global__ void __launch_bounds__(256)
    grad_norm_finish_kernel(const double* __restrict__ partials, int n, NormOut out) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) acc += partials[i];
  acc = block_sum_d(acc);
  if (threadIdx.x == 0) out.write(acc);
}

// ---------------------------------------------------------------------------
// Host side

inline int dtype_size(int d) { return d == CS_F32 ? 4 : 2; }
inline bool aligned_to(const void* q, int bytes) {
  return (reinterpret_cast<uintptr_t>(q) & (uintptr_t)(bytes - 1)) == 0;
}

struct GroupBuilder {
  AdamGroup g[CS_ADAMW_MAX_GROUPS];
  int fill(const cs_adamw_group* groups, int n, bool counted, uint32_t seed) {
    for (int i = 0; i < n; ++i) {
      const cs_adamw_group& s = groups[i];
      if (!(s.beta1 >= 0.0 && s.beta1 < 1.0 && s.beta2 >= 0.0 && s.beta2 < 1.0)) return CS_ERR_ARG;
      if ((!counted && s.step < 1) || !aligned_to(s.lr_device, 4)) return CS_ERR_ARG;
      AdamGroup& d = g[i];
      d.b1 = (float)s.beta1;
      d.omb1 = (float)(1.0 - s.beta1);
      d.b2 = (float)s.beta2;
      d.omb2 = (float)(1.0 - s.beta2);
      d.eps = (float)s.eps;
      d.lr = (float)s.lr;
      d.wd = (float)s.weight_decay;
      d.lr_dev = s.lr_device;
      d.ibc1 = d.rbc2 = 0.0f;
      d.key = 0;
      if (!counted) {
        d.ibc1 = (float)(1.0 / (1.0 - std::pow(s.beta1, (double)s.step)));
        d.rbc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(s.beta2, (double)s.step)));
        d.key = step_key(seed, (uint32_t)s.step);
      }
    }
    for (int i = n; i < CS_ADAMW_MAX_GROUPS; ++i) g[i] = AdamGroup{};
    return CS_OK;
  }
};

// An entry holds elements [at, at + n) of a tensor.  Wide accesses need
// parameters and gradients (in cs_adamw8_moments the outputs) aligned to
// `width` bytes.
inline void make_entry(const cs_adamw_tensor& s, int place, int width, int64_t at, int64_t n,
                       AdamEntry& e) {
  const int64_t bytes = at * dtype_size(s.dtype);
  e.p = static_cast<char*>(s.param) + bytes;
  e.g = static_cast<const char*>(s.grad) + bytes;
  e.m = static_cast<float*>(s.exp_avg) + at;
  e.v = static_cast<float*>(s.exp_avg_sq) + at;
  e.numel = n;
  const bool moments = aligned_to(e.m, 16) && aligned_to(e.v, 16);
  e.word = entry_word(s.dtype, moments && aligned_to(e.p, width) && aligned_to(e.g, width),
                      moments, s.group, place);
  e.pad = 0;
}

inline void make_entry(const cs_adamw_tensor& s, int place, int width, int64_t at, int64_t n,
                       AdamEntry8& e) {
  const int64_t bytes = at * dtype_size(s.dtype), block = at / kBlock8;
  e.p = static_cast<char*>(s.param) + bytes;
  e.g = static_cast<const char*>(s.grad) + bytes;
  e.m = static_cast<uint8_t*>(s.exp_avg) + at;
  e.v = static_cast<uint8_t*>(s.exp_avg_sq) + at;
  e.ms = s.exp_avg_scales + block;
  e.vs = s.exp_avg_sq_scales + block;
  e.numel = n;
  const bool moments = aligned_to(e.m, 8) && aligned_to(e.v, 8);
  e.word = entry_word(s.dtype, moments && aligned_to(e.p, width) && aligned_to(e.g, width),
                      moments, s.group, place);
  e.block0 = (uint32_t)block;
}

// A CTA takes several chunks (a power of two) where enough CTAs are left an SM:
// eight for two chunks and 16 for more, or 56 where all parameters are float32,
// whose next block is not prefetched, so that only the end of the launch counts.
// Measured with 8-bit moments: 7 M elements in 300 tensors of all types 22 us
// with one chunk, 18 with two; 33 M bfloat16 elements 31 us with 16 CTAs an SM,
// 37 with 56; 150 M float32 elements 372 and 358 us.
constexpr int64_t ctas_wanted(int shift, bool half) {
  return 148 * (shift == 1 ? 8 : half ? 16 : 56);
}

// The kernels of one table type, by name.
struct RunStep {
  static constexpr int kWidth = 16, kMostPer = 1, kMomentBytes = 4;
  template <int N>
  static void launch(const Table<AdamEntry, N>& t, int chunks, cudaStream_t st) {
    adamw_kernel<N><<<chunks, kChunkThreads, 0, st>>>(t);
  }
};
struct RunStep8 {
  static constexpr int kWidth = 16, kMostPer = 32, kMomentBytes = 1;
  template <int N>
  static void launch(const Table<AdamEntry8, N>& t, int chunks, cudaStream_t st) {
    adamw8_kernel<N><<<chunks, kChunkThreads, 0, st>>>(t);
  }
};
struct RunMoments8 {
  static constexpr int kWidth = 32, kMostPer = 1, kMomentBytes = 1;
  template <int N>
  static void launch(const Table<AdamEntry8, N>& t, int chunks, cudaStream_t st) {
    adamw8_moments_kernel<N><<<chunks, kChunkThreads, 0, st>>>(t);
  }
};

// What a table holds beside its tensors.
struct Common {
  const AdamGroup* groups;  // CS_ADAMW_MAX_GROUPS, or NULL
  const float* coef;
  bool each;
  int first_place;
  const float* grad_scale;
};

// Packs tensors (empty ones left out) into tables of at most N entries and
// launches each full one.
template <class Run, class Entry, int N>
int launch_tables(const cs_adamw_tensor* tensors, int count, const Common& c, cudaStream_t st) {
  Table<Entry, N> t;
  t.one = 1.0f;
  t.place_key = place_key((uint32_t)c.first_place);
  t.grad_scale = c.grad_scale;
  t.coef = c.coef;
  t.each = c.each;
  for (int i = 0; i < CS_ADAMW_MAX_GROUPS; ++i)
    t.groups[i] = c.groups ? c.groups[i] : AdamGroup{};
  int64_t total = 0;
  bool half = false;
  for (int i = 0; i < count; ++i) {
    total += (tensors[i].numel + kChunk - 1) / kChunk;
    half |= tensors[i].dtype != CS_F32;
  }
  int shift = 0;
  while ((1 << shift) < Run::kMostPer &&
         (total >> (shift + 1)) >= ctas_wanted(shift + 1, half))
    ++shift;
  t.shift = shift;
  static_assert(kChunk == 1024, "10 bits");
  shift += 10;
  t.count = 0;
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    const cs_adamw_tensor& s = tensors[i];
    for (int64_t at = 0; at < s.numel; at += kMaxEntry) {
      const int64_t n = s.numel - at < kMaxEntry ? s.numel - at : kMaxEntry;
      const int64_t mine = (n + (int64_t(1) << shift) - 1) >> shift;
      if (t.count == N || chunks + mine > INT32_MAX) {
        Run::template launch<N>(t, (int)chunks, st);
        if (int rc = launch_status()) return rc;
        t.count = 0;
        chunks = 0;
      }
      make_entry(s, i, Run::kWidth, at, n, t.e[t.count]);
      t.first[t.count++] = (int)chunks;
      chunks += mine;
    }
  }
  if (t.count == 0) return CS_OK;
  Run::template launch<N>(t, (int)chunks, st);
  return launch_status();
}

// Everything that a call can refuse, before its first launch: `bytes` are those of
// a moment's element, one with scales beside it.
inline int check_tensors(const cs_adamw_tensor* tensors, int count, int groups, int bytes) {
  if (count < 0 || count > kMaxTensors || (count > 0 && !tensors)) return CS_ERR_ARG;
  for (int i = 0; i < count; ++i) {
    const cs_adamw_tensor& s = tensors[i];
    if (s.numel < 0 || s.numel > kMaxNumel || s.dtype < CS_F32 || s.dtype > CS_F16 ||
        s.group < 0 || s.group >= groups)
      return CS_ERR_ARG;
    const int size = dtype_size(s.dtype);
    if (!aligned_to(s.param, size) || !aligned_to(s.grad, size)) return CS_ERR_ARG;
    if (s.numel == 0) continue;
    if (!s.param || !s.grad || !s.exp_avg || !s.exp_avg_sq || !aligned_to(s.exp_avg, bytes) ||
        !aligned_to(s.exp_avg_sq, bytes) ||
        (bytes == 1 && (!s.exp_avg_scales || !s.exp_avg_sq_scales)))
      return CS_ERR_ARG;
  }
  return CS_OK;
}

// A call of few tensors takes a small table (its parameters stay below 4 KB).
template <class Run, class Entry, int kSmall, int kLarge>
int run_tables(const cs_adamw_tensor* tensors, int count, const Common& c, cudaStream_t st) {
  static_assert(sizeof(Table<Entry, kLarge>) <= 32764, "kernel parameter limit");
  if (count <= kSmall) return launch_tables<Run, Entry, kSmall>(tensors, count, c, st);
  return launch_tables<Run, Entry, kLarge>(tensors, count, c, st);
}

// Advances `count` device counters; that of tensor i belongs to group of(i).
template <int N, class Of>
int launch_advance(int64_t* const* steps, int count, const Of& of, const cs_adamw_group* groups,
                   int num_groups, uint32_t seed, float* coef, cudaStream_t st) {
  CountTable<N> a;
  a.seed = seed;
  for (int i = 0; i < CS_ADAMW_MAX_GROUPS; ++i) {
    a.b1[i] = i < num_groups ? groups[i].beta1 : 0.0;
    a.b2[i] = i < num_groups ? groups[i].beta2 : 0.0;
  }
  for (int at = 0; at < count; at += N) {
    a.count = count - at < N ? count - at : N;
    a.coef = coef + 4 * (int64_t)at;
    for (int i = 0; i < a.count; ++i) {
      a.step[i] = steps[at + i];
      a.group[i] = (uint8_t)of(at + i);
    }
    adamw_advance_kernel<N>
        <<<(a.count + kCountThreads - 1) / kCountThreads, kCountThreads, 0, st>>>(a);
    if (int rc = launch_status()) return rc;
  }
  return CS_OK;
}

// Counters of a launch.  The large table stays below 4 KB: a launch with 4 KB of
// parameters takes the host 2.3 us, with 32 KB 5.4.
constexpr int kCountSmall = 16, kCountLarge = 400;
static_assert(sizeof(CountTable<kCountLarge>) <= 4096, "a short launch");

// A step counted on the host, by device counters of the groups (coef, which
// cs_adamw_advance wrote), or by one of each tensor (steps, which are advanced
// here; work holds what they give).
template <class Run, class Entry, int kSmall, int kLarge>
int step_entry(const cs_adamw_tensor* tensors, int count, const cs_adamw_group* groups,
               int num_groups, int64_t* const* steps, float* work, const float* coef,
               uint32_t seed, int first_place, const float* grad_scale, void* stream) {
  if (num_groups < 1 || num_groups > CS_ADAMW_MAX_GROUPS || !groups || first_place < 0 ||
      !aligned_to(coef, 4) || !aligned_to(grad_scale, 4))
    return CS_ERR_ARG;
  if (int rc = check_tensors(tensors, count, num_groups, Run::kMomentBytes)) return rc;
  if (steps) {
    if (!work || !aligned_to(work, 4)) return CS_ERR_ARG;
    for (int i = 0; i < count; ++i)
      if (!steps[i] || !aligned_to(steps[i], 8)) return CS_ERR_ARG;
    coef = work;
  }
  GroupBuilder b;
  if (int rc = b.fill(groups, num_groups, coef != nullptr, seed)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (steps) {
    const auto of = [tensors](int i) { return tensors[i].group; };
    const int rc = count <= kCountSmall
                       ? launch_advance<kCountSmall>(steps, count, of, groups, num_groups, seed,
                                                     work, st)
                       : launch_advance<kCountLarge>(steps, count, of, groups, num_groups, seed,
                                                     work, st);
    if (rc) return rc;
  }
  return run_tables<Run, Entry, kSmall, kLarge>(
      tensors, count, Common{b.g, coef, steps != nullptr, first_place, grad_scale}, st);
}

template <int N>
void add_norm_entry(NormTable<N>& t, const cs_grad_tensor& s) {
  if (s.numel == 0) return;
  const int each = norm_chunk_of(s.dtype);
  t.e[t.count] = NormEntry{s.data, s.numel};
  t.word[t.count] = (uint8_t)(s.dtype | (aligned_to(s.data, 16) ? 4 : 0));
  t.first[t.count++] = t.chunks;
  t.chunks += (int)((s.numel + each - 1) / each);
}

template <int N>
int launch_norm(const cs_grad_tensor* tensors, int count, double* partials, int& used,
                cudaStream_t st) {
  NormTable<N> t;
  t.count = 0;
  t.chunks = 0;
  auto flush = [&]() {
    const int blocks = t.chunks < kNormBlocks ? t.chunks : kNormBlocks;
    t.partials = partials + used;
    grad_norm_kernel<N><<<blocks, kNormThreads, 0, st>>>(t);
    used += blocks;
    t.count = 0;
    t.chunks = 0;
    return launch_status();
  };
  for (int i = 0; i < count; ++i) {  // a tensor has at most 2^25 chunks
    if (t.count == N || t.chunks > INT32_MAX / 2)
      if (int rc = flush()) return rc;
    add_norm_entry(t, tensors[i]);
  }
  return t.count ? flush() : (int)CS_OK;
}

// Chunks of a call, and how many still go in one launch of one cluster.
constexpr int64_t kNormOneLaunch = 128;
inline int64_t norm_chunk_count(const cs_grad_tensor* tensors, int count) {
  int64_t n = 0;
  for (int i = 0; i < count; ++i) {
    const int each = norm_chunk_of(tensors[i].dtype);
    n += (tensors[i].numel + each - 1) / each;
  }
  return n;
}

// A call without chunks (nothing to add) goes that way too.
template <int N>
int launch_norm_small(const cs_grad_tensor* tensors, int count, const NormOut& out,
                      cudaStream_t st) {
  NormTable<N> t;
  t.count = 0;
  t.chunks = 0;
  t.partials = nullptr;
  for (int i = 0; i < count; ++i) add_norm_entry(t, tensors[i]);
  // a cluster of more than eight CTAs has to be asked for, on each device
  if (cudaFuncSetAttribute(grad_norm_small_kernel<N>,
                           cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return CS_ERR_CUDA;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = kNormCluster;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kNormCluster);
  cfg.blockDim = dim3(kNormThreads * kNormGroups);
  cfg.stream = st;
  cfg.attrs = &cluster;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, grad_norm_small_kernel<N>, t, out) != cudaSuccess)
    return CS_ERR_CUDA;
  return launch_status();
}

constexpr int kNormSmall = 128, kNormLarge = 1400;
static_assert(sizeof(NormTable<kNormLarge>) <= 32764, "kernel parameter limit");

}  // namespace cs

using namespace cs;

extern "C" {

int cs_adamw_step(const cs_adamw_tensor* tensors, int32_t count, const cs_adamw_group* groups,
                  int32_t num_groups, const float* coef, const float* grad_scale, void* stream) {
  return step_entry<RunStep, AdamEntry, 40, 560>(tensors, count, groups, num_groups, nullptr,
                                                 nullptr, coef, 0, 0, grad_scale, stream);
}

int cs_adamw_step_counted(const cs_adamw_tensor* tensors, int32_t count,
                          const cs_adamw_group* groups, int32_t num_groups, int64_t* const* steps,
                          float* workspace, const float* grad_scale, void* stream) {
  if (!steps) return CS_ERR_ARG;
  return step_entry<RunStep, AdamEntry, 40, 560>(tensors, count, groups, num_groups, steps,
                                                 workspace, nullptr, 0, 0, grad_scale, stream);
}

int cs_adamw8_step_at(const cs_adamw_tensor* tensors, int32_t count, const cs_adamw_group* groups,
                      int32_t num_groups, const float* coef, uint32_t seed, int32_t first_place,
                      const float* grad_scale, void* stream) {
  return step_entry<RunStep8, AdamEntry8, 36, 420>(tensors, count, groups, num_groups, nullptr,
                                                   nullptr, coef, seed, first_place, grad_scale,
                                                   stream);
}

int cs_adamw8_step(const cs_adamw_tensor* tensors, int32_t count, const cs_adamw_group* groups,
                   int32_t num_groups, const float* coef, uint32_t seed, const float* grad_scale,
                   void* stream) {
  return cs_adamw8_step_at(tensors, count, groups, num_groups, coef, seed, 0, grad_scale, stream);
}

int cs_adamw8_step_counted(const cs_adamw_tensor* tensors, int32_t count,
                           const cs_adamw_group* groups, int32_t num_groups, int64_t* const* steps,
                           float* workspace, uint32_t seed, int32_t first_place,
                           const float* grad_scale, void* stream) {
  if (!steps) return CS_ERR_ARG;
  return step_entry<RunStep8, AdamEntry8, 36, 420>(tensors, count, groups, num_groups, steps,
                                                   workspace, nullptr, seed, first_place,
                                                   grad_scale, stream);
}

int cs_adamw8_moments(const cs_adamw_tensor* tensors, int32_t count, void* stream) {
  if (int rc = check_tensors(tensors, count, 1, RunMoments8::kMomentBytes)) return rc;
  for (int i = 0; i < count; ++i)
    if (tensors[i].dtype != CS_F32) return CS_ERR_ARG;
  return run_tables<RunMoments8, AdamEntry8, 36, 420>(
      tensors, count, Common{nullptr, nullptr, false, 0, nullptr}, (cudaStream_t)stream);
}

int cs_adamw_advance(int64_t* const* steps, const cs_adamw_group* groups, int32_t num_groups,
                     uint32_t seed, float* coef, void* stream) {
  if (!steps || !groups || !coef || !aligned_to(coef, 4) || num_groups < 1 ||
      num_groups > CS_ADAMW_MAX_GROUPS)
    return CS_ERR_ARG;
  for (int i = 0; i < num_groups; ++i) {
    if (!steps[i] || !aligned_to(steps[i], 8)) return CS_ERR_ARG;
    for (int j = 0; j < i; ++j)
      if (steps[j] == steps[i]) return CS_ERR_ARG;  // each counter advances once
  }
  static_assert(CS_ADAMW_MAX_GROUPS <= kCountSmall, "one launch");
  return launch_advance<kCountSmall>(steps, num_groups, [](int i) { return i; }, groups,
                                     num_groups, seed, coef, (cudaStream_t)stream);
}

size_t cs_grad_norm_workspace_size(const cs_grad_tensor* tensors, int32_t count) {
  if (count <= 0 || count > kMaxTensors || !tensors) return 0;
  const int64_t chunks = norm_chunk_count(tensors, count);
  if (chunks <= kNormOneLaunch) return 0;
  const int each = count <= kNormSmall ? kNormSmall : kNormLarge;
  const size_t launches = (size_t)(count / each + 1 + chunks / (INT32_MAX / 2));
  return launches * kNormBlocks * sizeof(double);
}

int cs_grad_norm(const cs_grad_tensor* tensors, int32_t count, double max_norm, double eps,
                 float* norm, float* scale, void* workspace, void* stream) {
  if (count < 0 || count > kMaxTensors || (count > 0 && !tensors) || !norm ||
      !aligned_to(norm, 4) || !aligned_to(scale, 4) || !aligned_to(workspace, 8))
    return CS_ERR_ARG;
  for (int i = 0; i < count; ++i)
    if (tensors[i].numel < 0 || tensors[i].numel > kMaxNumel || tensors[i].dtype < CS_F32 ||
        tensors[i].dtype > CS_F16 || (tensors[i].numel > 0 && !tensors[i].data) ||
        !aligned_to(tensors[i].data, dtype_size(tensors[i].dtype)))
      return CS_ERR_ARG;
  cudaStream_t st = (cudaStream_t)stream;
  const NormOut out{max_norm, eps, norm, scale};
  if (norm_chunk_count(tensors, count) <= kNormOneLaunch) {
    // a tensor with elements has a chunk, so the table holds them all
    static_assert(kNormOneLaunch <= kNormSmall, "one entry a chunk at most");
    return launch_norm_small<kNormSmall>(tensors, count, out, st);
  }
  if (!workspace) return CS_ERR_ARG;
  double* partials = static_cast<double*>(workspace);
  int used = 0;
  const int rc = count <= kNormSmall
                     ? launch_norm<kNormSmall>(tensors, count, partials, used, st)
                     : launch_norm<kNormLarge>(tensors, count, partials, used, st);
  if (rc) return rc;
  grad_norm_finish_kernel<<<1, 256, 0, st>>>(partials, used, out);
  return launch_status();
}

}  // extern "C"
