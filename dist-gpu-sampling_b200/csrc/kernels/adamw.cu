// One AdamW step over a list of tensors, moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = (1 - lr wd) p - (m / (sqrt(v) / sqrt(1 - b2^t) + eps)) (lr / (1 - b1^t)),  copy = p in the copy's type
//
// Every element is read and written once: bound by HBM with moments in 32 bits (313 M parameters, gradients and copies in 16 bits:
// 1.44 ms, 6.1 TB/s), by issue slots in 8 bits (60 M parameters: nearest codes 252 us,
// 3.8 TB/s, some hundred instructions an element; unbiased ones 358).
//
// The moments lie in flat buffers in which every tensor has a slot of whole 256-element blocks, so a warp's 256 elements are one
// block of the 8-bit form and the list needs three pointers a tensor.  The list travels in the kernel's parameters (nothing is
// copied to the device and nothing is kept), a CTA finds its tensor by bisecting the list's chunk numbers.
//
// 8 bits, per block: m = a sgn(c) (c / 127)^2 with a = max |m|, and sqrt(v) = a (c / 255)^2 with a = max sqrt(v).  The
// squares give small values finer steps; the second moment is held as its root because that is what divides, and a root
// that is not zero never gets the code zero, which would make its element's step arbitrarily large.
//
// A code is the nearest one, or (unbiased) the one below or above with the probabilities that leave the moment its mean.  The nearest
// code is the better one for a single step, and over many it holds a moment fast: with b2 = 0.999 a moment changes by at most
// 0.1 % a step downwards, and half a code is 2 / c of it, 0.8 % at c = 255, so beside a moment that grows or stays the
// others of its block hardly fall, and grow only by large gradients.  256 elements, the gradients of half of them cut tenfold at
// step 2000: their stored roots are 2.6 times the exact ones at step 4000 and 9.6 times at 8000, and the parameters have moved
// 31 % wrong; unbiased, 0.99 times (a single one up to 1.3) and 6 %.  The random words are Philox's of (seed, step, element),
// so the same call gives the same bits, whatever the launch.
//
// The arithmetic is 32-bit, operation by operation as written above: no contraction to fused multiply-add, IEEE division
// and square root.  A moment that falls between two codes is then rounded the same way wherever the formula is evaluated
// in 32 bits.
#include <cmath>
#include <type_traits>

#include "philox.cuh"
#include "train_common.cuh"

namespace dgs {
namespace {

constexpr int AW_THREADS = 256;
constexpr int AW_BLOCK = 256;                                // elements that share a scale: 8 a lane
constexpr int AW_VALUES = 8;
constexpr int64_t AW_CHUNK = AW_THREADS * AW_VALUES;         // elements a CTA takes at a time: 8 blocks
constexpr int AW_SMALL_LIST = 64, AW_LARGE_LIST = 512;       // tensors of one launch (parameters of 3.6 and 28 KB)

struct Entry {
  void* param;
  const void* grad;
  void* copy;
  int64_t n;
  int64_t at;          // first element of the slot in the moments
  int64_t first_chunk;
  int8_t param_dtype, grad_dtype, copy_dtype;
  int8_t whole;        // every pointer allows accesses of 8 elements
};
template <int N>
struct List {
  Entry e[N];
};
struct Scalars {
  float keep, b1, c1, b2, c2, root2, eps, step;
};

struct Moments32 {
  float* m;
  float* v;
};
struct Moments8 {
  int8_t* m;
  float* m_scale;
  uint8_t* v;
  float* v_scale;
};
struct Moments8Unbiased : Moments8 {
  uint64_t key;  // of the step's random words
};

// the new parameter; `root` receives that of the second moment
__device__ __forceinline__ float update(float p, float g, float& m, float& v, float& root, const Scalars& k) {
  m = __fadd_rn(__fmul_rn(m, k.b1), __fmul_rn(g, k.c1));
  v = __fadd_rn(__fmul_rn(v, k.b2), __fmul_rn(__fmul_rn(g, g), k.c2));
  root = __fsqrt_rn(v);
  const float under = __fadd_rn(__fmul_rn(root, k.root2), k.eps);
  return __fsub_rn(__fmul_rn(p, k.keep), __fmul_rn(__fdiv_rn(m, under), k.step));
}

// the largest of the warp's non-negative values; a NaN counts as larger than any (its bits are)
__device__ __forceinline__ float warp_max_bits(uint32_t bits) { return __uint_as_float(__reduce_max_sync(FULL_MASK, bits)); }

// Codes and values.  A byte becomes a float by standing in the low bits of 2^23 (8388608), and a float its nearest whole number
// there by adding 1.5 * 2^23 (12582912): the units that convert take 16 values a clock and SM, which square roots and divisions
// need here.
constexpr float kByte = 8388608.0f, kRound = 12582912.0f;
template <bool SIGNED>
__device__ __forceinline__ float code_value(uint32_t word, int byte) {  // byte 0..3 of a word of codes (known when compiled)
  const uint32_t bits = __byte_perm(SIGNED ? word ^ 0x80808080u : word, 0x4B000000u, 0x7440u + byte);
  return __fsub_rn(__uint_as_float(bits), SIGNED ? kByte + 128.0f : kByte);
}
// Two at a time where nothing but multiplications follow one another (a packed addition behind a packed multiplication may become
// one operation with one rounding).
__device__ __forceinline__ uint64_t both(float v) { return two(v, v); }
__device__ __forceinline__ uint64_t abs2(uint64_t v) { return v & 0x7fffffff7fffffffull; }
// of bytes `byte` and byte + 1
__device__ __forceinline__ void first_moments(uint32_t word, int byte, float scale, float* m0, float* m1) {
  const uint64_t u = mul2(two(code_value<true>(word, byte), code_value<true>(word, byte + 1)), both(1.0f / 127.0f));
  split2(mul2(mul2(u, abs2(u)), both(scale)), m0, m1);
}
__device__ __forceinline__ void second_moments(uint32_t word, int byte, float scale, float* v0, float* v1) {
  const uint64_t u = mul2(two(code_value<false>(word, byte), code_value<false>(word, byte + 1)), both(1.0f / 255.0f));
  const uint64_t r = mul2(mul2(u, u), both(scale));
  split2(mul2(r, r), v0, v1);
}

__device__ __forceinline__ float sqrt_near(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The code of x is rint(steps * sqrt(x / scale)), 0 <= x <= scale, each operation rounded to nearest.
__device__ __forceinline__ float exact_code(float x, float scale, float steps) {
  // (a scale of zero, or one that is no number, leaves the code zero)
  return scale > 0.0f ? rintf(__fmul_rn(__fsqrt_rn(__fdiv_rn(x, scale)), steps)) : 0.0f;
}
// The same for two without the IEEE division and root: the values before rint are within steps * 4.3e-7 of those above (six
// roundings of 2^-24, two of them halved by the root, and sqrt.approx with 2^-23), so the codes are the same unless one stands that
// near to a half.  `far` collects how far the values are from their codes; `inverse` = 1 / scale.
__device__ __forceinline__ void quick_codes(uint64_t x, float inverse, float steps, float& far, float* c0, float* c1) {
  float a, b;
  split2(mul2(x, both(inverse)), &a, &b);
  const uint64_t value = mul2(two(sqrt_near(a), sqrt_near(b)), both(steps));
  const uint64_t whole = add2(add2(value, both(kRound)), both(-kRound));
  split2(fma2(whole, both(-1.0f), value), &a, &b);
  far = fmaxf(far, fmaxf(fabsf(a), fabsf(b)));
  split2(whole, c0, c1);
}
// The code below a value, or the one above with the probability that leaves the value its mean.  A whole number may count as the one
// above its predecessor with probability one.  The largest value's code is the last one.  Of an element's 32 random bits 11 are
// the first moment's and 21 the second's, whose small changes go by small probabilities (0.001 c / 4 with b2 = 0.999).
__device__ __forceinline__ float whole_below(float x) { return __fsub_rn(__fadd_rn(__fsub_rn(x, 0.5f), kRound), kRound); }
// (`bits` of 23, as a number between 0 and 1)
__device__ __forceinline__ float unit(uint32_t bits, float half) { return __uint_as_float(0x3f800000u | bits) - (1.0f - half); }
__device__ __forceinline__ float unbiased_first(float part, uint32_t random) {  // part of the scale = (c / 127)^2
  const float q = part * 16129.0f, c = whole_below(sqrt_near(q)), u = unit((random & 2047u) << 12, 0x1p-12f);
  return fminf(u * (2.0f * c + 1.0f) < q - c * c ? c + 1.0f : c, 127.0f);
}
__device__ __forceinline__ float unbiased_second(float part, uint32_t random) {  // part of the scale = (c / 255)^2, of its square ^4
  const float s = part * 65025.0f, c = whole_below(sqrt_near(s)), cc = c * c, above = cc + (2.0f * c + 1.0f);
  const float u = unit((random >> 11) << 2, 0x1p-22f);
  return fminf(u * ((above - cc) * (above + cc)) < (s - cc) * (s + cc) ? c + 1.0f : c, 255.0f);
}
// the low bytes of four whole numbers
__device__ __forceinline__ uint32_t bytes_of(float a, float b, float c, float d) {
  const uint32_t ab = __byte_perm(__float_as_uint(a + kRound), __float_as_uint(b + kRound), 0x0040);
  const uint32_t cd = __byte_perm(__float_as_uint(c + kRound), __float_as_uint(d + kRound), 0x0040);
  return __byte_perm(ab, cd, 0x5410);
}

template <int N, typename Moments>
__global__ void __launch_bounds__(AW_THREADS) adamw_kernel(const __grid_constant__ List<N> list, const int count,
                                                           const int64_t chunks, const Moments mo,
                                                           const __grid_constant__ Scalars k) {
  constexpr bool kEight = std::is_base_of<Moments8, Moments>::value, kUnbiased = std::is_same<Moments, Moments8Unbiased>::value;
  pdl_enter();
  for (int64_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (list.e[mid].first_chunk <= chunk) lo = mid;
      else hi = mid - 1;
    }
    const Entry& e = list.e[lo];
    const int64_t i = (chunk - e.first_chunk) * AW_CHUNK + static_cast<int64_t>(threadIdx.x) * AW_VALUES;
    // whole warps leave together: a warp that has any element takes part with all its lanes (the scales of a block)
    if (e.n - (i - static_cast<int64_t>(threadIdx.x & 31) * AW_VALUES) <= 0) continue;
    const int left = e.n - i >= AW_VALUES ? AW_VALUES : e.n > i ? static_cast<int>(e.n - i) : 0;  // this thread's elements
    float p[AW_VALUES], g[AW_VALUES], m[AW_VALUES], v[AW_VALUES], root[AW_VALUES];
    const bool full = e.whole && left == AW_VALUES;
    if (full) {
      load_vec_as_float<AW_VALUES>(e.param, e.param_dtype, i, p);
      load_vec_as_float<AW_VALUES>(e.grad, e.grad_dtype, i, g);
    } else {
#pragma unroll
      for (int j = 0; j < AW_VALUES; ++j) {
        p[j] = j < left ? load_as_float(e.param, e.param_dtype, i + j) : 0.0f;
        g[j] = j < left ? load_as_float(e.grad, e.grad_dtype, i + j) : 0.0f;
      }
    }
    const int64_t at = e.at + i;
    if constexpr (kEight) {
      // a slot is whole blocks, so all eight codes are there; those beyond the tensor's end count as zero
      const uint2 mc = *reinterpret_cast<const uint2*>(mo.m + at), vc = *reinterpret_cast<const uint2*>(mo.v + at);
      const float ma = mo.m_scale[at / AW_BLOCK], va = mo.v_scale[at / AW_BLOCK];
#pragma unroll
      for (int j = 0; j < AW_VALUES; j += 2) {
        first_moments(j < 4 ? mc.x : mc.y, j & 3, ma, &m[j], &m[j + 1]);
        second_moments(j < 4 ? vc.x : vc.y, j & 3, va, &v[j], &v[j + 1]);
      }
    } else {
      load_vec<float, AW_VALUES>(mo.m + at, m);
      load_vec<float, AW_VALUES>(mo.v + at, v);
    }
#pragma unroll
    for (int j = 0; j < AW_VALUES; ++j) p[j] = update(p[j], g[j], m[j], v[j], root[j], k);
    if (full) {
      store_vec_from_float<AW_VALUES>(e.param, e.param_dtype, i, p);
      if (e.copy != nullptr) store_vec_from_float<AW_VALUES>(e.copy, e.copy_dtype, i, p);
    } else {
#pragma unroll
      for (int j = 0; j < AW_VALUES; ++j) {
        if (j < left) {
          store_from_float(e.param, e.param_dtype, i + j, p[j]);
          if (e.copy != nullptr) store_from_float(e.copy, e.copy_dtype, i + j, p[j]);
        }
      }
    }
    if constexpr (kEight) {
      if (left < AW_VALUES) {
#pragma unroll
        for (int j = 0; j < AW_VALUES; ++j)
          if (j >= left) m[j] = root[j] = 0.0f;
      }
      uint32_t mb = 0, vb = 0;
#pragma unroll
      for (int j = 0; j < AW_VALUES; ++j) {
        mb = max(mb, __float_as_uint(fabsf(m[j])));
        vb = max(vb, __float_as_uint(root[j]));
      }
      const float ma = warp_max_bits(mb), va = warp_max_bits(vb);
      const bool plain = ma >= 1e-30f && ma <= 1e30f && va >= 1e-30f && va <= 1e30f;  // scales that have an inverse
      const float mi = __fdiv_rn(1.0f, ma), vi = __fdiv_rn(1.0f, va);
      float mc[AW_VALUES], vc[AW_VALUES];
      if constexpr (kUnbiased) {
#pragma unroll
        for (int j = 0; j < AW_VALUES; j += 4) {
          const uint64_t four_of = static_cast<uint64_t>(at + j) >> 2;
          const Philox4 r = philox4x32_10(mo.key, static_cast<uint32_t>(four_of), static_cast<uint32_t>(four_of >> 32), 0u, 0u);
          const uint32_t random[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float mp = plain ? fabsf(m[j + i]) * mi : ma > 0.0f ? __fdiv_rn(fabsf(m[j + i]), ma) : 0.0f;
            const float vp = plain ? root[j + i] * vi : va > 0.0f ? __fdiv_rn(root[j + i], va) : 0.0f;
            mc[j + i] = unbiased_first(mp, random[i]);
            vc[j + i] = unbiased_second(vp, random[i]);
          }
        }
      } else {
        float far_m = 0.0f, far_v = 0.0f;
#pragma unroll
        for (int j = 0; j < AW_VALUES; j += 2) {
          quick_codes(abs2(two(m[j], m[j + 1])), mi, 127.0f, far_m, &mc[j], &mc[j + 1]);
          quick_codes(two(root[j], root[j + 1]), vi, 255.0f, far_v, &vc[j], &vc[j + 1]);
        }
        if (!plain || far_m >= 0.5f - 127.0f * 4.3e-7f || far_v >= 0.5f - 255.0f * 4.3e-7f) {  // some lane of one warp in fourteen
#pragma unroll
          for (int j = 0; j < AW_VALUES; ++j) {
            mc[j] = exact_code(fabsf(m[j]), ma, 127.0f);
            vc[j] = exact_code(root[j], va, 255.0f);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < AW_VALUES; ++j) {
        mc[j] = copysignf(mc[j], m[j]);
        if (root[j] > 0.0f) vc[j] = fmaxf(vc[j], 1.0f);
      }
      *reinterpret_cast<uint2*>(mo.m + at) = uint2{bytes_of(mc[0], mc[1], mc[2], mc[3]), bytes_of(mc[4], mc[5], mc[6], mc[7])};
      *reinterpret_cast<uint2*>(mo.v + at) = uint2{bytes_of(vc[0], vc[1], vc[2], vc[3]), bytes_of(vc[4], vc[5], vc[6], vc[7])};
      if ((threadIdx.x & 31) == 0) {
        mo.m_scale[at / AW_BLOCK] = ma;
        mo.v_scale[at / AW_BLOCK] = va;
      }
    } else {
      if (left >= AW_VALUES) {
        store_vec<float, AW_VALUES>(mo.m + at, m);
        store_vec<float, AW_VALUES>(mo.v + at, v);
      } else {
#pragma unroll
        for (int j = 0; j < AW_VALUES; ++j) {
          if (j < left) {
            mo.m[at + j] = m[j];
            mo.v[at + j] = v[j];
          }
        }
      }
    }
  }
}

// Four codes a lane at a time, so that a warp's stores lie side by side, and four such groups under way.
template <bool SECOND>
__global__ void __launch_bounds__(AW_THREADS) adamw_values_kernel(const uint32_t* __restrict__ codes, const float* __restrict__ scales,
                                                                  const int64_t words, float4* __restrict__ out) {
  constexpr int U = 4;
  pdl_enter();
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * (AW_THREADS * U) + threadIdx.x; i0 < words;
       i0 += static_cast<int64_t>(gridDim.x) * (AW_THREADS * U)) {
    uint32_t c[U];
    float scale[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * AW_THREADS;
      c[u] = i < words ? codes[i] : 0u;
      scale[u] = i < words ? scales[i / (AW_BLOCK / 4)] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * AW_THREADS;
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        if (SECOND) second_moments(c[u], j, scale[u], &v[j], &v[j + 1]);
        else first_moments(c[u], j, scale[u], &v[j], &v[j + 1]);
      }
      if (i < words) out[i] = float4{v[0], v[1], v[2], v[3]};
    }
  }
}

int make_scalars(const char* who, double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step, Scalars* k) {
  DGS_REQUIRE(lr >= 0.0 && eps >= 0.0 && weight_decay >= 0.0, DGS_ERR_INVALID, "%s: lr, eps and weight_decay must be >= 0", who);
  DGS_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, DGS_ERR_INVALID, "%s: betas must lie in [0, 1)", who);
  DGS_REQUIRE(step >= 1, DGS_ERR_INVALID, "%s: steps count from 1", who);
  const double t = static_cast<double>(step);
  k->keep = static_cast<float>(1.0 - lr * weight_decay);
  k->b1 = static_cast<float>(beta1);
  k->c1 = static_cast<float>(1.0 - beta1);
  k->b2 = static_cast<float>(beta2);
  k->c2 = static_cast<float>(1.0 - beta2);
  k->root2 = static_cast<float>(1.0 / sqrt(1.0 - pow(beta2, t)));
  k->eps = static_cast<float>(eps);
  k->step = static_cast<float>(lr / (1.0 - pow(beta1, t)));
  return DGS_OK;
}

int check_tensor(const char* who, const dgs_adamw_tensor& t) {
  DGS_REQUIRE(t.n >= 0, DGS_ERR_INVALID, "%s: a tensor of %lld elements", who, static_cast<long long>(t.n));
  DGS_REQUIRE(t.at >= 0 && t.at % AW_BLOCK == 0, DGS_ERR_INVALID, "%s: a slot begins at a multiple of %d elements", who, AW_BLOCK);
  DGS_REQUIRE(t.n == 0 || (t.param != nullptr && t.grad != nullptr), DGS_ERR_INVALID, "%s: null tensor", who);
  DGS_REQUIRE(dtype_bytes(t.param_dtype) != 0 && dtype_bytes(t.grad_dtype) != 0 &&
                  (t.copy == nullptr || dtype_bytes(t.copy_dtype) != 0),
              DGS_ERR_UNSUPPORTED, "%s: element type", who);
  return DGS_OK;
}

template <int N, typename Moments>
int launch_list(const dgs_adamw_tensor* ts, int32_t count, const Moments& mo, const Scalars& k, cudaStream_t s) {
  List<N> list;
  int used = 0;
  int64_t chunks = 0;
  for (int32_t i = 0; i < count; ++i) {
    const dgs_adamw_tensor& t = ts[i];
    if (t.n == 0) continue;
    const bool whole = aligned_to(t.param, 16) && aligned_to(t.grad, 16) && aligned_to(t.copy, 16);
    list.e[used++] = Entry{t.param, t.grad, t.copy, t.n, t.at, chunks, static_cast<int8_t>(t.param_dtype),
                           static_cast<int8_t>(t.grad_dtype), static_cast<int8_t>(t.copy_dtype), static_cast<int8_t>(whole)};
    chunks += (t.n + AW_CHUNK - 1) / AW_CHUNK;
  }
  if (used == 0) return DGS_OK;
  const int64_t most = static_cast<int64_t>(sm_count()) * 8;
  DGS_CUDA_TRY(launch_training(adamw_kernel<N, Moments>, dim3(static_cast<unsigned>(chunks < most ? chunks : most)), AW_THREADS, 0,
                               s, list, used, chunks, mo, k));
  return DGS_OK;
}

template <typename Moments>
int step_all(const char* who, const dgs_adamw_tensor* ts, int32_t count, const Moments& mo, const Scalars& k, cudaStream_t s) {
  DGS_REQUIRE(count >= 0 && (count == 0 || ts != nullptr), DGS_ERR_INVALID, "%s: %d tensors", who, count);
  for (int32_t i = 0; i < count; ++i)
    if (int rc = check_tensor(who, ts[i])) return rc;
  for (int32_t done = 0; done < count;) {
    const int32_t left = count - done;
    const int32_t now = left < AW_LARGE_LIST ? left : AW_LARGE_LIST;
    const int rc = now <= AW_SMALL_LIST ? launch_list<AW_SMALL_LIST>(ts + done, now, mo, k, s)
                                        : launch_list<AW_LARGE_LIST>(ts + done, now, mo, k, s);
    if (rc != DGS_OK) return rc;
    done += now;
  }
  return DGS_OK;
}

}  // namespace
}  // namespace dgs

using namespace dgs;

extern "C" int64_t dgs_adamw_slot_elems(int64_t n) { return n <= 0 ? 0 : (n + AW_BLOCK - 1) / AW_BLOCK * AW_BLOCK; }

extern "C" int dgs_adamw_step(const dgs_adamw_tensor* tensors, int32_t count, float* exp_avg, float* exp_avg_sq, double lr,
                              double beta1, double beta2, double eps, double weight_decay, int64_t step, dgs_stream_t stream) {
  Scalars k;
  if (int rc = make_scalars("adamw_step", lr, beta1, beta2, eps, weight_decay, step, &k)) return rc;
  DGS_REQUIRE(count <= 0 || (exp_avg != nullptr && exp_avg_sq != nullptr && aligned_to(exp_avg, 16) && aligned_to(exp_avg_sq, 16)),
              DGS_ERR_INVALID, "adamw_step: moments that are null or not 16-byte aligned");
  return step_all("adamw_step", tensors, count, Moments32{exp_avg, exp_avg_sq}, k, static_cast<cudaStream_t>(stream));
}

static int step_8bit(const char* who, const dgs_adamw_tensor* tensors, int32_t count, const Moments8& mo, const uint64_t* seed, double lr,
                     double beta1, double beta2, double eps, double weight_decay, int64_t step, dgs_stream_t stream) {
  Scalars k;
  if (int rc = make_scalars(who, lr, beta1, beta2, eps, weight_decay, step, &k)) return rc;
  DGS_REQUIRE(count <= 0 || (mo.m != nullptr && mo.v != nullptr && mo.m_scale != nullptr && mo.v_scale != nullptr && aligned_to(mo.m, 8) &&
                             aligned_to(mo.v, 8)),
              DGS_ERR_INVALID, "%s: moments that are null or not 8-byte aligned", who);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (seed == nullptr) return step_all(who, tensors, count, mo, k, s);
  return step_all(who, tensors, count, Moments8Unbiased{mo, fold_rng_key(*seed, static_cast<uint64_t>(step))}, k, s);
}

extern "C" int dgs_adamw_step_8bit(const dgs_adamw_tensor* tensors, int32_t count, int8_t* exp_avg, float* exp_avg_scale,
                                   uint8_t* exp_avg_sq, float* exp_avg_sq_scale, double lr, double beta1, double beta2,
                                   double eps, double weight_decay, int64_t step, dgs_stream_t stream) {
  return step_8bit("adamw_step_8bit", tensors, count, Moments8{exp_avg, exp_avg_scale, exp_avg_sq, exp_avg_sq_scale}, nullptr, lr, beta1,
                   beta2, eps, weight_decay, step, stream);
}

extern "C" int dgs_adamw_step_8bit_unbiased(const dgs_adamw_tensor* tensors, int32_t count, int8_t* exp_avg, float* exp_avg_scale,
                                            uint8_t* exp_avg_sq, float* exp_avg_sq_scale, double lr, double beta1, double beta2,
                                            double eps, double weight_decay, int64_t step, uint64_t seed, dgs_stream_t stream) {
  return step_8bit("adamw_step_8bit_unbiased", tensors, count, Moments8{exp_avg, exp_avg_scale, exp_avg_sq, exp_avg_sq_scale}, &seed, lr,
                   beta1, beta2, eps, weight_decay, step, stream);
}

extern "C" int dgs_adamw_state_values(const void* codes, int32_t second, const float* scales, int64_t n, float* out,
                                      dgs_stream_t stream) {
  DGS_REQUIRE(n >= 0 && n % AW_BLOCK == 0, DGS_ERR_INVALID, "adamw_state_values: whole blocks of %d codes", AW_BLOCK);
  if (n == 0) return DGS_OK;
  DGS_REQUIRE(codes != nullptr && scales != nullptr && out != nullptr && aligned_to(codes, 8) && aligned_to(out, 16), DGS_ERR_INVALID,
              "adamw_state_values: null or unaligned argument");
  const int64_t words = n / 4, need = (words + AW_THREADS * 4 - 1) / (AW_THREADS * 4), most = static_cast<int64_t>(sm_count()) * 8;
  const dim3 grid(static_cast<unsigned>(need < most ? need : most));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DGS_CUDA_TRY(launch_training(second != 0 ? adamw_values_kernel<true> : adamw_values_kernel<false>, grid, AW_THREADS, 0, s,
                               static_cast<const uint32_t*>(codes), scales, words, reinterpret_cast<float4*>(out)));
  return DGS_OK;
}
