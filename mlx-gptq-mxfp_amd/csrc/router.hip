// The router's choice: the k largest of E logits of each row, ties to the lowest index,
// and their softmax weights, with the gradient of the weights.
//
//   m = max l,  w_j = exp(l_j - m) / Z,  Z = sum of exp(l - m) over the chosen (renorm)
//   or over all experts
//   renorm:  dl_j = w_j (dw_j - sum_i w_i dw_i) for the chosen, 0 for the others
//   else:    dl_e = [e chosen] w_e dw_e - p_e sum_i w_i dw_i,  p = softmax of the row
//
// 16 lanes take a row (a DPP row, so that maxima and sums cross lanes in four
// instructions), a wave four rows. A logit becomes an unsigned key whose order is (logit,
// then lower index first); logits of -infinity (experts that the row may not use) get
// key 0 and are never chosen.
//
// Bound by instructions, not by bytes: 65536 rows of 128 bf16 logits with k = 8 take 14.3 us
// (23 MB) and the gradient 13.0 us (40 MB), 1.6 and 3.1 TB/s. Eight keys of a lane are sorted
// once (16 us where each choice looked through all of them); the gradient's chosen terms
// go to their places through LDS (15.5 us where every lane compared its experts with all k).
// More than 128 experts are looked through for every choice: 65536 rows of 256, 512 and 1024
// take 21, 36 and 86 us in bf16 (renormalized, k = 8) and 38, 84 and 297 in fp32, whose 64-bit
// keys of 1024 experts leave room for one wave a SIMD; the gradient 14, 25 and 49 (21, 32 and 78).
// One row: 2.8 us, a launch.
#include "linear_common.h"

namespace mgq {
namespace {

constexpr int kLanes = 16;
constexpr int kMaxTopK = 16;
constexpr int kMaxExperts = 1024;

struct RouterArgs {
  const char* logits;
  int64_t ld;  // bytes
  int64_t T;
  int E, k;
  int64_t* index;      // [T, k]
  float* weights;      // [T, k]
  const float* dw;     // [T, k]
  char* dlogits;       // [T, E]
};

// v of the lane n above in the row of 16, going round.
template <int N, typename T>
__device__ __forceinline__ T row_ror(T v) {
  if constexpr (sizeof(T) == 8) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = row_ror<N>(static_cast<uint32_t>(u)), hi = row_ror<N>(static_cast<uint32_t>(u >> 32));
    return __builtin_bit_cast(T, static_cast<uint64_t>(hi) << 32 | lo);
  } else {
    return __builtin_bit_cast(
        T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + N, 0xf, 0xf, true));
  }
}
// Lane N of the row, in all of its lanes.
template <int N, typename T>
__device__ __forceinline__ T row_lane(T v) {
  return __builtin_bit_cast(
      T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x150 + N, 0xf, 0xf, true));
}
template <typename T>
__device__ __forceinline__ T row_max(T v) {
  auto up = [](T a, T b) { return a > b ? a : b; };
  v = up(v, row_ror<8>(v));
  v = up(v, row_ror<4>(v));
  v = up(v, row_ror<2>(v));
  return up(v, row_ror<1>(v));
}
__device__ __forceinline__ float row_sum(float v) {
  v += row_ror<8>(v);
  v += row_ror<4>(v);
  v += row_ror<2>(v);
  return v + row_ror<1>(v);
}

// Keys. 16-bit logits: 32 bits, the ordered logit above 0xffff - index; float: 64 bits,
// 0x3ff above the ordered logit above 0xfffff - index, read as a double in [1, 2), whose
// maximum is one instruction (no key is 0 there, so a masked one is 0.0).
template <int TYPE>
struct Key {
  typedef uint32_t type;
  static __device__ __forceinline__ type make(uint32_t bits, int e) {
    const uint32_t inf = TYPE == kF16 ? 0x7c00 : 0x7f80, a = bits & 0x7fff;
    uint32_t s = bits & 0x8000 ? 0xffff - bits : bits | 0x8000;
    s = a == 0 ? 0x8000 : a > inf ? 0xffff : s;  // both zeros alike, no number above all
    return bits == (inf | 0x8000) ? 0 : s << 16 | (0xffff - e);
  }
  static __device__ __forceinline__ int index(type key) { return 0xffff - (key & 0xffff); }
  static __device__ __forceinline__ float value(type key) {
    const uint32_t s = key >> 16, bits = s & 0x8000 ? s & 0x7fff : 0xffff - s;
    return TYPE == kF16 ? f16_to_f32(bits) : bf16_to_f32(bits);
  }
};
template <>
struct Key<kF32> {
  typedef double type;
  static __device__ __forceinline__ type make(uint32_t bits, int e) {
    const uint32_t a = bits & 0x7fffffff;
    uint32_t s = bits & 0x80000000 ? 0xffffffff - bits : bits | 0x80000000;
    s = a == 0 ? 0x80000000 : a > 0x7f800000 ? 0xffffffff : s;
    const uint64_t key = uint64_t(0x3ff) << 52 | static_cast<uint64_t>(s) << 20 | (0xfffff - e);
    return bits == 0xff800000 ? 0.0 : __builtin_bit_cast(double, key);
  }
  static __device__ __forceinline__ uint64_t bits(type key) { return __builtin_bit_cast(uint64_t, key); }
  static __device__ __forceinline__ int index(type key) {
    return 0xfffff - static_cast<int>(bits(key) & 0xfffff);
  }
  static __device__ __forceinline__ float value(type key) {
    const uint32_t s = static_cast<uint32_t>(bits(key) >> 20);
    return u2f(s & 0x80000000 ? s & 0x7fffffff : 0xffffffff - s);
  }
};

template <int TYPE>
__device__ __forceinline__ float as_float(uint32_t bits) {
  return TYPE == kF32 ? u2f(bits) : TYPE == kF16 ? f16_to_f32(bits) : bf16_to_f32(bits);
}
template <int TYPE>
constexpr uint32_t masked_bits() {
  return TYPE == kF32 ? 0xff800000u : TYPE == kF16 ? 0xfc00u : 0xff80u;
}

// Element i of lane `l`: chunks of VEC elements are dealt to the lanes in turn.
template <int VEC>
__device__ __forceinline__ int element(int l, int i) {
  return (i / VEC * kLanes + l) * VEC + i % VEC;
}
template <int TYPE, int VEC, int VPL>
__device__ __forceinline__ void load_row(const char* row, int l, int E, uint32_t (&bits)[VPL]) {
  constexpr int ES = TYPE == kF32 ? 4 : 2;
#pragma unroll
  for (int i = 0; i < VPL; i += VEC) {
    const int e = element<VEC>(l, i);
    if constexpr (VEC == 1) {
      bits[i] = masked_bits<TYPE>();
      if (e < E) bits[i] = ES == 4 ? reinterpret_cast<const uint32_t*>(row)[e]
                                   : reinterpret_cast<const uint16_t*>(row)[e];
    } else {
      lin_u32x4_t v;
      v = e < E ? *reinterpret_cast<const lin_u32x4_t*>(row + e * ES)
                : lin_u32x4_t(masked_bits<TYPE>() * (ES == 4 ? 1u : 0x10001u));
#pragma unroll
      for (int j = 0; j < VEC; ++j) bits[i + j] = ES == 4 ? v[j] : v[j / 2] >> (16 * (j & 1)) & 0xffff;
    }
  }
}

template <int TYPE, int VEC, int VPL, bool RENORM>
__global__ void __launch_bounds__(256) top_k_kernel(const RouterArgs a) {
  typedef Key<TYPE> K;
  const int l = threadIdx.x & (kLanes - 1);
  const int64_t rows = static_cast<int64_t>(gridDim.x) * (256 / kLanes);
  // (whole waves go round: the lanes of rows past the end repeat the last row)
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * (256 / kLanes); r0 < a.T; r0 += rows) {
    const int64_t r = r0 + threadIdx.x / kLanes, t = r < a.T ? r : a.T - 1;
    uint32_t bits[VPL];
    load_row<TYPE, VEC, VPL>(a.logits + t * a.ld, l, a.E, bits);
    typename K::type key[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) key[i] = K::make(bits[i], element<VEC>(l, i));
    // Eight keys of a lane in descending order: its largest is then in its first register,
    // and a choice that was this lane's moves the others up.
    constexpr bool SORTED = VPL <= 8;
    if constexpr (SORTED) {
      static_assert(VPL == 8, "network of eight");
      auto order = [&](int i, int j) {
        const typename K::type x = key[i], y = key[j];
        key[i] = x > y ? x : y;
        key[j] = x > y ? y : x;
      };
      // Batcher's odd-even merge of eight
      order(0, 1); order(2, 3); order(4, 5); order(6, 7);
      order(0, 2); order(1, 3); order(4, 6); order(5, 7);
      order(1, 2); order(5, 6);
      order(0, 4); order(1, 5); order(2, 6); order(3, 7);
      order(2, 4); order(3, 5);
      order(1, 2); order(3, 4); order(5, 6);
    }
    typename K::type mine = 0;  // lane j keeps choice j
    float m = 0, z = 0;
    for (int j = 0; j < a.k; ++j) {
      typename K::type best = key[0];
      if constexpr (!SORTED) {
#pragma unroll
        for (int i = 1; i < VPL; ++i) best = key[i] > best ? key[i] : best;
      }
      best = row_max(best);
      if (j == 0) {
        m = best > 0 ? K::value(best) : 0.0f;
        if constexpr (!RENORM) {
#pragma unroll
          for (int i = 0; i < VPL; ++i) z += expf(as_float<TYPE>(bits[i]) - m);
        }
      }
      if (l == j) mine = best;
      if constexpr (SORTED) {
        const bool own = key[0] == best;
#pragma unroll
        for (int i = 0; i + 1 < VPL; ++i) key[i] = own ? key[i + 1] : key[i];
        key[VPL - 1] = own ? 0 : key[VPL - 1];
      } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i) key[i] = key[i] == best ? 0 : key[i];
      }
    }
    const bool some = mine > 0;
    const float w = some ? expf(K::value(mine) - m) : 0.0f;
    z = row_sum(RENORM ? w : z);
    if (r < a.T && l < a.k) {
      a.index[t * a.k + l] = some ? K::index(mine) : -1;
      a.weights[t * a.k + l] = some ? w / z : 0.0f;
    }
  }
}

template <int TYPE, int VEC, int VPL, bool RENORM>
__global__ void __launch_bounds__(256) top_k_grad_kernel(const RouterArgs a) {
  constexpr int ES = TYPE == kF32 ? 4 : 2;
  // What the chosen experts get, at its place of the row: each row its own part, written
  // and read by the 16 lanes that share it (one wave). Short rows only.
  constexpr bool PLACED = VPL <= 16;
  constexpr int PITCH = VPL * kLanes + 4;  // (the four rows of a wave start in other banks)
  __shared__ __attribute__((aligned(16))) float placed[PLACED ? 256 / kLanes * PITCH : 4];
  float* const place = placed + (PLACED ? threadIdx.x / kLanes * PITCH : 0);
  const int l = threadIdx.x & (kLanes - 1);
  const int64_t rows = static_cast<int64_t>(gridDim.x) * (256 / kLanes);
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * (256 / kLanes); r0 < a.T; r0 += rows) {
    const int64_t r = r0 + threadIdx.x / kLanes, t = r < a.T ? r : a.T - 1;
    const char* row = a.logits + t * a.ld;
    // lane j: choice j
    int chosen = -1;
    float dw = 0, logit = -INFINITY;
    if (l < a.k) {
      const int64_t e = a.index[t * a.k + l];
      chosen = e >= 0 && e < a.E ? static_cast<int>(e) : -1;
      dw = a.dw[t * a.k + l];
    }
    if (chosen >= 0)
      logit = as_float<TYPE>(ES == 4 ? reinterpret_cast<const uint32_t*>(row)[chosen]
                                     : reinterpret_cast<const uint16_t*>(row)[chosen]);
    float p[VPL];
    float m, z = 0;
    auto top = [](float x, float y) { return x > y ? x : y; };  // (a NaN shows in z)
    if constexpr (RENORM) {
      m = row_max(logit);
      m = m > -INFINITY ? m : 0.0f;
    } else {
      uint32_t bits[VPL];
      load_row<TYPE, VEC, VPL>(row, l, a.E, bits);
      float mine = -INFINITY;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        p[i] = as_float<TYPE>(bits[i]);
        mine = top(p[i], mine);
      }
      m = row_max(mine);
      m = m > -INFINITY ? m : 0.0f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        p[i] = expf(p[i] - m);
        z += p[i];
      }
    }
    float w = chosen >= 0 ? expf(logit - m) : 0.0f;
    z = row_sum(RENORM ? w : z);
    w = chosen >= 0 && z != 0.0f ? w / z : 0.0f;  // (a row without experts)
    const float wd = w != 0.0f ? w * dw : 0.0f;
    const float dot = row_sum(wd);
    const float add = !RENORM ? wd : w != 0.0f ? w * (dw - dot) : 0.0f;
    const float scale = RENORM || z == 0.0f ? 0.0f : -dot / z;
#pragma unroll
    for (int i = 0; i < VPL; ++i) p[i] = RENORM || z == 0.0f ? 0.0f : p[i] * scale;
    // An index that stands twice in a row gets the sum, in the order of the row.
    bool again = false;
    float sum = add;
    static_for<kMaxTopK>([&](auto j) {
      if (j < a.k) {
        const int e = row_lane<j>(chosen);
        const float v = row_lane<j>(add);
        if constexpr (PLACED) {
          if (e == chosen && j != l) {
            again |= j < l;
            sum += v;
          }
        } else {
#pragma unroll
          for (int i = 0; i < VPL; ++i) p[i] += element<VEC>(l, i) == e ? v : 0.0f;
        }
      }
    });
    if constexpr (PLACED) {
      // (LDS serves a wave in order; the fences keep the compiler to that)
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < VPL; i += 4) *reinterpret_cast<float4*>(place + 4 * l + 64 * (i / 4)) = float4{0, 0, 0, 0};
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (chosen >= 0 && !again) place[chosen] = sum;
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int i = 0; i < VPL; i += VEC) {
        const int e = element<VEC>(l, i);
#pragma unroll
        for (int j = 0; j < VEC; ++j) p[i + j] += place[e + j];
      }
      __builtin_amdgcn_wave_barrier();
    }
    if (r >= a.T) continue;
    char* out = a.dlogits + t * a.E * ES;
#pragma unroll
    for (int i = 0; i < VPL; i += VEC) {
      const int e = element<VEC>(l, i);
      if (e >= a.E) continue;
      if constexpr (VEC == 1) {
        if constexpr (ES == 4)
          reinterpret_cast<float*>(out)[e] = p[i];
        else
          reinterpret_cast<uint16_t*>(out)[e] = lin_round16(p[i], TYPE);
      } else {
        lin_u32x4_t v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (ES == 4)
            v[j] = f2u(p[i + j]);
          else
            v[j] = lin_pack2<TYPE>(p[i + 2 * j], p[i + 2 * j + 1]);
        }
        *reinterpret_cast<lin_u32x4_t*>(out + e * ES) = v;
      }
    }
  }
}

template <int TYPE, int VEC, int VPL>
int launch(const RouterArgs& a, bool renorm, bool grad, hipStream_t s, const char* what) {
  const int64_t blocks = ceil_div(a.T, 256 / kLanes);
  const unsigned grid = static_cast<unsigned>(blocks < (1 << 20) ? blocks : 1 << 20);
  if (grad) {
    if (renorm) top_k_grad_kernel<TYPE, VEC, VPL, true><<<grid, 256, 0, s>>>(a);
    else top_k_grad_kernel<TYPE, VEC, VPL, false><<<grid, 256, 0, s>>>(a);
  } else {
    if (renorm) top_k_kernel<TYPE, VEC, VPL, true><<<grid, 256, 0, s>>>(a);
    else top_k_kernel<TYPE, VEC, VPL, false><<<grid, 256, 0, s>>>(a);
  }
  return check_launch(what);
}
template <int TYPE, int VEC>
int sized(const RouterArgs& a, bool renorm, bool grad, hipStream_t s, const char* what) {
  if (a.E <= 128) return launch<TYPE, VEC, 8>(a, renorm, grad, s, what);
  if (a.E <= 256) return launch<TYPE, VEC, 16>(a, renorm, grad, s, what);
  if (a.E <= 512) return launch<TYPE, VEC, 32>(a, renorm, grad, s, what);
  return launch<TYPE, VEC, 64>(a, renorm, grad, s, what);
}
// Rows in 16-byte pieces where all of them start and end on such boundaries.
template <int TYPE>
int typed(const RouterArgs& a, bool renorm, bool grad, hipStream_t s, const char* what) {
  constexpr int ES = TYPE == kF32 ? 4 : 2;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.dlogits) |
                       static_cast<uintptr_t>(a.ld | static_cast<int64_t>(a.E) * ES);
  return at & 15 ? sized<TYPE, 1>(a, renorm, grad, s, what)
                 : sized<TYPE, 16 / ES>(a, renorm, grad, s, what);
}
int run(const RouterArgs& a, int dtype, bool renorm, bool grad, hipStream_t s, const char* what) {
  if (dtype == kF32) return typed<kF32>(a, renorm, grad, s, what);
  if (dtype == kF16) return typed<kF16>(a, renorm, grad, s, what);
  return typed<kBF16>(a, renorm, grad, s, what);
}

int check(const char* what, int dtype, int64_t T, int64_t E, int64_t ld, int64_t k) {
  MGQ_REQUIRE(dtype == kF32 || dtype == kBF16 || dtype == kF16, MGQ_ERR_VALUE,
              "%s: float32, bfloat16 or float16 logits only", what);
  MGQ_REQUIRE(T >= 0 && E >= 1 && E <= kMaxExperts, MGQ_ERR_SHAPE, "%s: %lld rows of %lld logits (1 .. %d)",
              what, (long long)T, (long long)E, kMaxExperts);
  MGQ_REQUIRE(ld >= E, MGQ_ERR_SHAPE, "%s: a row pitch is shorter than a row", what);
  MGQ_REQUIRE(k >= 1 && k <= kMaxTopK && k <= E, MGQ_ERR_SHAPE, "%s: %lld of %lld experts (1 .. %d)", what,
              (long long)k, (long long)E, kMaxTopK);
  return MGQ_OK;
}

}  // namespace
}  // namespace mgq

using namespace mgq;

extern "C" int mgq_top_k_softmax(const void* logits, int dtype, int64_t T, int64_t E, int64_t ld,
                                 int64_t k, int renormalize, int64_t* index, float* weights,
                                 void* stream) {
  clear_error();
  const char* what = "top_k_softmax";
  if (int rc = check(what, dtype, T, E, ld, k)) return rc;
  if (T == 0) return MGQ_OK;
  RouterArgs a = {};
  a.logits = static_cast<const char*>(logits);
  a.ld = ld * (dtype == kF32 ? 4 : 2);
  a.T = T;
  a.E = static_cast<int>(E);
  a.k = static_cast<int>(k);
  a.index = index;
  a.weights = weights;
  return run(a, dtype, renormalize != 0, false, as_stream(stream), what);
}

extern "C" int mgq_top_k_softmax_grad(const float* dw, const void* logits, int dtype, int64_t T,
                                      int64_t E, int64_t ld, const int64_t* index, int64_t k,
                                      int renormalize, void* dlogits, void* stream) {
  clear_error();
  const char* what = "top_k_softmax_grad";
  if (int rc = check(what, dtype, T, E, ld, k)) return rc;
  if (T == 0) return MGQ_OK;
  RouterArgs a = {};
  a.logits = static_cast<const char*>(logits);
  a.ld = ld * (dtype == kF32 ? 4 : 2);
  a.T = T;
  a.E = static_cast<int>(E);
  a.k = static_cast<int>(k);
  a.index = const_cast<int64_t*>(index);
  a.dw = dw;
  a.dlogits = static_cast<char*>(dlogits);
  return run(a, dtype, renormalize != 0, true, as_stream(stream), what);
}
