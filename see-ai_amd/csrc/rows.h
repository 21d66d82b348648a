// rows.h -- rows of f32 or bf16 held in registers, a row over kTPR threads of a
// workgroup: loads, stores and sums, for the norms (k_norm.hip) and what stands
// between two blocks (k_join.hip).
#pragma once

#include "common.h"

namespace seeai {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Sixteen bytes on a float's or a bf16's own alignment: global memory takes them.
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4), may_alias));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2), may_alias));

template <class T> struct Io;
template <> struct Io<float> {
  static constexpr int kV = 4;  // elements of a 16-byte access
  static __device__ __forceinline__ void Load(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  }
  static __device__ __forceinline__ void Store(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
  static __device__ __forceinline__ void LoadAny(const float* p, float* v) {
    const f32x4u a = *reinterpret_cast<const f32x4u*>(p);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  }
  static __device__ __forceinline__ void StoreAny(float* p, const float* v) {
    *reinterpret_cast<f32x4u*>(p) = f32x4u{v[0], v[1], v[2], v[3]};
  }
  static __device__ __forceinline__ float Get(const float* p) { return *p; }
  static __device__ __forceinline__ void Put(float* p, float v) { *p = v; }
};
template <> struct Io<uint16_t> {  // bf16
  static constexpr int kV = 8;
  static __device__ __forceinline__ void Load(const uint16_t* p, float* v) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ bf16x8 Pack(const float* v) {
    bf16x8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = static_cast<__bf16>(v[i]);
    return o;
  }
  static __device__ __forceinline__ void Store(uint16_t* p, const float* v) {
    *reinterpret_cast<bf16x8*>(p) = Pack(v);
  }
  static __device__ __forceinline__ void LoadAny(const uint16_t* p, float* v) {
    const u32x4u a = *reinterpret_cast<const u32x4u*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ void StoreAny(uint16_t* p, const float* v) {
    *reinterpret_cast<u32x4u*>(p) = __builtin_bit_cast(u32x4u, Pack(v));
  }
  static __device__ __forceinline__ float Get(const uint16_t* p) { return Bf16ToF32(*p); }
  static __device__ __forceinline__ void Put(uint16_t* p, float v) { *p = F32ToBf16(v); }
};

// Where lane t's element e of a row lies, and whether it lies in the row.
// kVec: groups of kV neighbours, kTPR groups apart (16-byte accesses, rows a
// multiple of kV long); else single elements kTPR apart.  kAny, with kVec: the
// same groups where rows are of any length and begin anywhere, the row's last,
// short group element by element.
template <class T, int kTPR, bool kVec>
__device__ __forceinline__ int ColOf(int t, int e) {
  constexpr int kV = Io<T>::kV;
  return kVec ? ((e / kV) * kTPR + t) * kV + e % kV : e * kTPR + t;
}
template <class T, int kTPR, int kE, bool kVec, bool kAny = false>
__device__ __forceinline__ void LoadRow(const T* row, int t, int cols, float (&v)[kE]) {
  constexpr int kV = Io<T>::kV;
  if constexpr (kAny) {
#pragma unroll
    for (int e = 0; e < kE; e += kV) {
      const int c = ColOf<T, kTPR, true>(t, e);
      if (c + kV <= cols) {
        Io<T>::LoadAny(row + c, v + e);
      } else {
#pragma unroll
        for (int i = 0; i < kV; ++i) v[e + i] = c + i < cols ? Io<T>::Get(row + c + i) : 0.0f;
      }
    }
  } else if constexpr (kVec) {
#pragma unroll
    for (int e = 0; e < kE; e += kV) {
      const int c = ColOf<T, kTPR, true>(t, e);
      if (c < cols) {
        Io<T>::Load(row + c, v + e);
      } else {
#pragma unroll
        for (int i = 0; i < kV; ++i) v[e + i] = 0.0f;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const int c = ColOf<T, kTPR, false>(t, e);
      v[e] = c < cols ? Io<T>::Get(row + c) : 0.0f;
    }
  }
}
template <class T, int kTPR, int kE, bool kVec, bool kAny = false>
__device__ __forceinline__ void StoreRow(T* row, int t, int cols, const float (&v)[kE]) {
  constexpr int kV = Io<T>::kV;
  if constexpr (kAny) {
#pragma unroll
    for (int e = 0; e < kE; e += kV) {
      const int c = ColOf<T, kTPR, true>(t, e);
      if (c + kV <= cols) {
        Io<T>::StoreAny(row + c, v + e);
      } else {
#pragma unroll
        for (int i = 0; i < kV; ++i)
          if (c + i < cols) Io<T>::Put(row + c + i, v[e + i]);
      }
    }
  } else if constexpr (kVec) {
#pragma unroll
    for (int e = 0; e < kE; e += kV) {
      const int c = ColOf<T, kTPR, true>(t, e);
      if (c < cols) Io<T>::Store(row + c, v + e);
    }
  } else {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const int c = ColOf<T, kTPR, false>(t, e);
      if (c < cols) Io<T>::Put(row + c, v[e]);
    }
  }
}
// The f32 vector at the same columns.
template <class T, int kTPR, int kE, bool kVec, bool kAny = false>
__device__ __forceinline__ void LoadVec(const float* w, int t, int cols, float (&v)[kE]) {
  if constexpr (kAny) {
#pragma unroll
    for (int e = 0; e < kE; e += 4) {
      const int c = ColOf<T, kTPR, true>(t, e);
      if (c + 4 <= cols) {
        Io<float>::LoadAny(w + c, v + e);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[e + i] = c + i < cols ? w[c + i] : 0.0f;
      }
    }
  } else if constexpr (kVec) {
#pragma unroll
    for (int e = 0; e < kE; e += 4) {
      const int c = ColOf<T, kTPR, true>(t, e);
      if (c < cols) {
        Io<float>::Load(w + c, v + e);
      } else {
        v[e] = v[e + 1] = v[e + 2] = v[e + 3] = 0.0f;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      const int c = ColOf<T, kTPR, false>(t, e);
      v[e] = c < cols ? w[c] : 0.0f;
    }
  }
}

// Sums and maxima by lane moves within registers: MoveAdd adds what the DPP
// control brings (0 where it brings nothing).
template <int kCtrl, int kRows = 0xf>
__device__ __forceinline__ float MoveAdd(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, kRows, 0xf, false));
}
template <int kCtrl, int kRows = 0xf>
__device__ __forceinline__ float MoveMax(float v) {
  const int i = __float_as_int(v);
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(i, i, kCtrl, kRows, 0xf, false)));
}
__device__ __forceinline__ float Lane63(float v) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
// Over the wave; every lane gets it.
__device__ __forceinline__ float LanesSum(float v) {
  v = MoveAdd<0x111>(v);  // from 1, 2, 4, 8 lanes before, within rows of 16
  v = MoveAdd<0x112>(v);
  v = MoveAdd<0x114>(v);
  v = MoveAdd<0x118>(v);
  v = MoveAdd<0x142, 0xa>(v);  // lane 15 of a row to the next row
  return Lane63(MoveAdd<0x143, 0xc>(v));  // lane 31 to the upper half
}
template <int kCtrl, int kRows = 0xf>
__device__ __forceinline__ double MoveAddD(double v) {
  const int lo = __double2loint(v), hi = __double2hiint(v);
  return v + __hiloint2double(__builtin_amdgcn_update_dpp(0, hi, kCtrl, kRows, 0xf, false),
                              __builtin_amdgcn_update_dpp(0, lo, kCtrl, kRows, 0xf, false));
}
__device__ __forceinline__ double LanesSumD(double v) {
  v = MoveAddD<0x111>(v);
  v = MoveAddD<0x112>(v);
  v = MoveAddD<0x114>(v);
  v = MoveAddD<0x118>(v);
  v = MoveAddD<0x142, 0xa>(v);
  v = MoveAddD<0x143, 0xc>(v);
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), 63),
                          __builtin_amdgcn_readlane(__double2loint(v), 63));
}
__device__ __forceinline__ float LanesMax(float v) {  // (a NaN is passed over)
  v = MoveMax<0x111>(v);
  v = MoveMax<0x112>(v);
  v = MoveMax<0x114>(v);
  v = MoveMax<0x118>(v);
  v = MoveMax<0x142, 0xa>(v);
  return Lane63(MoveMax<0x143, 0xc>(v));
}

// Sums over the kTPR threads of each row of a workgroup: within the wave, then
// over a row's waves through LDS (two floats a wave).
template <int kTPR, int kN>
__device__ __forceinline__ void RowSum(float (&s)[kN], float* lds) {
#pragma unroll
  for (int i = 0; i < kN; ++i) s[i] = WaveSumF(s[i]);
  if constexpr (kTPR > kWave) {
    constexpr int kWaves = kTPR / kWave;
    const int w = threadIdx.x / kWave, first = w / kWaves * kWaves;
    __syncthreads();  // the sums before these have been read
    if (threadIdx.x % kWave == 0)
#pragma unroll
      for (int i = 0; i < kN; ++i) lds[w * kN + i] = s[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      s[i] = 0.0f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) s[i] += lds[(first + k) * kN + i];
    }
  }
}

// A row as it lies in memory, for loads that run ahead of their use.
template <class T, int kTPR, int kE, bool kVec>
struct RawRow {
  static constexpr int kV = Io<T>::kV;
  uint4 q[kVec ? kE / kV : 1];
  T e[kVec ? 1 : kE];
  __device__ __forceinline__ void Load(const T* row, int t, int cols) {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kE / kV; ++i) {
        const int c = ColOf<T, kTPR, true>(t, i * kV);
        q[i] = c < cols ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) {
        const int c = ColOf<T, kTPR, false>(t, i);
        e[i] = c < cols ? row[c] : T(0);
      }
    }
  }
  __device__ __forceinline__ void Get(float (&v)[kE]) const {
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kE / kV; ++i) Io<T>::Load(reinterpret_cast<const T*>(&q[i]), v + i * kV);
    } else {
#pragma unroll
      for (int i = 0; i < kE; ++i) v[i] = Io<T>::Get(&e[i]);
    }
  }
};

}  // namespace seeai
