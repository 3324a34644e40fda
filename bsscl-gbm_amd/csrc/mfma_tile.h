// Tiles of C(m, n) = sum_k A(m, k) B(n, k) on the matrix cores of gfx950, for
// bf16, fp16 and float32 operands with float32 sums.
//
// A workgroup holds a BM x BN tile in registers, WM x WN per wave in blocks of
// 32 x 32 (v_mfma 32x32x16, for float32 32x32x2), and walks k in steps.  Both
// operands' steps go from memory straight to LDS (buffer loads with the lds
// bit: no registers), into a ring of buffers.  An operand lies in memory with
// k contiguous (rows of m or n) or with m or n contiguous (rows of k):
//   k contiguous   LDS rows of one step's bytes; a lane reads 16 bytes of a row
//   k across rows  LDS rows of the tile's m (n) range; 16-bit fragments come
//                  from transposing reads (ds_read_b64_tr_b16: a group of 16
//                  lanes reads 4 k x 16 m and gets k in registers), and chunk
//                  c of row k lies in place c ^ 4 (k & 3), so that the four
//                  rows of a group touch different banks
// An LDS place is lane-linear in the load, so the swizzles permute the lanes'
// addresses in memory.  Reads outside the operand return 0 (the buffer
// descriptor's bound), so edges need no other care: offsets of lanes that
// are not to read are 2^31, beyond every bound.
//
// Fragment of the 32x32 blocks, lane l: row (column) l % 32 and 16 bytes of k
// from 16 (l / 32) on; result register r: m = 8 (r / 4) + 4 (l / 32) + r % 4,
// n = l % 32.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

namespace bsscl {

typedef int Int4 __attribute__((ext_vector_type(4)));
typedef float Acc16 __attribute__((ext_vector_type(16)));
typedef __bf16 Bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 F16x8 __attribute__((ext_vector_type(8)));
typedef short Short4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kNoRead = 0x80000000u;  // a lane's offset beyond every bound

// acc += a b over one 16-byte fragment of k.
template <typename T>
__device__ __forceinline__ Acc16 mma(Int4 a, Int4 b, Acc16 acc) {
  if constexpr (std::is_same<T, __bf16>::value) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Bf16x8, a),
                                                   __builtin_bit_cast(Bf16x8, b), acc, 0, 0, 0);
  } else if constexpr (std::is_same<T, _Float16>::value) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(F16x8, a),
                                                  __builtin_bit_cast(F16x8, b), acc, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(float, (int)a[j]),
                                                 __builtin_bit_cast(float, (int)b[j]), acc, 0, 0,
                                                 0);
    return acc;
  }
}

// 16 bytes per lane from memory to LDS at lds_at + 16 lane.  In assembly
// because the compiler would wait for it before every transposing read; the
// walk below waits itself.
__device__ __forceinline__ void load_to_lds(Int4 rsrc, uint32_t offset, uint32_t lds_at) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds_at), "v"(offset), "s"(rsrc)
               : "memory");
}

__device__ __forceinline__ Int4 buffer_of(const char *base, uint32_t bytes) {
  const uint64_t a = (uint64_t)(uintptr_t)base;
  return Int4{(int)(uint32_t)a, (int)(uint32_t)(a >> 32), (int)bytes, 0x00020000};
}

// One operand of a tile: MN rows (columns) of C, `across`: k across rows;
// STEP: bytes of k in one step.
template <typename T, int MN, bool ACROSS, int WAVES, int STEP>
struct Operand {
  static constexpr int kES = (int)sizeof(T);
  static constexpr int kStep = STEP / kES;  // k of one step
  static constexpr int kBytes = MN * STEP;  // LDS of one step
  static constexpr int kRowBytes = ACROSS ? MN * kES : STEP;
  static constexpr int kChunks = kRowBytes / 16;  // of an LDS row
  static constexpr int kRowsPerLoad = 64 / kChunks;
  static constexpr int kLoads = kBytes / 1024 / WAVES;  // of each wave in a step
  static_assert(kLoads >= 1 && kLoads * 1024 * WAVES == kBytes && kChunks <= 64, "tile shape");

  // The place of chunk c of LDS row r.  Sixteen lanes read 16 bytes each in one
  // go: with k contiguous, of one chunk of 16 rows, which lie in all 16
  // chunks of a bank line (256 bytes: kPerLine rows).
  static constexpr int kPerLine = 256 / kRowBytes > 0 ? 256 / kRowBytes : 1;
  __device__ static __forceinline__ int place_of(int c, int r) {
    if constexpr (!ACROSS) return c ^ ((r / kPerLine) & (kChunks - 1));
    else if constexpr (kES == 2) return c ^ (((r & 3) * 4) & (kChunks - 1));
    else return c;
  }

  const char *base;
  int64_t stride;  // bytes from row to row
  int32_t valid;   // rows (k contiguous) or values of a row (across) inside
  uint32_t offset[kLoads];
  uint32_t chunk;  // the lane's chunk in memory

  // first: the tile's first m (n) in the operand; limit: their number.
  __device__ __forceinline__ void init(const T *p, int64_t row_stride, int32_t first,
                                       int32_t limit) {
    stride = row_stride * kES;
    valid = min(limit - first, MN);
    base = reinterpret_cast<const char *>(p) +
           (ACROSS ? (int64_t)first * kES : (int64_t)first * stride);
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = (i * WAVES + wave) * kRowsPerLoad + lane / kChunks;
      const int place = lane % kChunks;
      chunk = (uint32_t)place_of(place, row);  // its own inverse
      if constexpr (!ACROSS) {
        offset[i] = (uint32_t)(row * stride) + chunk * 16;
      } else {
        offset[i] = (int)(chunk * (16 / kES)) < valid ? (uint32_t)(row * stride) + chunk * 16
                                                      : kNoRead;
      }
    }
  }

  // The step that begins at k of k_end, into LDS at lds_at: its buffer
  // descriptor, and the wave's loads one by one.
  struct Step {
    Int4 rsrc;
    uint32_t at;
    int32_t bytes;
  };
  __device__ __forceinline__ Step step(int64_t k, int64_t k_end, uint32_t lds_at) const {
    const int64_t left = k_end - k;
    Step s;
    s.at = lds_at + ((uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) << 10);
    if constexpr (!ACROSS) {
      // (Rows are padded to whole chunks.)
      s.bytes = (int32_t)min((left * kES + 15) & ~int64_t(15), (int64_t)STEP);
      s.rsrc = buffer_of(base + k * kES,
                         valid > 0 ? (uint32_t)((valid - 1) * stride) + (uint32_t)s.bytes : 0);
    } else {
      const int32_t rows = (int32_t)min(left, (int64_t)kStep);
      s.bytes = STEP;
      s.rsrc = buffer_of(base + k * stride, valid > 0 ? (uint32_t)((rows - 1) * stride) +
                                                            (uint32_t)(valid * kES)
                                                      : 0);
    }
    return s;
  }
  __device__ __forceinline__ void load(const Step &s, int i) const {
    const bool in = ACROSS || (int)(chunk * 16) < s.bytes;
    load_to_lds(s.rsrc, in ? offset[i] : kNoRead, s.at + (uint32_t)(i * WAVES * 1024));
  }

  // The fragment of k part `part` (of STEP / 32) and the 32 rows from `first` on.
  __device__ static __forceinline__ Int4 fragment(const char *lds, int first, int part) {
    const int l = (int)threadIdx.x & 63;
    if constexpr (!ACROSS) {
      return *reinterpret_cast<const Int4 *>(lds + (first + (l & 31)) * STEP +
                                             (place_of(part * 2 + (l >> 5), l & 31) << 4));
    } else if constexpr (kES == 2) {
      const int k = part * 16 + (l >> 5) * 8 + ((l & 15) >> 2);
      const int m = first + ((l >> 4) & 1) * 16 + (l & 3) * 4;
      const int c = place_of(m >> 3, k);
      const char *p = lds + k * kRowBytes + (c << 4) + (m & 4) * 2;
      typedef __attribute__((address_space(3))) Short4 *LdsShort4;
      const Short4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4)(p));
      const Short4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4)(p + 4 * kRowBytes));
      typedef short Short8 __attribute__((ext_vector_type(8)));
      return __builtin_bit_cast(Int4, (Short8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const char *p = lds + (part * 8 + (l >> 5) * 4) * kRowBytes + (first + (l & 31)) * 4;
      Int4 f;
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = *reinterpret_cast<const int *>(p + j * kRowBytes);
      return f;
    }
  }
};

template <int VM>
__device__ __forceinline__ void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(VM) : "memory");
}

// A tile's shape: BM x BN per workgroup, WM x WN per wave; STEP bytes of k at
// a time, STAGES (at least 3) of them in LDS.
template <typename T_, int BM_, int BN_, int WM_, int WN_, bool A_ACROSS, bool B_ACROSS, int STEP,
          int STAGES>
struct Tile {
  using T = T_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kWavesM = BM / WM, kWavesN = BN / WN, kWaves = kWavesM * kWavesN;
  static constexpr int kThreads = kWaves * 64;
  static constexpr int MI = WM / 32, NI = WN / 32;
  using A = Operand<T, BM, A_ACROSS, kWaves, STEP>;
  using B = Operand<T, BN, B_ACROSS, kWaves, STEP>;
  static constexpr int kStep = A::kStep, kParts = STEP / 32;
  static constexpr int kStage = A::kBytes + B::kBytes;
  static constexpr int kLds = STAGES * kStage;
  static_assert(kLds <= 160 * 1024 && STAGES >= 3 && kParts % 2 == 0, "tile shape");

  // acc[mi][ni] += products of k in [k_begin, k_end); k_begin is a multiple of
  // kStep.  Every thread of the workgroup calls it; LDS is free at its end.
  //
  // Step k is read while those up to k + STAGES - 1 load.  Fragments are read
  // one part ahead of the products that use them, the first part of a step
  // during the last products of the step before: there stands the step's one
  // barrier, when every wave has read the last of its buffer and the next
  // step's loads have landed.  Reads and loads are dealt out among the
  // products (A's loads to the first part, B's to the last), so that no more
  // than a few are issued between two of them: the matrix cores multiply on
  // meanwhile.
  __device__ static __forceinline__ void walk(const A &a, const B &b, int64_t k_begin,
                                              int64_t k_end, char *lds, Acc16 (&acc)[MI][NI]) {
    const int wave = (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / kWavesN * WM, wn = wave % kWavesN * WN;
    const uint32_t lds_at =
        (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    constexpr int kReads = MI + NI;
    Int4 fa[2][MI], fb[2][NI];
    auto read = [&](const char *cur, int part, int set, int i) {
      if (i < NI)
        fb[set][i] = B::fragment(cur + A::kBytes, wn + i * 32, part);
      else
        fa[set][i - NI] = A::fragment(cur, wm + (i - NI) * 32, part);
    };
    for (int s = 0; s < STAGES - 1; ++s) {
      const int64_t k = k_begin + s * kStep;
      if (k >= k_end) break;
      const auto sa = a.step(k, k_end, lds_at + (uint32_t)(s * kStage));
      const auto sb = b.step(k, k_end, lds_at + (uint32_t)(s * kStage + A::kBytes));
#pragma unroll
      for (int i = 0; i < A::kLoads; ++i) a.load(sa, i);
#pragma unroll
      for (int i = 0; i < B::kLoads; ++i) b.load(sb, i);
    }
    wait_and_meet<0>();
#pragma unroll
    for (int i = 0; i < kReads; ++i) read(lds, 0, 0, i);
    int buf = 0;
    // MORE: there is a step to load.
    auto one_step = [&](int64_t k, auto more) {
      constexpr bool MORE = decltype(more)::value;
      const int next = buf + 1 == STAGES ? 0 : buf + 1;
      const char *cur = lds + buf * kStage, *then = lds + next * kStage;
      typename A::Step sa;
      typename B::Step sb;
      if constexpr (MORE) {
        const uint32_t at = lds_at + (uint32_t)((buf == 0 ? STAGES - 1 : buf - 1) * kStage);
        sa = a.step(k + (STAGES - 1) * kStep, k_end, at);
        sb = b.step(k + (STAGES - 1) * kStep, k_end, at + A::kBytes);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        const int set = part & 1;
        if (part == kParts - 1)
          wait_and_meet<MORE ? (STAGES - 3) * (A::kLoads + B::kLoads) + A::kLoads : 0>();
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          if constexpr (MORE) {
            if (part == 0)
#pragma unroll
              for (int e = i * A::kLoads / MI; e < (i + 1) * A::kLoads / MI; ++e) a.load(sa, e);
            if (part == kParts - 1)
#pragma unroll
              for (int e = i * B::kLoads / MI; e < (i + 1) * B::kLoads / MI; ++e) b.load(sb, e);
          }
#pragma unroll
          for (int e = i * kReads / MI; e < (i + 1) * kReads / MI; ++e)
            read(part < kParts - 1 ? cur : then, part < kParts - 1 ? part + 1 : 0, set ^ 1, e);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < NI; ++j) acc[i][j] = mma<T>(fa[set][i], fb[set][j], acc[i][j]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      buf = next;
    };
    int64_t k = k_begin;
    for (; k + (STAGES - 1) * kStep < k_end; k += kStep) one_step(k, std::true_type());
    for (; k < k_end; k += kStep) one_step(k, std::false_type());
    wait_and_meet<0>();
  }

  // The tile as rows of n (row n: BM values of m) in LDS, chunk c of row n in
  // place c ^ (n mod chunks): value(i, j, r) gives lane values as T.
  static constexpr int kOutRow = BM * (int)sizeof(T), kOutChunks = kOutRow / 16;
  static constexpr int kLdsOut = kLds > BN * kOutRow ? kLds : BN * kOutRow;
  template <typename F>
  __device__ static __forceinline__ void stage_out(char *lds, F &&value) {
    static_assert(kLdsOut <= 160 * 1024, "the tile fits LDS");
    const int wave = (int)threadIdx.x >> 6, l = (int)threadIdx.x & 63;
    const int wm = wave / kWavesN * WM, wn = wave % kWavesN * WN;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = wn + j * 32 + (l & 31), m = wm + i * 32 + q * 8 + (l >> 5) * 4;
          typedef T T4 __attribute__((ext_vector_type(4)));
          T4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = value(i, j, q * 4 + e);
          const int at = m * (int)sizeof(T), c = (at >> 4) ^ (n & (kOutChunks - 1));
          *reinterpret_cast<T4 *>(lds + n * kOutRow + (c << 4) + (at & 15)) = v;
        }
  }
  // Calls f(n, m, the 16 bytes of T at m ..) for the chunks of this thread.
  template <typename F>
  __device__ static __forceinline__ void read_out(const char *lds, F &&f) {
    for (int e = (int)threadIdx.x; e < BN * kOutChunks; e += kThreads) {
      const int n = e / kOutChunks, c = e % kOutChunks;
      f(n, c * (16 / (int)sizeof(T)),
        *reinterpret_cast<const Int4 *>(lds + n * kOutRow +
                                        ((c ^ (n & (kOutChunks - 1))) << 4)));
    }
  }
  // f(n, m, value) for the values of this thread, neighbours side by side.
  template <typename F>
  __device__ static __forceinline__ void read_out_one(const char *lds, F &&f) {
    for (int e = (int)threadIdx.x; e < BN * BM; e += kThreads) {
      const int n = e / BM, m = e % BM, at = m * (int)sizeof(T);
      const int c = (at >> 4) ^ (n & (kOutChunks - 1));
      f(n, m, *reinterpret_cast<const T *>(lds + n * kOutRow + (c << 4) + (at & 15)));
    }
  }
};

// Workgroup b of `count` in an order that gives each of the 8 XCDs (which take
// workgroups in turn) one contiguous part: its L2 then serves neighbours.
__device__ __forceinline__ uint32_t xcd_order(uint32_t b, uint32_t count) {
  const uint32_t x = b & 7, q = count >> 3, r = count & 7;
  return x * q + min(x, r) + (b >> 3);
}

}  // namespace bsscl
