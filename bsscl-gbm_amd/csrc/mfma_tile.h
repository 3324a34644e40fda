// Tiles of C(m, n) = sum_k A(m, k) B(n, k) on the matrix cores of gfx950, for
// bf16, fp16 and float32 operands with float32 sums.
//
// A workgroup holds a BM x BN tile in registers, WM x WN per wave in blocks of
// 16 x 16 (v_mfma 16x16x32, for float32 16x16x4: at the card's power limit they
// reach 1.9 PFLOP/s in bf16 from registers, 32x32x16 1.7), and walks k in
// steps.  Both operands' steps go from memory straight to LDS (buffer loads with
// the lds bit: no registers), into a ring of buffers.  An operand lies in
// memory with k contiguous (rows of m or n) or with m or n contiguous (rows of
// k):
//   k contiguous   LDS rows of one step's bytes; a lane reads 16 bytes of a row
//   k across rows  LDS rows of the tile's m (n) range; 16-bit fragments come
//                  from transposing reads (ds_read_b64_tr_b16: a group of 16
//                  lanes reads 4 k x 16 m and gets k in registers)
// An LDS place is lane-linear in the load, so the places of 16-byte chunks
// (place_of, which keeps what is read at once on different banks) permute the
// lanes' addresses in memory.  Reads outside the operand return 0 (the buffer
// descriptor's bound), so edges need no other care: offsets of lanes that are
// not to read are 2^31, beyond every bound.
//
// Fragment of a 16 x 16 block, lane l: row (column) l % 16 and 16 bytes of k
// from 16 (l / 16) on; result register r: m = 4 (l / 16) + r, n = l % 16.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

namespace bsscl {

typedef int Int4 __attribute__((ext_vector_type(4)));
typedef float Acc4 __attribute__((ext_vector_type(4)));
typedef __bf16 Bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 F16x8 __attribute__((ext_vector_type(8)));
typedef short Short4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kNoRead = 0x80000000u;  // a lane's offset beyond every bound

// acc += a b over one 16-byte fragment of k.
template <typename T>
__device__ __forceinline__ Acc4 mma(Int4 a, Int4 b, Acc4 acc) {
  if constexpr (std::is_same<T, __bf16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Bf16x8, a),
                                                   __builtin_bit_cast(Bf16x8, b), acc, 0, 0, 0);
  } else if constexpr (std::is_same<T, _Float16>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(F16x8, a),
                                                  __builtin_bit_cast(F16x8, b), acc, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, (int)a[j]),
                                                 __builtin_bit_cast(float, (int)b[j]), acc, 0, 0,
                                                 0);
    return acc;
  }
}

// 16 bytes per lane from memory to LDS at lds_at + 16 lane.  In assembly
// because the compiler would wait for it before every transposing read; the
// walk below waits itself.  The compiler sees no load here and inserts no wait
// states: one after the write of m0 (which it reserves and has no use of its own
// for), and five after a vector instruction that wrote a register of rsrc.  The
// move and four of s_nop are these five, whatever stands before them (up to 1% of
// the products; with s_nop 0 they depended on what the compiler put there).
__device__ __forceinline__ void load_to_lds(Int4 rsrc, uint32_t offset, uint32_t lds_at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
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
  static_assert(kLoads >= 1 && kLoads * 1024 * WAVES == kBytes && kChunks <= 64 &&
                    WAVES % 2 == 0,  // (a lane then has one chunk in all its loads)
                "tile shape");

  // The place of chunk c of LDS row r, its own inverse.  Banks repeat every 256
  // bytes.  Sixteen lanes read at once
  //   k contiguous: 16 bytes each, one chunk of 16 rows, kPerLine of which
  //     share a line of 256 bytes: these rows' places follow from the others';
  // or 32 lanes
  //   k across, 16 bits: two chunks of rows k + 0..3 and k + 8..11;
  //   k across, float32: four chunks of rows k and k + 4 (k + 8, k + 12).
  static constexpr int kPerLine = 256 / kRowBytes > 0 ? 256 / kRowBytes : 1;
  __device__ static __forceinline__ int place_of(int c, int r) {
    int x;
    if constexpr (!ACROSS) x = r / kPerLine;
    else if constexpr (kES == 2) x = (r & 3) * 4 + ((r >> 3) & 1) * 2;
    else x = ((r >> 2) & 3) * 4;
    return c ^ (x & (kChunks - 1));
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

  // The step that begins at k of k_end (zeros from there on), into LDS at
  // lds_at: its buffer descriptor, and the wave's loads one by one.
  struct Step {
    Int4 rsrc;
    uint32_t at;
    int32_t bytes;
  };
  __device__ __forceinline__ Step step(int64_t k, int64_t k_end, uint32_t lds_at) const {
    const int64_t left = max(k_end - k, (int64_t)0);
    const bool any = valid > 0 && left > 0;
    Step s;
    s.at = lds_at + ((uint32_t)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) << 10);
    if constexpr (!ACROSS) {
      // (Rows are padded to whole chunks.)
      s.bytes = (int32_t)min((left * kES + 15) & ~int64_t(15), (int64_t)STEP);
      s.rsrc = buffer_of(base + k * kES,
                         any ? (uint32_t)((valid - 1) * stride) + (uint32_t)s.bytes : 0);
    } else {
      const int32_t rows = (int32_t)min(left, (int64_t)kStep);
      s.bytes = STEP;
      s.rsrc = buffer_of(base + k * stride,
                         any ? (uint32_t)((rows - 1) * stride) + (uint32_t)(valid * kES) : 0);
    }
    return s;
  }
  __device__ __forceinline__ void load(const Step &s, int i) const {
    const bool in = ACROSS || (int)(chunk * 16) < s.bytes;
    load_to_lds(s.rsrc, in ? offset[i] : kNoRead, s.at + (uint32_t)(i * WAVES * 1024));
  }

  // The fragment of k part `part` (of STEP / 64) and the 16 rows from `first` on.
  __device__ static __forceinline__ Int4 fragment(const char *lds, int first, int part) {
    const int l = (int)threadIdx.x & 63, g = l >> 4;
    if constexpr (!ACROSS) {
      return *reinterpret_cast<const Int4 *>(lds + (first + (l & 15)) * STEP +
                                             (place_of(part * 4 + g, l & 15) << 4));
    } else if constexpr (kES == 2) {
      const int k = part * 32 + g * 8 + ((l & 15) >> 2), m = first + (l & 3) * 4;
      const char *p = lds + k * kRowBytes + (place_of(m >> 3, k) << 4) + (m & 4) * 2;
      typedef __attribute__((address_space(3))) Short4 *LdsShort4;
      const Short4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4)(p));
      const Short4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsShort4)(p + 4 * kRowBytes));
      typedef short Short8 __attribute__((ext_vector_type(8)));
      return __builtin_bit_cast(Int4, (Short8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int k = part * 16 + g * 4, m = first + (l & 15);
      const char *p = lds + k * kRowBytes + (place_of(m >> 2, k) << 4) + (m & 3) * 4;
      Int4 f;
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = *reinterpret_cast<const int *>(p + j * kRowBytes);
      return f;
    }
  }
};

// In every wave: all reads of LDS have arrived, and all but the last VM loads
// to it have landed.
template <int VM>
__device__ __forceinline__ void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(VM) : "memory");
}

// A tile's shape: BM x BN per workgroup, WM x WN per wave; STEP bytes of k at
// a time, STAGES of them in LDS.
template <typename T_, int BM_, int BN_, int WM_, int WN_, bool A_ACROSS, bool B_ACROSS, int STEP,
          int STAGES>
struct Tile {
  using T = T_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kWavesM = BM / WM, kWavesN = BN / WN, kWaves = kWavesM * kWavesN;
  static constexpr int kThreads = kWaves * 64;
  static constexpr int MI = WM / 16, NI = WN / 16;
  using A = Operand<T, BM, A_ACROSS, kWaves, STEP>;
  using B = Operand<T, BN, B_ACROSS, kWaves, STEP>;
  static constexpr int kStep = A::kStep, kParts = STEP / 64;
  static constexpr int kJoin = !A_ACROSS && MI * NI <= 8 ? 4 : 0;  // steps of a sum; 0: all
  static constexpr int kStage = A::kBytes + B::kBytes;
  static constexpr int kLds = STAGES * kStage;
  static_assert(kLds <= 160 * 1024 && STAGES >= 2 && MI >= 2 && kParts % 2 == 0, "tile shape");

  // total[mi][ni] += products of k in [k_begin, k_end); k_begin is a multiple of
  // kStep.  Every thread of the workgroup calls it; LDS is free at its end.
  //
  // Score tiles with registers left add up kJoin steps by themselves (128 float32
  // terms, 256 of 16 bits) and those sums then: in one chain, 65,536 equal float32
  // terms were off by 3e-4 of their sum, and the losses of 200 rows of 8,192 by
  // 1.1e-6, now 1e-7 (times level: 420 us against 424, 700 x 1,024 x 30,011).  256 x
  // 256 tiles have none left; their terms are of 16 bits, 32 to a link.  The
  // products' chains are level with those of plain products, and joins took 10% of
  // them (1,024 x 2,048 x 50,257 float32).
  //
  // Fragments are read one part ahead of the products that use them: a row of
  // blocks done, its A fragment of the next part is read in its place.  A step
  // has one barrier, in its last part: every wave has read all of the step, into
  // whose buffer the loads of step k + STAGES go from there on, and step k + 1
  // has landed in every wave and is read from there on.  (It stands behind the
  // part's first row of blocks, by which the last reads have arrived.)  Reads
  // and loads are dealt out among the products, so that no more than a few are
  // issued between two of them and the matrix cores multiply on.  256 x 256 bf16
  // tiles reach 1.25 to 1.3 PFLOP/s (products of 6,144 x 4,096 x 131,072), the
  // matrix cores 0.7 busy at the 1.8 GHz that the power limit leaves; with the
  // reads in front of the products it was 1.15, and with steps of half the bytes
  // in four or five buffers 1.2 (k contiguous: half lines, twice the requests).
  __device__ static __forceinline__ void walk(const A &a, const B &b, int64_t k_begin,
                                              int64_t k_end, char *lds, Acc4 (&total)[MI][NI]) {
    const int wave = (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / kWavesN * WM, wn = wave % kWavesN * WN;
    const uint32_t lds_at =
        (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    constexpr int kLoads = A::kLoads + B::kLoads;
    Int4 fa[MI], fb[2][NI];
    for (int s = 0; s < STAGES; ++s) {
      const int64_t k = k_begin + s * kStep;
      const auto sa = a.step(k, k_end, lds_at + (uint32_t)(s * kStage));
      const auto sb = b.step(k, k_end, lds_at + (uint32_t)(s * kStage + A::kBytes));
#pragma unroll
      for (int i = 0; i < A::kLoads; ++i) a.load(sa, i);
#pragma unroll
      for (int i = 0; i < B::kLoads; ++i) b.load(sb, i);
    }
    wait_and_meet<(STAGES - 1) * kLoads>();
#pragma unroll
    for (int j = 0; j < NI; ++j) fb[0][j] = B::fragment(lds + A::kBytes, wn + j * 16, 0);
#pragma unroll
    for (int i = 0; i < MI; ++i) fa[i] = A::fragment(lds, wm + i * 16, 0);
    int buf = 0;
    Acc4 own[kJoin ? MI : 1][kJoin ? NI : 1] = {};
    Acc4(&acc)[MI][NI] = [&]() -> Acc4(&)[MI][NI] {
      if constexpr (kJoin > 0) return own;
      else return total;
    }();
    auto join = [&] {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          total[i][j] += acc[i][j];
          acc[i][j] = Acc4{0.f, 0.f, 0.f, 0.f};
        }
    };
    int steps = 0;
    for (int64_t k = k_begin; k < k_end; k += kStep) {
      const int next = buf + 1 == STAGES ? 0 : buf + 1;
      const char *cur = lds + buf * kStage, *then = lds + next * kStage;
      const uint32_t at = lds_at + (uint32_t)(buf * kStage);
      const auto sa = a.step(k + STAGES * kStep, k_end, at);
      const auto sb = b.step(k + STAGES * kStep, k_end, at + A::kBytes);
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        const bool last = part == kParts - 1;
        const int set = part & 1;  // (the step's parts are even in number)
        const char *from = last ? then : cur;
        const int np = last ? 0 : part + 1;
        // Rows of blocks beside which reads and loads are issued.
        const int r0 = last ? 1 : 0, rows = MI - r0;
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          __builtin_amdgcn_sched_barrier(0);
          if (last && i == 1) {
            wait_and_meet<(STAGES - 2) * kLoads>();
            fa[0] = A::fragment(from, wm, np);
          }
          if (last && i >= r0) {
#pragma unroll
            for (int e = (i - r0) * kLoads / rows; e < (i - r0 + 1) * kLoads / rows; ++e) {
              if (e < A::kLoads)
                a.load(sa, e);
              else
                b.load(sb, e - A::kLoads);
            }
          }
          if (i >= r0)
#pragma unroll
            for (int j = (i - r0) * NI / rows; j < (i - r0 + 1) * NI / rows; ++j)
              fb[set ^ 1][j] = B::fragment(from + A::kBytes, wn + j * 16, np);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < NI; ++j) acc[i][j] = mma<T>(fa[i], fb[set][j], acc[i][j]);
          if (i >= r0) fa[i] = A::fragment(from, wm + i * 16, np);
        }
      }
      buf = next;  // (Loads beyond k_end are of zeros.)
      if constexpr (kJoin > 0)
        if (++steps == kJoin) {
          join();
          steps = 0;
        }
    }
    if constexpr (kJoin > 0) join();
    __builtin_amdgcn_sched_barrier(0);
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
      for (int j = 0; j < NI; ++j) {
        const int n = wn + j * 16 + (l & 15), m = wm + i * 16 + (l >> 4) * 4;
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = value(i, j, r);
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
