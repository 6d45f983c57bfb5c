// Causal attention of whole prompts: packed sequences of different lengths, grouped heads.
//
//   o_i = sum_{j <= i} exp(s_ij - m_i) v_j / sum_{j <= i} exp(s_ij - m_i),   s_ij = scale q_i . k_j
//
// with a running maximum, sum and output over steps of 128 keys.  A block works on two tiles of 128 query rows that share
// their keys and values -- two heads of a group at the same tokens, or 256 tokens of a head -- so that the tensor cores have
// one tile's products to do while the other tile's exponentials are taken:
//
//   warp 0        copies (TMA): queries, then keys and values in turn through a ring
//   warp 2        plans: which tiles, ahead of the others
//   warps 1 and 3 a tile each, tcgen05.mma: S = Q K^T from shared memory, O += P V with P from tensor memory (one thread for
//                 both kept each waiting for the other's weights: 2048 tokens of 32 heads 44.6 us, 42.5 with two)
//   warps 4-7 and 8-11, one group to a tile: a thread has one row; it takes S from tensor memory, the row's maximum, the
//                 exponentials, and leaves P, rounded, where S was
//
// Scores, exponentials, product and next scores are a chain for each row; so that the exponential unit is not left waiting for
// the tensor cores, the next scores have to be there when a group is done.  Tensor memory has 512 columns.  With heads of 128
// values S and O take all of it, and a step goes through in two halves of 64 keys, each with its own place for S and P: while
// one half is multiplied, the exponentials of the other are taken.  (2048 tokens of 32 heads: in whole steps 46.4 us, in
// halves 41.5.  The products of 64 columns cost the tensor cores a quarter more time, and 8192 tokens of 64 heads gained
// nothing: 1013, 1031.)  With heads of 64 values there is room for P beside S, and the next
// scores are sent for as soon as these are read (whole steps with P in S's place 540 us, halves 549, P apart 528).
//
// The output is rescaled only when a row's maximum has grown by more than 2^8 since the last time (the weights stay in
// either type's range, the sum is in fp32), so most steps leave O alone.  Bounds: for heads of 128 values a tile's two
// products of a step take the tensor cores 1300 clocks (1024 at their best), its 16384 exponentials 1024.
//
// What a row may not attend to must not reach it, whatever it holds: scores are replaced where masked, but 0 x NaN is NaN in
// the product with V.  So before the last step of a tile's rows the group clears rows of V behind the sequence's end and
// looks for values that are not finite; where there are any, the threads add that step's product up themselves.
#include <limits>

#include "attention.cuh"

namespace mp {
namespace {

using namespace attn;
using namespace tc;

constexpr int kTile = 128;                     // query rows of a tile and keys of a step
// Four warps of copies, products and planning, and two groups of four.  Registers: the block starts with 168 a
// thread, 64512 in all; the first four warps give back what the others take, 128 x 72 + 256 x 216 = 64512.
constexpr int kWarps = 12, kThreads = 32 * kWarps;
constexpr int kFewRegisters = 72, kManyRegisters = 216;
constexpr int kTmemCols = 512;
constexpr float kGrowth = 8.0f;                // log2 of how far a row's maximum may grow before it is taken
// Weights are 2^(s - m + lift), rounded to the type before the product with V, since that is what the tensor cores multiply (their
// sum is of the unrounded ones; results are off by 2.6e-4 of their norm in fp16 and 2.0e-3 in bf16, with 32-bit weights 2.0e-4 and
// 1.5e-3): below 2^15 in fp16, where many weights beneath the type's 24 bits below 1 would be lost together.
template <typename T> constexpr float kLift = __is_same(T, __half) ? 15.0f - kGrowth : 0.0f;
constexpr int kAhead = 4;                      // items that the planning warp is ahead
constexpr int kSortedBatch = 256;              // sequences whose tiles are taken longest first

template <int DP>
struct Prefill {
  static constexpr int kBoxes = DP / 64;                       // copies of 64 columns
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kStages = 4;
  // P beside S, and a step in one part; or a step in two, whose weights take their scores' place
  static constexpr bool kApart = DP == 64;
  static constexpr int kParts = kApart ? 1 : 2, kPart = kTile / kParts;
  // tensor memory: S of either tile, O of either tile, and P
  static constexpr int kWeights = kApart ? 2 * (kTile + DP) : 0, kWeightStep = kApart ? kTile / 2 : kTile;
  static constexpr int kMultiplied = DP == 64 ? 1 : 2;         // of eight pairs of weights
  static constexpr int kBarBytes = 512;
  static constexpr int kOutColumns = DP / 2;
  static constexpr int kOutBytes = 8 * 32 * 2 * kOutColumns;   // 32 rows of these for each of eight warps
  static constexpr int kSmem = 2 * kTileBytes + kStages * kTileBytes + kOutBytes + kBarBytes + 1024;
};

struct MapOrder {
  int token_first;                             // the tensor map's dimensions are D, token, head; else D, head, token
  int one_head;                                // all heads are the same rows
};

struct PrefillParams {
  const int* cu_seqlens;
  char* out;
  int* index_word;
  int* error_word;
  int tokens, batch, q_heads, group, dim;
  int pair_heads;                              // the block's two tiles: 1 two heads, 0 two tiles of a head
  int slots, per_slot;                         // numbers of row tiles, and the items of each
  float scale_log2;                            // |scale| log2 e
  uint32_t negate;                             // scale < 0: the bit of the products' descriptor that negates Q
  MapOrder q_order, k_order, v_order;
};

// Products with a descriptor's low word and the high word that all of a layout share; ACC: added to what is there.
template <bool ACC>
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t a_hi, uint32_t b, uint32_t b_hi, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .b64 a, b;\n\t.reg .pred p;\n\tmov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t}"
      ::"r"(d), "r"(a), "r"(a_hi), "r"(b), "r"(b_hi), "r"(idesc), "n"(ACC ? 1 : 0) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .b64 b;\n\t.reg .pred p;\n\tmov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(b_hi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// one column of the warp's 32 lanes, complete on return
__device__ __forceinline__ uint32_t tmem_ld_column(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;" : "=r"(r) : "r"(taddr) : "memory");
  return r;
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// Eight values times zero, added to a pair: NaN from the first value on that is infinite or NaN.
template <typename T> struct Pair;
template <> struct Pair<__half> { using type = __half2; };
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
template <typename T> __device__ __forceinline__ uint32_t add_zeros(uint32_t acc, const uint4& v) {
  using P = typename Pair<T>::type;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w}, zero = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    acc = bits(__hfma2(*reinterpret_cast<const P*>(&w[i]), *reinterpret_cast<const P*>(&zero), *reinterpret_cast<P*>(&acc)));
  return acc;
}

// Larger of three, NaN if one is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Pairs of fp32 values in one instruction.  (volatile: in the order they are written in, which exp2_batch is about)
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(F2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm volatile("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm volatile("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float exp2_ordered(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Weights 2^(s scale - ref) of 16 scores, their sum added to `sum` and the weights rounded to eight words.  E of the eight
// pairs are computed by multiplications while the exponential unit has the others: x = n + f with n the nearest integer, 2^f
// by a polynomial of degree 5 (minimax on [-1/2, 1/2], found by exchange; relative error 2^-22.6 with the constants rounded to
// fp32, 2^-22.1 as evaluated), n added to the exponent.
// x is at most about 2^7; below -127 it counts as -127, which gives 2^-149, 0 when rounded.  (A NaN does not come through there: see the maximum.)
// The unit takes 16 values a clock and SM, 1024 clocks for a tile.  In this order, by hand, the instructions of a warp that
// is alone on its scheduler keep it busy; as the compiler orders a plain loop they took 1650.  With none, one, two of eight by
// multiplications: 2048 tokens of 32 heads 43.0, 42.5, 41.9 us, 8192 tokens of 64 heads 1085, 1070, 1050; prompts with heads
// of 64 values, whose products are short, with one or two 527, 549.
// between(m), m < 8 - E: what else can be done meanwhile.
template <typename T, int E, typename F>
__device__ __forceinline__ void exp2_batch(const uint32_t* s, F2 scale, F2 minus_ref, F2& sum, uint32_t* packed, F between) {
  constexpr float kMagic = 12582912.0f;        // 1.5 * 2^23: added, the sum's low bits are the nearest integer
  constexpr float kC[6] = {1.3276472454890609e-3f, 9.675540961325169e-3f, 5.550713092088699e-2f,
                           0.24022120237350464f, 0.6931469440460205f, 1.0000001192092896f};
  constexpr int U = 8 - E;                     // pairs that the unit takes
  static_assert(E == 1 || E == 2, "");
  F2 x[8], t[8], f[8], r[8];
  float v[16];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = fma2(f2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), scale, minus_ref);
#pragma unroll
  for (int e = U; e < 8; ++e) {
    float a, b;
    split(x[e], a, b);
    x[e] = f2(fmaxf(a, -127.0f), fmaxf(b, -127.0f));
    t[e] = add2(x[e], f2(kMagic, kMagic));
  }
#pragma unroll
  for (int m = 0; m < U; ++m) {
    float a, b;
    split(x[m], a, b);
    v[2 * m] = exp2_ordered(a);
    v[2 * m + 1] = exp2_ordered(b);
#pragma unroll
    for (int e = U; e < 8; ++e) {
      const int step = m + 7 - U;              // (of seven; the first two together if there are six turns)
      if (m == 0) f[e] = fma2(t[e], f2(-1.0f, -1.0f), f2(kMagic, kMagic));
      if (step == 1) f[e] = add2(x[e], f[e]);
      if (step == 2) r[e] = fma2(f2(kC[0], kC[0]), f[e], f2(kC[1], kC[1]));
      if (step > 2 && step <= 6) r[e] = fma2(r[e], f[e], f2(kC[step - 1], kC[step - 1]));
    }
    between(m);
  }
#pragma unroll
  for (int e = U; e < 8; ++e) {
    float a, b, t0, t1;
    split(r[e], a, b);
    split(t[e], t0, t1);
    v[2 * e] = __uint_as_float(__float_as_uint(a) + (__float_as_uint(t0) << 23));
    v[2 * e + 1] = __uint_as_float(__float_as_uint(b) + (__float_as_uint(t1) << 23));
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    sum = add2(sum, f2(v[2 * e], v[2 * e + 1]));
    packed[e] = pack2<T>(v[2 * e], v[2 * e + 1]);
  }
}

// Descriptor of V as the B operand [dims x keys] whose rows in memory are keys (128 bytes of 64 dims, 128-byte swizzle):
// eight keys are 1024 bytes apart, the next 64 dims one box of the tile.
__device__ __forceinline__ uint64_t umma_desc_rows_sw128(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((kTile * 128) >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// What a block does next: one tile's queries of a sequence, or none (no steps).
struct Work {
  int begin, len;              // the sequence
  int row[2], head[2];         // the two tiles' first rows within it, and their heads
  int steps[2];                // tiles of keys; 0: there is no such tile
  int kv;
};

// The items of a block, in turn, found by a warp.  With up to 256 sequences the tiles of rows are taken by how many keys they
// have, longest first, and dealt to the blocks back and forth, so that all blocks have about as much to do (one prompt of
// 2048 tokens and 32 heads dealt in one direction: a third of the SMs' time idle).  With more, in
// the order of the batch.  (In order and by length: 40 prompts of about 200 tokens, of very different lengths, 100 and 80 us, 40
// of 1000 1172 and 1175; 256 of 100 318 and 326, 256 of 400 1586 and 1510: with many tiles a block the order matters little.)
struct Planner {
  const PrefillParams& p;
  int lane, rows, round = 0;
  int tiles[kSortedBatch / 32];            // of sequences lane, lane + 32, ...
  int total;                               // tiles of rows in all (sorted), numbers for them (not sorted)
  int level;                               // tiles with this many in front of them in their sequence are in turn

  __device__ __forceinline__ bool sequence(int b, int& begin, int& len) const {
    begin = __ldg(p.cu_seqlens + b);
    const int end = __ldg(p.cu_seqlens + b + 1);
    const bool good = begin >= 0 && end >= begin && end <= p.tokens;
    if (!good && p.index_word) *p.index_word = kBadIndex;
    len = good ? end - begin : 0;
    return good;
  }
  // Not sorted, next() looks at the sequences that its search arrives at, which ends out of order mislead.  All of them are
  // looked at when the block's last item is planned, a share by each block.
  __device__ __forceinline__ void check_ends() const {
    if (p.batch <= kSortedBatch) return;
    for (long long b = static_cast<long long>(blockIdx.x) * 32 + lane; b < p.batch; b += gridDim.x * 32) {
      int begin, len;
      sequence(static_cast<int>(b), begin, len);
    }
  }
  __device__ __forceinline__ int beyond(int l) const {        // tiles with at least l in front of them
    int n = 0;
#pragma unroll
    for (int k = 0; k < kSortedBatch / 32; ++k) n += max(0, tiles[k] - l);
    return __reduce_add_sync(0xffffffffu, n);
  }
  __device__ __forceinline__ Planner(const PrefillParams& params, int lane_)
      : p(params), lane(lane_), rows(params.pair_heads ? kTile : 2 * kTile) {
    total = p.slots;
    level = 0;
    if (p.batch > kSortedBatch) return;
    int most = 0;
#pragma unroll
    for (int k = 0; k < kSortedBatch / 32; ++k) {
      int begin, len = 0;
      if (k * 32 + lane < p.batch) sequence(k * 32 + lane, begin, len);
      tiles[k] = (len + rows - 1) / rows;
      most = max(most, tiles[k]);
    }
    level = max(0, __reduce_max_sync(0xffffffffu, most) - 1);
    total = beyond(0);
  }
  // (the whole warp)
  __device__ __forceinline__ bool next(Work& w) {
    for (;; ++round) {
      const int item = round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
      // (a round's items are all beyond those of the round before)
      if (item >= total * p.per_slot) return false;
      const int rank = item / p.per_slot, at = item - rank * p.per_slot;
      int b, row;
      if (p.batch <= kSortedBatch) {
        int lo = 0;                          // the largest level <= the present one with beyond(level) > rank
        while (lo < level) {
          const int mid = (lo + level + 1) / 2;
          if (beyond(mid) > rank) lo = mid; else level = mid - 1;
        }
        int index = rank - beyond(level + 1);
        b = 0;
#pragma unroll
        for (int k = 0; k < kSortedBatch / 32; ++k) {
          const uint32_t there = __ballot_sync(0xffffffffu, tiles[k] > level);
          const bool me = tiles[k] > level && __popc(there & ((1u << lane) - 1)) == index;
          const uint32_t who = __ballot_sync(0xffffffffu, me);
          if (who) b = k * 32 + __ffs(who) - 1;
          index -= __popc(there);
        }
        row = level * rows;
      } else {
        // Numbers of row tiles: sequence b has those from cu[b] / rows + b on, which is room for all its tiles, so that a
        // tile's sequence is found without the others' sum.
        const int number = p.slots - 1 - rank;
        int lo = 0, hi = p.batch;
        while (hi - lo > 1) {
          const int mid = (lo + hi) / 2;
          if (__ldg(p.cu_seqlens + mid) / rows + mid <= number) lo = mid; else hi = mid;
        }
        b = lo;
        row = (number - __ldg(p.cu_seqlens + b) / rows - b) * rows;
      }
      if (!sequence(b, w.begin, w.len) || row < 0 || row >= w.len) continue;
      ++round;
      w.row[0] = row;
      w.row[1] = p.pair_heads ? row : row + kTile;
      w.head[0] = p.pair_heads ? 2 * at : at;
      w.head[1] = p.pair_heads ? 2 * at + 1 : at;
      w.kv = w.head[0] / p.group;
#pragma unroll
      for (int i = 0; i < 2; ++i) w.steps[i] = w.row[i] < w.len ? w.row[i] / kTile + 1 : 0;
      return true;
    }
  }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1)
prefill_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
               const __grid_constant__ CUtensorMap map_v, const PrefillParams p) {
  using C = Prefill<DP>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (2 + C::kStages) * C::kTileBytes + C::kOutBytes);
  const uint32_t q_tile = smem_u32(smem), ring = q_tile + 2 * C::kTileBytes;
  const uint32_t kv_full = smem_u32(bars), kv_empty = kv_full + 8 * C::kStages, q_full = kv_empty + 8 * C::kStages,
                 q_empty = q_full + 16, s_full = q_empty + 16 /* [tile][part of the step] */, p_ready = s_full + 32 /* the same */,
                 o_done = p_ready + 32 /* the same */, scanned = o_done + 32, s_read = scanned + 16,
                 work_full = s_read + 16, work_empty = work_full + 8 * kAhead;
  constexpr int kBars = 2 * C::kStages + 20 + 2 * kAhead;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // [tile][item's parity]: the last product of the tile's item is not the MMA's
  volatile int* odd_values = reinterpret_cast<volatile int*>(tmem_slot + 2);
  Work* works = reinterpret_cast<Work*>(tmem_slot + 6);
  static_assert(8 * kBars + 24 + kAhead * sizeof(Work) <= C::kBarBytes, "");

  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(kv_full + 8 * s, 1);
      mbar_init(kv_empty + 8 * s, 2);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + 8 * i, 1);
      mbar_init(q_empty + 8 * i, 1);
      for (int part = 0; part < 2; ++part) {
        mbar_init(s_full + 16 * i + 8 * part, 1);
        mbar_init(p_ready + 16 * i + 8 * part, 4);
        mbar_init(o_done + 16 * i + 8 * part, 1);
      }
      mbar_init(s_read + 8 * i, 4);
      mbar_init(scanned + 8 * i, 4);
      odd_values[2 * i] = odd_values[2 * i + 1] = 0;
    }
    for (int a = 0; a < kAhead; ++a) {
      mbar_init(work_full + 8 * a, 1);
      mbar_init(work_empty + 8 * a, 11);       // the copying and the two multiplying threads, eight warps
    }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  chain_wait();
  chain_release();

  Work w;
  int taken = 0;                               // items this role has taken
  // (each side's code hangs below its own setmaxnreg, or the compiler holds all of it to the smaller number)
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
    // the next item, for a role of one thread
    auto take = [&](Work& x) {
      const int a = taken % kAhead;
      if (!mbar_wait(work_full + 8 * a, (taken / kAhead) & 1, abort_flag)) return false;
      x = works[a];
      mbar_arrive(work_empty + 8 * a);
      ++taken;
      return x.steps[0] != 0;
    };
    if (warp == 0 && elect_one()) {
      int load = 0;                            // copies of keys and values so far
      uint32_t q_phase[2] = {1, 1};
      bool ok = true;
      auto copy = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, const MapOrder& order, int head, int token) {
        if (order.one_head) head = 0;
#pragma unroll
        for (int b = 0; b < C::kBoxes; ++b)
          tma_load_3d(dst + b * kTile * 128, map, bar, b * 64, order.token_first ? token : head, order.token_first ? head : token);
      };
      auto next_slot = [&](uint32_t& dst, uint32_t& bar) {
        const int s = load % C::kStages;
        dst = ring + s * C::kTileBytes;
        bar = kv_full + 8 * s;
        if (!mbar_wait(kv_empty + 8 * s, ((load / C::kStages) & 1) ^ 1, abort_flag)) return false;
        mbar_arrive_expect_tx(bar, C::kTileBytes);
        ++load;
        return true;
      };
      while (ok && take(w)) {
        const int steps = max(w.steps[0], w.steps[1]);
        uint32_t dst, bar;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!w.steps[i]) continue;
          if (!mbar_wait(q_empty + 8 * i, q_phase[i], abort_flag)) { ok = false; break; }
          q_phase[i] ^= 1;
          mbar_arrive_expect_tx(q_full + 8 * i, C::kTileBytes);
          copy(q_tile + i * C::kTileBytes, &map_q, q_full + 8 * i, p.q_order, w.head[i], w.begin + w.row[i]);
          if (i == 0) {
            if (!next_slot(dst, bar)) { ok = false; break; }
            copy(dst, &map_k, bar, p.k_order, w.kv, w.begin);
          }
        }
        for (int j = 0; ok && j < steps; ++j) {
          if (j) {
            if (!next_slot(dst, bar)) { ok = false; break; }
            copy(dst, &map_k, bar, p.k_order, w.kv, w.begin + j * kTile);
          }
          if (!next_slot(dst, bar)) { ok = false; break; }
          copy(dst, &map_v, bar, p.v_order, w.kv, w.begin + j * kTile);
        }
      }
    }
    if ((warp == 1 || warp == 3) && elect_one()) {
      const int i = warp >> 1;                 // its tile
      constexpr uint32_t kFormats = kIdescDFormatF32 | (__is_same(T, __half) ? 0u : (1u << 7) | (1u << 10));
      const uint32_t idesc_qk = umma_idesc(kFormats, kTile, C::kPart) | p.negate;
      constexpr uint32_t kIdescPV = umma_idesc(kFormats, kTile, DP) | (1u << 16);      // B's rows in memory are K
      const uint64_t k_desc = umma_desc_k_sw128(ring), v_desc = umma_desc_rows_sw128(ring);
      const uint32_t k_lo = static_cast<uint32_t>(k_desc), k_hi = static_cast<uint32_t>(k_desc >> 32);
      const uint32_t v_lo = static_cast<uint32_t>(v_desc), v_hi = static_cast<uint32_t>(v_desc >> 32);
      const uint32_t q_lo = static_cast<uint32_t>(umma_desc_k_sw128(q_tile));
      constexpr uint32_t kTileStep = C::kTileBytes >> 4;
      auto wait = [&](uint32_t bar, uint32_t phase) { return mbar_wait(bar, phase, abort_flag); };
      struct Slot {                            // of the ring, in the order of the copies
        uint32_t at = 0, phase = 0;
        __device__ __forceinline__ void step(int n) {
          at += n;
          phase ^= (at / C::kStages) & 1;
          at %= C::kStages;
        }
      };
      uint32_t q_phase = 0, p_phase = 0, parity = 0;
      auto full = [&](const Slot& s) { return wait(kv_full + 8 * s.at, s.phase); };
      auto scores = [&](const Slot& s, int part) {            // S_i = Q_i K^T of a part of the step's keys
        const uint32_t a = q_lo + i * kTileStep, b = k_lo + s.at * kTileStep + part * ((C::kPart * 128) >> 4);
        const uint32_t d = tmem + i * kTile + part * C::kPart;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint32_t at = (k >> 2) * ((kTile * 128) >> 4) + 2 * (k & 3);
          if (k == 0) umma_ss<false>(d, a + at, k_hi, b + at, k_hi, idesc_qk);
          else umma_ss<true>(d, a + at, k_hi, b + at, k_hi, idesc_qk);
        }
        umma_commit(s_full + 16 * i + 8 * part);
      };
      // what this tile has used, or has no use for
      auto release = [&](const Slot& s, bool used) {
        if (used) umma_commit(kv_empty + 8 * s.at);
        else if (full(s)) mbar_arrive(kv_empty + 8 * s.at);
      };
      int steps, then, most, then_most;
      auto take_steps = [&]() {                // of the next item
        const int a = taken % kAhead;
        if (!wait(work_full + 8 * a, (taken / kAhead) & 1)) return false;
        then = works[a].steps[i];
        then_most = max(works[a].steps[0], works[a].steps[1]);
        const bool there = works[a].steps[0] != 0;
        mbar_arrive(work_empty + 8 * a);
        ++taken;
        return there;
      };
      // The first scores of an item follow the last product of the one before: the ring has room for the two copies that tile 0
      // may be ahead of tile 1.
      auto first_scores = [&](const Slot& s, int part) {
        if (part == 0) {
          if (!wait(q_full + 8 * i, q_phase)) return false;
          q_phase ^= 1;
        }
        if (!full(s)) return false;
        scores(s, part);
        if (part + 1 == C::kParts && then == 1) umma_commit(q_empty + 8 * i);
        return true;
      };
      auto all_first_scores = [&](const Slot& s) { return first_scores(s, 0) && (C::kParts == 1 || first_scores(s, 1)); };
      Slot k;
      bool more = take_steps(), ok = true;
      if (more && then) ok = all_first_scores(k);
      while (ok && more) {
        steps = then;
        most = then_most;
        Slot v = k, next = k;                  // this step's values, the next item's first keys
        v.step(1);
        next.step(2 * most);
        release(k, steps != 0);
        k.step(2);                             // the next step's keys
        more = take_steps();
        for (int j = 0; ok && j < most; ++j) {
          const bool last = j + 1 >= steps;
          if (j < steps) {
            auto next_scores = [&](int part) {
              if (!full(k)) return false;
              scores(k, part);
              if (part + 1 == C::kParts && j + 2 == steps) umma_commit(q_empty + 8 * i);
              return true;
            };
            if (C::kApart) {                   // (S of this step has been read)
              ok = wait(s_read + 8 * i, p_phase);
              tcgen05_fence_after();
              if (ok && !last) ok = next_scores(0);
            }
            ok = ok && full(v);
#pragma unroll
            for (int part = 0; part < C::kParts; ++part) {
              if (!ok || !wait(p_ready + 16 * i + 8 * part, p_phase)) { ok = false; continue; }
              tcgen05_fence_after();
              if (!last || odd_values[2 * i + parity] == 0) {
                const uint32_t b = v_lo + v.at * kTileStep + part * (C::kPart * 128 >> 4);
#pragma unroll
                for (int k = 0; k < C::kPart / 16; ++k)
                  umma_ts(tmem + 2 * kTile + i * DP, tmem + C::kWeights + i * C::kWeightStep + part * C::kPart + k * 8,
                          b + k * ((16 * 128) >> 4), v_hi, kIdescPV, part + k != 0 ? 1u : j != 0);
              }
              umma_commit(o_done + 16 * i + 8 * part);
              if (!last) {
                if (!C::kApart) ok = next_scores(part);
              } else if (more && then) {
                ok = first_scores(next, part);
              }
            }
            p_phase ^= 1;
            if (last) parity ^= 1;
            if (!ok) break;
          }
          release(v, j < steps);
          if (j + 1 < most) {
            release(k, !last);
            k.step(2);
          }
          v.step(2);
        }
        k = next;
        if (ok && more && !steps && then) ok = all_first_scores(k);
      }
    }
    if (warp == 2) {
      Planner plan(p, lane);
      for (bool more = true; more; ++taken) {
        w.steps[0] = 0;
        more = plan.next(w);
        if (!more) w.steps[0] = 0;
        const int a = taken % kAhead;
        if (!__all_sync(0xffffffffu, mbar_wait(work_empty + 8 * a, ((taken / kAhead) & 1) ^ 1, abort_flag))) break;
        if (lane == 0) {
          works[a] = w;
          mbar_arrive(work_full + 8 * a);
        }
        __syncwarp();
      }
      plan.check_ends();
    }
  } else {
    // ---- one row of tile i to a thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
    const int i = warp >= 8, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_tmem = tmem + lanes + i * kTile, o_tmem = tmem + lanes + 2 * kTile + i * DP;
    const uint32_t p_tmem = tmem + lanes + C::kWeights + i * C::kWeightStep;
    uint32_t turn = 0, scan_phase = 0;         // parity of the steps so far, which is that of their scores and products
    int load = 0;
    bool ok = true;
    const F2 scale2 = f2(p.scale_log2, p.scale_log2);
    auto wait_all = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0; };
    while (ok) {
      const int slot = taken % kAhead;
      if (!wait_all(work_full + 8 * slot, (taken / kAhead) & 1)) break;
      const Work& next = works[slot];
      const int steps = next.steps[i], row_begin = next.row[i], head = next.head[i], seq_begin = next.begin, len = next.len;
      const int item_steps = max(next.steps[0], next.steps[1]);
      const bool end = next.steps[0] == 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(work_empty + 8 * slot);
      ++taken;
      if (end) break;
      const int first_load = load;
      load += 2 * item_steps;
      if (!steps) continue;
      float m = kNegInf, sum = 0.0f;
      uint32_t tile_v = 0;                     // of the last step
#pragma unroll 1
      for (int h = 0; h < C::kParts * steps; ++h) {
        const int part = C::kParts == 1 ? 0 : h & 1;
        const uint32_t p_part = p_tmem + part * C::kPart;
        // the tile's product before this part's: of the step before, or of its first half
        auto wait_before = [&]() {
          if (C::kParts == 1) return wait_all(o_done + 16 * i, turn ^ 1);
          return wait_all(o_done + 16 * i + 8 * (part ^ 1), turn ^ (part ^ 1));
        };
        if (!wait_all(s_full + 16 * i + 8 * part, turn)) { ok = false; break; }
        tcgen05_fence_after();
        const bool last = h + C::kParts >= C::kParts * steps;
        uint32_t s[C::kPart / 32][32];
#pragma unroll
        for (int c = 0; c < C::kPart / 32; ++c) tmem_ld_32x32(s_tmem + part * C::kPart + 32 * c, s[c]);
        tmem_ld_wait();
        if (C::kApart) {
          tcgen05_fence_before();
          mbar_arrive_warp(s_read + 8 * i, lane);
        }
        auto value = [&](int c) -> uint32_t& { return s[c >> 5][c & 31]; };
        if (last) {
#pragma unroll
          for (int c = 0; c < C::kPart; ++c) value(c) = part * C::kPart + c <= row ? value(c) : __float_as_uint(kNegInf);
        }
        // The weights are taken with the maximum of the parts before (the first one's own at first): it is still good if no
        // score exceeds it by 8.  The scores' maximum is found beside the exponentials; where it exceeds, they are taken once
        // more.  A NaN anywhere makes the maximum NaN, and with it the whole row; so does plus infinity.
        float top[4];
        auto look = [&](int c) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            top[e] = max3(c ? top[e] : __uint_as_float(value(e)), __uint_as_float(value(c + e)), __uint_as_float(value(c + e + 4)));
        };
        auto maximum = [&]() { return max3(m, max3(top[0], top[1], top[2]) * p.scale_log2, top[3] * p.scale_log2); };
        auto usable = [&](float now) { return now == -kNegInf ? __uint_as_float(0x7fffffffu) : now; };
        if (h == 0) {
#pragma unroll
          for (int c = 0; c < C::kPart; c += 8) look(c);
          m = usable(maximum());
        }
        F2 weights, minus_ref;
        uint32_t packed[32];
        for (bool again = h == 0;; again = true) {
          const float ref = m == kNegInf ? 0.0f : m;
          minus_ref = f2(kLift<T> - ref, kLift<T> - ref);
          weights = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b)
            exp2_batch<T, C::kMultiplied>(&value(16 * b), scale2, minus_ref, weights, packed + 8 * b, [&](int step) {
              if (step < C::kPart / 32) look(C::kPart / 4 * b + 8 * step);
            });
          const float now = maximum();
          if (again || !__any_sync(0xffffffffu, !(now <= m + kGrowth))) break;
          if (!wait_before()) { ok = false; break; }
          tcgen05_fence_after();
          const float grown = usable(now), keep = grown == kNegInf ? 1.0f : exp2_fast(m - grown);
          sum *= keep;
          m = grown;
#pragma unroll 1
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32(o_tmem + 32 * c, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
            tmem_st_32x32(o_tmem + 32 * c, o);
          }
        }
        if (!ok) break;
        if (C::kApart && !wait_before()) { ok = false; break; }        // P of the step before has been used
        tmem_st_32x32(p_part, packed);
        if (C::kPart == 128) {
#pragma unroll
          for (int b = 4; b < C::kPart / 16; ++b)
            exp2_batch<T, C::kMultiplied>(&value(16 * b), scale2, minus_ref, weights, packed + 8 * (b - 4), [](int) {});
          tmem_st_32x32(p_part + 32, packed);
        }
        float weight[2];
        split(weights, weight[0], weight[1]);
        sum += weight[0] + weight[1];
        if (last && part == 0) {
          // ---- V's rows behind the sequence's end, and values that are not finite
          const int n = first_load + 2 * h / C::kParts + 1, valid = len - h * C::kPart;
          if (!wait_all(kv_full + 8 * (n % C::kStages), (n / C::kStages) & 1)) { ok = false; break; }
          tile_v = ring + (n % C::kStages) * C::kTileBytes;
          uint32_t zeros = 0;
#pragma unroll 2
          for (int c = 0; c < 8 * C::kBoxes; ++c) {
            const int r = (c & 7) * 16 + quarter * 4 + (lane >> 3);       // 16 rows of eight pieces
            const uint32_t at = tile_v + (c >> 3) * kTile * 128 + r * 128 + (lane & 7) * 16;
            if (r < valid) zeros = add_zeros<T>(zeros, lds16(at));
            else asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(at), "r"(0u) : "memory");
          }
          if (valid < kTile) fence_proxy_async_smem();
          if (__any_sync(0xffffffffu, (zeros & 0x7fff7fffu) != 0) && lane == 0) odd_values[2 * i + scan_phase] = 1;
          // (whoever read the other one, for the item before, has done so: that item's last product is complete)
          if (quarter == 0 && lane == 0) odd_values[2 * i + (scan_phase ^ 1)] = 0;
          mbar_arrive_warp(scanned + 8 * i, lane);
          if (!wait_all(scanned + 8 * i, scan_phase)) { ok = false; break; }
          scan_phase ^= 1;
        }
        if (last && odd_values[2 * i + (scan_phase ^ 1)]) {
          // this row's product with the keys it attends to, 32 columns at a time
          tmem_st_wait();
          if (h > 0) {
            if (!wait_before()) { ok = false; break; }
            tcgen05_fence_after();
          }
#pragma unroll 1
          for (int d0 = 0; d0 < DP; d0 += 32) {
            uint32_t o[32];
            if (h > 0) {
              tmem_ld_32x32(o_tmem + d0, o);
              tmem_ld_wait();
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = 0u;
            }
#pragma unroll 1
            for (int c = 0; c < C::kPart; c += 2) {
              const float2 pair = unpack2<T>(tmem_ld_column(p_part + c / 2));
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int key = part * C::kPart + c + k;
                const bool attends = key <= row;       // (by selection: 0 x NaN is not to be added)
                const float weight = k ? pair.y : pair.x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint4 v = lds16(tile_v + (d0 >> 6) * kTile * 128 + key * 128 + ((((d0 & 63) / 8 + e) ^ (key & 7)) << 4));
                  const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                  for (int x = 0; x < 4; ++x) {
                    const float2 y = unpack2<T>(words[x]);
                    uint32_t &o0 = o[e * 8 + 2 * x], &o1 = o[e * 8 + 2 * x + 1];
                    o0 = attends ? __float_as_uint(fmaf(weight, y.x, __uint_as_float(o0))) : o0;
                    o1 = attends ? __float_as_uint(fmaf(weight, y.y, __uint_as_float(o1))) : o1;
                  }
                }
              }
              __syncwarp();                    // rows attend to different keys; all lanes are at the next load together
            }
            tmem_st_32x32(o_tmem + d0, o);
          }
        }
        tmem_st_wait();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + 16 * i + 8 * part);
        if (part + 1 == C::kParts) turn ^= 1;
      }
      if (!ok) break;
      // ---- the row's result
      if (!wait_all(o_done + 16 * i + 8 * (C::kParts - 1), turn ^ 1)) { ok = false; break; }
      tcgen05_fence_after();
      const float inv = 1.0f / sum;            // (0 where no score is above minus infinity: the row becomes 0 x infinity, NaN)
      // Half a head's columns at a time through shared memory, so that a warp's stores are whole lines or sectors (a row to a
      // thread took 3000 clocks of an item's end).  All of this code has to be fetched again when its turn comes, so a loop
      // gains where rows are short: heads of 64 values by 64 columns 518 us, by 32 512; of 128 values by 64 41.4, by 32 42.0.
      constexpr int kColumns = C::kOutColumns, kPieces = kColumns / 8;
      const uint32_t staged = ring + C::kStages * C::kTileBytes + ((warp - 4) * 32) * (kColumns * 2);
      const int first_row = row_begin + quarter * 32, own_row = lane / kPieces, piece = lane % kPieces;
      char* dst = p.out + ((static_cast<long long>(seq_begin) + first_row + own_row) * p.q_heads + head) * p.dim * 2 + piece * 16;
      const long long next_rows = static_cast<long long>(p.q_heads) * p.dim * (2 * 32 / kPieces);
#pragma unroll 1
      for (int c = 0; c < DP; c += kColumns) {
        uint32_t o[kColumns / 32][32];
#pragma unroll
        for (int x = 0; x < kColumns / 32; ++x) tmem_ld_32x32(o_tmem + c + 32 * x, o[x]);
        tmem_ld_wait();
        // (pieces of a row change places so that eight lanes write to all banks)
#pragma unroll
        for (int e = 0; e < kPieces; ++e) {
          uint32_t word[4];
#pragma unroll
          for (int x = 0; x < 4; ++x)
            word[x] = pack2<T>(__uint_as_float(o[e >> 2][(e & 3) * 8 + 2 * x]) * inv, __uint_as_float(o[e >> 2][(e & 3) * 8 + 2 * x + 1]) * inv);
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(staged + lane * (kColumns * 2) + ((e ^ (lane * kPieces / 8 % kPieces)) << 4)),
                       "r"(word[0]), "r"(word[1]), "r"(word[2]), "r"(word[3]) : "memory");
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < kPieces; ++e) {
          const int r = e * (32 / kPieces) + own_row;
          const uint4 v = lds16(staged + r * (kColumns * 2) + ((piece ^ (r * kPieces / 8 % kPieces)) << 4));
          if (first_row + r < len && c + piece * 8 < p.dim) *reinterpret_cast<uint4*>(dst + e * next_rows + c * 2) = v;
        }
        __syncwarp();
      }
      tcgen05_fence_before();
    }
  }

  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0 && p.error_word) atomicExch(p.error_word, 1);
    // give copies and products still in flight time to end before their memory goes away
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// [T, heads, D] as a tensor of three dimensions, the one of token and head with the smaller stride first; boxes of one head,
// 128 tokens and 64 columns.  Heads that are one and the same in memory become one.
int head_map(CUtensorMap* map, int dtype, const HeadRows& r, int tokens, int heads, int dim, MapOrder* order) {
  if (r.head_stride == 0) heads = 1;
  const uint64_t token = tokens > 1 ? r.token_stride : 16, head = heads > 1 ? r.head_stride : 16;
  order->token_first = token < head;
  order->one_head = heads == 1;
  const bool first = order->token_first;
  const uint64_t dims[3] = {static_cast<uint64_t>(dim), static_cast<uint64_t>(first ? tokens : heads),
                            static_cast<uint64_t>(first ? heads : tokens)};
  const uint64_t strides[2] = {first ? token : head, first ? head : token};
  const uint32_t box[3] = {64, first ? static_cast<uint32_t>(kTile) : 1u, first ? 1u : static_cast<uint32_t>(kTile)};
  return encode_tensor_map_3d(map, dtype == 0 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, r.data, dims,
                              strides, box);
}

template <typename T, int DP>
int launch_prefill(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const PrefillParams& p, cudaStream_t st) {
  using C = Prefill<DP>;
  static thread_local int configured_device = -1;
  int device = 0;
  MP_CUDA_TRY(cudaGetDevice(&device));
  if (configured_device != device) {
    MP_CUDA_TRY(cudaFuncSetAttribute(prefill_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    configured_device = device;
  }
  const long long items = static_cast<long long>(p.slots) * p.per_slot;
  const int grid = static_cast<int>(items < kSmCount ? items : kSmCount);
  return launch_chained(prefill_kernel<T, DP>, dim3(grid), dim3(kThreads), C::kSmem, st, q, k, v, p);
}

}  // namespace
}  // namespace mp

extern "C" int mp_attention_prefill(int dtype, const mp_head_rows* q, const mp_head_rows* k, const mp_head_rows* v, int T,
                                    int Hq, int Hkv, int D, const void* cu_seqlens_i32, int B, float scale, void* out,
                                    int* index_word, int* error_word, mp_stream_t stream) {
  using namespace mp;
  HeadRows qr, kr, vr;
  int rc;
  if ((rc = check_head_rows(q, D, &qr)) || (rc = check_head_rows(k, D, &kr)) || (rc = check_head_rows(v, D, &vr))) return rc;
  if (!cu_seqlens_i32 || !out || T <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0) return MP_ERR_INVALID_ARG;
  if ((dtype != 0 && dtype != 1) || Hq % Hkv || Hq > 65535) return MP_ERR_UNSUPPORTED;
  if (T > 1 && (qr.token_stride == 0 || kr.token_stride == 0 || vr.token_stride == 0)) return MP_ERR_UNSUPPORTED;
  if (!aligned(out, 16)) return MP_ERR_ALIGNMENT;
  PrefillParams p{};
  p.cu_seqlens = static_cast<const int*>(cu_seqlens_i32);
  p.out = static_cast<char*>(out);
  p.index_word = index_word;
  p.error_word = error_word;
  p.tokens = T;
  p.batch = B;
  p.q_heads = Hq;
  p.group = Hq / Hkv;
  p.dim = D;
  p.pair_heads = p.group % 2 == 0;
  p.slots = T / (p.pair_heads ? kTile : 2 * kTile) + B;
  p.per_slot = p.pair_heads ? Hq / 2 : Hq;
  if (static_cast<long long>(p.slots) * p.per_slot > 0x7fff0000LL) return MP_ERR_UNSUPPORTED;
  // Masked scores, minus infinity, are multiplied too: a scale of 0 becomes the smallest number above it, with which no finite
  // score exceeds 2^-21.  A NaN stays one.
  const float size = fabsf(scale) * attn::kLog2e;
  p.scale_log2 = size == 0.0f ? std::numeric_limits<float>::denorm_min() : size;
  p.negate = scale < 0.0f ? 1u << 13 : 0u;
  CUtensorMap mq, mk, mv;
  if ((rc = head_map(&mq, dtype, qr, T, Hq, D, &p.q_order)) || (rc = head_map(&mk, dtype, kr, T, Hkv, D, &p.k_order)) ||
      (rc = head_map(&mv, dtype, vr, T, Hkv, D, &p.v_order)))
    return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (D <= 64) return dtype == 0 ? launch_prefill<__half, 64>(mq, mk, mv, p, st) : launch_prefill<__nv_bfloat16, 64>(mq, mk, mv, p, st);
  return dtype == 0 ? launch_prefill<__half, 128>(mq, mk, mv, p, st) : launch_prefill<__nv_bfloat16, 128>(mq, mk, mv, p, st);
}
