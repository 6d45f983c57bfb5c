// Attention of one new token per sequence over a paged cache of keys and values.
//
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   s_j = scale q . k_j,   m = max_j s_j
//
// with a running m, sum and o, in one pass over the cache: 2 len Hkv D 16-bit values per sequence, which HBM bounds.  The
// query heads that share a head of keys are the rows of a 16-row matrix product, so keys and values are read once for all
// of them (mma.sync: at HBM's rate an SM multiplies one 16 x 16 piece of the cache in about 10 clocks, far below what even
// this path of the tensor cores takes; tcgen05's 128 rows would be 7/8 padding or more).
//
// All lengths are known on the device only (a captured launch serves every later step), so the work is cut there: the
// sequence of (sequence, head) pairs, each in steps of a few keys, is cut evenly over the blocks, two to an SM.  A warp is a
// stream of its own: it copies its tiles of keys and values to its part of shared memory, several ahead, also across the ends
// of sequences, and keeps its own maximum, sum and output until the block joins its four warps.  Where a sequence spans
// blocks they leave (m, sum, o) in the workspace, and the one that arrives last joins them in the blocks' order, so results
// do not depend on which one that was.
#include "attention.cuh"

namespace mp {
namespace {

using namespace attn;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStages = 3;
constexpr int kBlocksPerSm = 2;
constexpr int kMaxGrid = kSmCount * kBlocksPerSm;
constexpr int kRows = 16;                                     // query heads per tile
constexpr int kMaxD = 128;
// Steps that a block takes at least, before more blocks share a short cache.
constexpr int kMinSteps = 1;

// A block's two parts of sequences that it shares: the one it begins within (0) and the one it ends within (1).
struct PartialTile {
  float m[kRows], sum[kRows];
  float o[kRows][kMaxD];
};
constexpr size_t kCounterBytes = 4096;
static_assert(kMaxGrid * sizeof(int) <= kCounterBytes, "");
constexpr size_t kWorkspaceBytes = kCounterBytes + sizeof(PartialTile) * kMaxGrid * 2;

struct DecodeParams {
  HeadRows q;
  CacheSide kc, vc;
  const int* page_table;
  const int* seq_lens;
  char* out;
  int* counters;               // one per block: arrivals at the sequence that the block ends within
  PartialTile* partials;
  int* index_word;
  int batch, q_heads, kv_heads, dim;
  int group, row_tiles;        // query heads per head of keys, tiles of rows they take
  int table_pages, pages;
  long long capacity;          // tokens that a row of the table has room for
  float scale_log2;
  FastDiv by_page;
};

// DP: head size rounded up.  HALF: at most eight rows are in use.
template <typename T, int DP, bool HALF>
struct Decode {
  static constexpr int kKeys = DP <= 64 ? 32 : 16;            // keys per warp and tile: 8 KB of keys and values
  static constexpr int kStepKeys = kKeys * kWarps;
  static constexpr int kPieces = DP / 8;                      // of 16 bytes per row
  static constexpr int kSideBytes = kKeys * DP * 2;
  static constexpr int kTileBytes = 2 * kSideBytes;
  static constexpr int kRingBytes = kWarps * kStages * kTileBytes;
  static constexpr int kJoinBytes = kWarps * 8 * DP * 4;      // eight rows of every warp's output
  static constexpr int kSmem = kRingBytes + kJoinBytes;
};

struct Item {          // a sequence, a head of keys and a tile of its query heads
  int seq, head, row_tile, len;
};

template <typename T, int DP, bool HALF>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) paged_decode_kernel(const DecodeParams p) {
  using C = Decode<T, DP, HALF>;
  extern __shared__ __align__(128) char smem[];
  __shared__ float s_m[kWarps][kRows], s_sum[kWarps][kRows];
  __shared__ int s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  chain_wait();
  chain_release();

  // ---- this block's run of steps.  Every warp adds up the lengths, 1/32 of them to a lane.
  auto length_of = [&](int seq) {
    int n = __ldg(p.seq_lens + seq);
    if (n < 0 || n > p.capacity) {
      if (p.index_word) *p.index_word = kBadIndex;
      n = n < 0 ? 0 : static_cast<int>(p.capacity);
    }
    return n;
  };
  auto steps_of = [&](int len) { return max(1, (len + C::kStepKeys - 1) / C::kStepKeys); };
  const int heads = p.kv_heads * p.row_tiles;                 // items of a sequence
  const int slice = (p.batch + 31) / 32, lo = min(lane * slice, p.batch), hi = min(lo + slice, p.batch);
  long long mine = 0;
  for (int s = lo; s < hi; ++s) mine += steps_of(length_of(s));
  long long before = mine;                                    // of this lane's slice and those in front of it
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long other = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += other;
  }
  const long long total = __shfl_sync(0xffffffffu, before, 31) * heads;
  const long long wanted = (total + kMinSteps - 1) / kMinSteps;
  const long long grid = wanted < gridDim.x ? wanted : gridDim.x;
  if (blockIdx.x >= grid) return;
  long long at = total * blockIdx.x / grid;
  const long long end = total * (blockIdx.x + 1) / grid;

  // the item that step `at` is in, and its first step
  Item item;
  long long item_begin;
  {
    const bool here = before * heads > at;
    const int who = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    long long base = before - mine;
    int s = lo;
    if (lane == who) {
      while ((base + steps_of(length_of(s))) * heads <= at) base += steps_of(length_of(s++));
    }
    base = __shfl_sync(0xffffffffu, base, who);
    s = __shfl_sync(0xffffffffu, s, who);
    item.seq = s;
    item.len = length_of(s);
    const int h = static_cast<int>((at - base * heads) / steps_of(item.len));
    item.head = h / p.row_tiles;
    item.row_tile = h - item.head * p.row_tiles;
    item_begin = base * heads + static_cast<long long>(h) * steps_of(item.len);
  }
  auto next_item = [&](Item& it) {
    if (++it.row_tile < p.row_tiles) return;
    it.row_tile = 0;
    if (++it.head < p.kv_heads) return;
    it.head = 0;
    if (++it.seq < p.batch) it.len = length_of(it.seq);
  };

  // ---- copies: this warp's tile of a step, lanes 0-15 know the keys' rows and lanes 16-31 the values' (two each at D <= 64)
  const uint32_t ring = tc::smem_u32(smem) + warp * (kStages * C::kTileBytes);
  Item load_item = item;
  long long load_at = at, load_begin = item_begin;
  int load_stage = 0;
  auto issue = [&]() {
    if (load_at < end) {
      const int key0 = (static_cast<int>(load_at - load_begin) * kWarps + warp) * C::kKeys;
      constexpr int kPer = C::kKeys / 16;
      const CacheSide& side = lane < 16 ? p.kc : p.vc;
      const char* base[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int key = key0 + i * 16 + (lane & 15);
        base[i] = nullptr;
        if (key < load_item.len) {
          const int slot = fast_div(key, p.by_page), offset = key - slot * static_cast<int>(p.by_page.d);
          const int page = __ldg(p.page_table + static_cast<long long>(load_item.seq) * p.table_pages + slot);
          if (page < 0 || page >= p.pages) {
            if (p.index_word) *p.index_word = kBadIndex;
          } else {
            base[i] = side.data + page * side.page_stride + load_item.head * side.head_stride + offset * side.token_stride;
          }
        }
      }
      const uint32_t dst = ring + load_stage * C::kTileBytes;
      // 32 pieces per instruction: rows of 16, 12 or 8 pieces
      constexpr int kCopies = C::kKeys * C::kPieces / 32;
#pragma unroll
      for (int sidx = 0; sidx < 2; ++sidx) {
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
          const int i = c * 32 + lane, row = i / C::kPieces, piece = i - row * C::kPieces;
          const int from = sidx * 16 + (row & 15);
          unsigned long long src = 0;
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const unsigned long long v = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(base[j]), from);
            if (j == row / 16) src = v;
          }
          const bool valid = src != 0 && piece * 8 < p.dim;
          copy16_async(dst + sidx * C::kSideBytes + piece_at<DP>(row, piece),
                       valid ? reinterpret_cast<const char*>(src) + piece * 16 : p.kc.data, valid);
        }
      }
      if (++load_stage == kStages) load_stage = 0;
      ++load_at;
      if (load_at - load_begin == steps_of(load_item.len)) {
        load_begin = load_at;
        next_item(load_item);
      }
    }
    copies_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue();

  constexpr int kNT = DP / 8;                                  // 8-column tiles of the output
  constexpr int kHalves = HALF ? 1 : 2;                        // rows lane / 4 and lane / 4 + 8
  int stage = 0;
  const int row0 = lane >> 2, col0 = (lane & 3) * 2;
  while (at < end) {
    // ---- one item, or this block's part of it
    const long long item_end = item_begin + steps_of(item.len);
    const int steps = static_cast<int>((item_end < end ? item_end : end) - at);
    const int row_base = item.head * p.group + item.row_tile * kRows;       // query head of row 0
    const int rows = min(kRows, p.group - item.row_tile * kRows);
    uint32_t qf[DP / 16][4];
    {
      const char* q = p.q.data + item.seq * p.q.token_stride + row_base * p.q.head_stride;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = row0 + (j & 1) * 8, c = k * 16 + col0 + (j >> 1) * 8;
          qf[k][j] = (HALF && (j & 1)) || r >= rows || c >= p.dim
                         ? 0u : __ldg(reinterpret_cast<const unsigned int*>(q + r * p.q.head_stride + c * 2));
        }
    }
    float o[kNT][4];
#pragma unroll
    for (int n = 0; n < kNT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    float m[2] = {kNegInf, kNegInf}, sum[2] = {0.0f, 0.0f};

    int key0 = (static_cast<int>(at - item_begin) * kWarps + warp) * C::kKeys;
    for (int step = 0; step < steps; ++step, key0 += C::kStepKeys) {
      issue();
      copies_wait<kStages - 1>();
      __syncwarp();
      const uint32_t tile_k = ring + stage * C::kTileBytes, tile_v = tile_k + C::kSideBytes;
      if (++stage == kStages) stage = 0;
      if (key0 < item.len) {
        constexpr int kST = C::kKeys / 8;
        float s[kST][4];
#pragma unroll
        for (int n = 0; n < kST; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
          for (int n = 0; n < kST / 2; ++n) {
            uint32_t b[4];
            ldmatrix_x4(b, tile_k + piece_at<DP>(n * 16 + (lane & 7) + (lane >> 4) * 8, k * 2 + ((lane >> 3) & 1)));
            mma_16816<T>(s[2 * n], qf[k], b[0], b[1]);
            mma_16816<T>(s[2 * n + 1], qf[k], b[2], b[3]);
          }
        const int left = item.len - key0;
        float keep[2] = {1.0f, 1.0f}, base[2];
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          float top = kNegInf;
#pragma unroll
          for (int n = 0; n < kST; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float& v = s[n][2 * h + j];
              v = n * 8 + col0 + j < left ? v * p.scale_log2 : kNegInf;
              top = fmaxf(top, v);
            }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float now = fmaxf(m[h], top);
          base[h] = now == kNegInf ? 0.0f : now;         // nothing but minus infinity yet: no difference of infinities
          keep[h] = exp2_fast(m[h] - base[h]);
          m[h] = now;
          sum[h] *= keep[h];
        }
        uint32_t pf[kST / 2][4];
#pragma unroll
        for (int n = 0; n < kST; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h < kHalves) {
              const float e0 = exp2_fast(s[n][2 * h] - base[h]), e1 = exp2_fast(s[n][2 * h + 1] - base[h]);
              sum[h] += e0 + e1;
              pf[n >> 1][(n & 1) * 2 + h] = pack2<T>(e0, e1);
            } else {
              pf[n >> 1][(n & 1) * 2 + h] = 0u;
            }
          }
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            o[n][2 * h] *= keep[h];
            o[n][2 * h + 1] *= keep[h];
          }
#pragma unroll
        for (int k = 0; k < kST / 2; ++k)
#pragma unroll
          for (int n = 0; n < kNT / 2; ++n) {
            uint32_t b[4];
            ldmatrix_x4_trans(b, tile_v + piece_at<DP>(k * 16 + (lane & 15), n * 2 + (lane >> 4)));
            mma_16816<T>(o[2 * n], pf[k], b[0], b[1]);
            mma_16816<T>(o[2 * n + 1], pf[k], b[2], b[3]);
          }
      }
      __syncwarp();            // the next copies overwrite this tile
    }

    // ---- the block's four warps
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
      sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
      if ((lane & 3) == 0) {
        s_m[warp][row0 + 8 * h] = m[h];
        s_sum[warp][row0 + 8 * h] = sum[h];
      }
    }
    __syncthreads();
    const bool whole = at == item_begin && item_end <= end;
    PartialTile* part = p.partials + (blockIdx.x * 2 + (at == item_begin ? 1 : 0));
    float* join = reinterpret_cast<float*>(smem + C::kRingBytes);
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      float top = kNegInf;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][row0 + 8 * h]);
      const float scale = exp2_fast(m[h] - (top == kNegInf ? 0.0f : top));
#pragma unroll
      for (int n = 0; n < kNT; ++n)
        *reinterpret_cast<float2*>(join + (warp * 8 + row0) * DP + n * 8 + col0) = make_float2(o[n][2 * h] * scale, o[n][2 * h + 1] * scale);
      __syncthreads();
      for (int i = threadIdx.x; i < 8 * DP / 4; i += kThreads) {
        const int r = i / (DP / 4), c = (i - r * (DP / 4)) * 4, row = r + 8 * h;
        if (row >= rows) break;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float row_top = kNegInf, row_sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) row_top = fmaxf(row_top, s_m[w][row]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 x = *reinterpret_cast<const float4*>(join + (w * 8 + r) * DP + c);
          acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
          row_sum += s_sum[w][row] * exp2_fast(s_m[w][row] - (row_top == kNegInf ? 0.0f : row_top));
        }
        if (whole) {
          if (c < p.dim) {
            const float inv = row_sum == 0.0f ? 0.0f : 1.0f / row_sum;
            char* dst = p.out + ((static_cast<long long>(item.seq) * p.q_heads + row_base + row) * p.dim + c) * 2;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
          }
        } else {
          __stcg(reinterpret_cast<float4*>(&part->o[row][c]), acc);
          if (c == 0) {
            __stcg(&part->m[row], row_top);
            __stcg(&part->sum[row], row_sum);
          }
        }
      }
      __syncthreads();
    }

    // ---- a sequence that spans blocks: whoever arrives last joins the parts
    if (!whole) {
      const long long last_step = item_end - 1;
      const int first = static_cast<int>(((item_begin + 1) * grid - 1) / total);
      const int last = static_cast<int>(((last_step + 1) * grid - 1) / total);
      if (threadIdx.x == 0) {
        __threadfence();
        const int n = atomicAdd(p.counters + first, 1);
        s_last = n == last - first;
        if (s_last) p.counters[first] = 0;
        __threadfence();
      }
      __syncthreads();
      if (s_last) {
        for (int i = threadIdx.x; i < rows * (DP / 4); i += kThreads) {
          const int row = i / (DP / 4), c = (i - row * (DP / 4)) * 4;
          if (c >= p.dim) continue;
          float top = kNegInf;
          for (int b = first; b <= last; ++b) top = fmaxf(top, __ldcg(&p.partials[b * 2 + (b == first)].m[row]));
          const float ref = top == kNegInf ? 0.0f : top;
          float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          float row_sum = 0.0f;
          for (int b = first; b <= last; ++b) {
            const PartialTile& t = p.partials[b * 2 + (b == first)];
            const float f = exp2_fast(__ldcg(&t.m[row]) - ref);
            const float4 x = __ldcg(reinterpret_cast<const float4*>(&t.o[row][c]));
            row_sum += __ldcg(&t.sum[row]) * f;
            acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
          }
          const float inv = row_sum == 0.0f ? 0.0f : 1.0f / row_sum;
          char* dst = p.out + ((static_cast<long long>(item.seq) * p.q_heads + row_base + row) * p.dim + c) * 2;
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
        }
      }
      __syncthreads();
    }
    at += steps;
    item_begin = item_end;
    next_item(item);
  }
  copies_wait<0>();
}

template <typename T, int DP, bool HALF>
int launch_decode(const DecodeParams& p, int grid, cudaStream_t st) {
  using C = Decode<T, DP, HALF>;
  static thread_local int configured_device = -1;
  int device = 0;
  MP_CUDA_TRY(cudaGetDevice(&device));
  if (configured_device != device) {
    MP_CUDA_TRY(cudaFuncSetAttribute(paged_decode_kernel<T, DP, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    configured_device = device;
  }
  return launch_chained(paged_decode_kernel<T, DP, HALF>, dim3(grid), dim3(kThreads), C::kSmem, st, p);
}

template <typename T>
int dispatch_decode(const DecodeParams& p, int grid, cudaStream_t st) {
  const bool half = p.group <= 8;
  if (p.dim <= 64) return half ? launch_decode<T, 64, true>(p, grid, st) : launch_decode<T, 64, false>(p, grid, st);
  if (p.dim <= 96) return half ? launch_decode<T, 96, true>(p, grid, st) : launch_decode<T, 96, false>(p, grid, st);
  return half ? launch_decode<T, 128, true>(p, grid, st) : launch_decode<T, 128, false>(p, grid, st);
}

}  // namespace
}  // namespace mp

extern "C" size_t mp_paged_attention_decode_workspace_bytes(void) { return mp::kWorkspaceBytes; }

extern "C" int mp_paged_attention_decode(int dtype, const mp_head_rows* q, int B, int Hq, int D, const mp_paged_cache* cache,
                                         const void* page_table_i32, int table_pages, const void* seq_lens_i32, float scale,
                                         void* out, void* workspace, size_t workspace_bytes, int* index_word,
                                         mp_stream_t stream) {
  using namespace mp;
  DecodeParams p{};
  int rc;
  if ((rc = check_head_rows(q, D, &p.q)) || (rc = check_cache(cache, D, &p.kc, &p.vc))) return rc;
  if (!page_table_i32 || !seq_lens_i32 || !out || B <= 0 || Hq <= 0 || table_pages <= 0) return MP_ERR_INVALID_ARG;
  if ((dtype != 0 && dtype != 1) || Hq % cache->kv_heads || Hq > 65535) return MP_ERR_UNSUPPORTED;
  if (!aligned(out, 16) || !aligned(workspace, 16)) return MP_ERR_ALIGNMENT;
  if (!workspace || workspace_bytes < kWorkspaceBytes) return MP_ERR_WORKSPACE;
  p.page_table = static_cast<const int*>(page_table_i32);
  p.seq_lens = static_cast<const int*>(seq_lens_i32);
  p.out = static_cast<char*>(out);
  p.counters = static_cast<int*>(workspace);
  p.partials = reinterpret_cast<PartialTile*>(static_cast<char*>(workspace) + kCounterBytes);
  p.index_word = index_word;
  p.batch = B;
  p.q_heads = Hq;
  p.kv_heads = cache->kv_heads;
  p.dim = D;
  p.group = Hq / cache->kv_heads;
  p.row_tiles = (p.group + kRows - 1) / kRows;
  p.table_pages = table_pages;
  p.pages = cache->pages;
  const long long room = static_cast<long long>(table_pages) * cache->page_size;
  p.capacity = room < 0x7fffff00LL ? room : 0x7fffff00LL;
  p.scale_log2 = scale * attn::kLog2e;
  p.by_page = make_fast_div(cache->page_size);
  // no more blocks than there can be steps
  const int step = D <= 64 ? Decode<__half, 64, true>::kStepKeys : Decode<__half, 128, true>::kStepKeys;
  const long long steps = static_cast<long long>(B) * p.kv_heads * p.row_tiles * ((p.capacity + step - 1) / step);
  const int grid = static_cast<int>(steps < kMaxGrid ? steps : kMaxGrid);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == 0 ? dispatch_decode<__half>(p, grid, st) : dispatch_decode<__nv_bfloat16>(p, grid, st);
}
