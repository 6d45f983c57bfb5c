// Position rotation of queries and keys, with keys and values appended to the paged cache, in one launch.
//
//   a' = a cos - b sin,   b' = b cos + a sin      for every pair (a, b) of a head's first `rotated` values
//
// in fp32, rounded once; the cosines and sines of a token's position come from the caller's table, so that scaled
// frequencies of any kind are the caller's.  Every value is read once and written once (keys twice where the caller wants
// them back): HBM bounds a prompt, the launch a decode step.  A thread takes both halves of its pairs, 16 bytes each, so no
// value is loaded twice and no exchange is needed; the table's rows are shared by all heads of a token and stay in L1.
#include "attention.cuh"

namespace mp {
namespace {

using namespace attn;

struct AppendParams {
  HeadRows q, k, v;
  CacheSide kc, vc;
  const float* table;
  const int* positions;
  const int* slots;
  char* q_out;
  char* k_out;                       // may be null
  int* index_word;                   // may be null
  int q_heads, kv_heads, head_bytes;
  int rotated, max_positions;
  int per_head, items;               // pieces of work of a rotated head, and of a token
  long long slot_count;
  FastDiv by_per_head, by_pieces, by_page;
};

// How a head's pairs lie: halves whose 16-byte pieces correspond; neighbours; halves that begin inside a piece.
enum { kHalves = 0, kNeighbours = 1, kOddHalves = 2 };
constexpr int kMostThreads = 256;

__device__ __forceinline__ uint4 load16(const char* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

template <typename T>
__device__ __forceinline__ void rotate_pieces(uint4& a, uint4& b, const float* cos, const float* sin) {
  uint32_t* pa = reinterpret_cast<uint32_t*>(&a);
  uint32_t* pb = reinterpret_cast<uint32_t*>(&b);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float4 c = __ldg(reinterpret_cast<const float4*>(cos) + h), s = __ldg(reinterpret_cast<const float4*>(sin) + h);
    const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 x = unpack2<T>(pa[2 * h + j]), y = unpack2<T>(pb[2 * h + j]);
      const float c0 = cs[2 * j], c1 = cs[2 * j + 1], s0 = sn[2 * j], s1 = sn[2 * j + 1];
      pa[2 * h + j] = pack2<T>(x.x * c0 - y.x * s0, x.y * c1 - y.y * s1);
      pb[2 * h + j] = pack2<T>(y.x * c0 + x.x * s0, y.y * c1 + x.y * s1);
    }
  }
}

// The piece at column `col` of a head whose pairs are neighbours, or whose halves do not begin at a piece.
template <typename T, int MODE>
__device__ __forceinline__ uint4 rotate_piece(uint4 raw, const char* head, int col, int rotated, const float* row) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&raw);
  const int half = rotated / 2;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = col + 2 * j;
    if (c >= rotated) break;
    const float2 x = unpack2<T>(w[j]);
    float out[2];
    if (MODE == kNeighbours) {
      const float cs = __ldg(row + c / 2), sn = __ldg(row + half + c / 2);
      out[0] = x.x * cs - x.y * sn;
      out[1] = x.y * cs + x.x * sn;
    } else {
      const T* values = reinterpret_cast<const T*>(head);
      const float own[2] = {x.x, x.y};
#pragma unroll
      for (int e = 0; e < 2; ++e) {      // a half may have an odd number of values: each value finds its own partner
        const int i = c + e, at = i < half ? i : i - half;
        const float other = static_cast<float>(values[i < half ? i + half : at]);
        const float cs = __ldg(row + at), sn = __ldg(row + half + at);
        out[e] = i < half ? own[e] * cs - other * sn : own[e] * cs + other * sn;
      }
    }
    w[j] = pack2<T>(out[0], out[1]);
  }
  return raw;
}

// Block (t, y): pieces of work blockDim y .. of token t: those of the q heads, the k heads, then the pieces of v.  The values
// are asked for before anything that hangs on the token's position and slot (one wait for memory, not two in a row: a prompt
// of 8192 tokens and 64 heads 68.6 us before).
template <typename T, int MODE>
__global__ void __launch_bounds__(kMostThreads, 2048 / kMostThreads) rotary_append_kernel(const AppendParams p) {
  chain_wait();
  chain_release();
  const int t = blockIdx.x, item = blockIdx.y * blockDim.x + threadIdx.x;
  if (item >= p.items) return;
  const int pos_there = __ldg(p.positions + t), slot = __ldg(p.slots + t);
  const int rotated_items = (p.q_heads + p.kv_heads) * p.per_head;
  const bool is_v = item >= rotated_items;
  const int i = is_v ? item - rotated_items : item;
  const int head = fast_div(i, is_v ? p.by_pieces : p.by_per_head), piece = i - head * (is_v ? static_cast<int>(p.by_pieces.d) : p.per_head);
  const bool is_q = !is_v && head < p.q_heads;
  const int own = is_q || is_v ? head : head - p.q_heads;
  const HeadRows& rows = is_v ? p.v : is_q ? p.q : p.k;
  const char* src = rows.data + static_cast<long long>(t) * rows.token_stride + own * rows.head_stride;
  const int pairs = p.rotated / 16;
  const bool turns = MODE == kHalves && !is_v && piece < pairs;             // both halves of eight pairs
  const int at = (MODE == kHalves && !is_v && piece >= pairs ? piece + pairs : piece) * 16;
  uint4 a = load16(src + at), b = make_uint4(0, 0, 0, 0);
  if (turns) b = load16(src + at + pairs * 16);

  const bool bad_pos = static_cast<unsigned>(pos_there) >= static_cast<unsigned>(p.max_positions);
  const bool bad = (slot >= 0 && bad_pos) || slot >= p.slot_count;
  if (bad && p.index_word && item == 0) *p.index_word = kBadIndex;
  const float* row = p.table + static_cast<long long>(bad_pos ? 0 : pos_there) * p.rotated;
  if (turns) rotate_pieces<T>(a, b, row + piece * 8, row + p.rotated / 2 + piece * 8);
  else if (MODE != kHalves && !is_v) a = rotate_piece<T, MODE>(a, src, piece * 8, p.rotated, row);
  auto put = [&](char* dst) {
    *reinterpret_cast<uint4*>(dst + at) = a;
    if (turns) *reinterpret_cast<uint4*>(dst + at + pairs * 16) = b;
  };
  char* out = is_v ? nullptr : is_q ? p.q_out : p.k_out;
  if (out) put(out + (static_cast<long long>(t) * (is_q ? p.q_heads : p.kv_heads) + own) * p.head_bytes);
  if (!is_q && slot >= 0 && !bad) {
    const CacheSide& side = is_v ? p.vc : p.kc;
    const int page = fast_div(slot, p.by_page), offset = slot - page * static_cast<int>(p.by_page.d);
    put(side.data + page * side.page_stride + own * side.head_stride + offset * side.token_stride);
  }
}

template <typename T>
int launch_append(const AppendParams& p, int mode, int tokens, cudaStream_t st) {
  // blocks of even size, so that few threads are idle
  const int blocks = (p.items + kMostThreads - 1) / kMostThreads, threads = ((p.items + blocks - 1) / blocks + 31) / 32 * 32;
  const dim3 grid(tokens, blocks), block(threads);
  switch (mode) {
    case kHalves: return launch_chained(rotary_append_kernel<T, kHalves>, grid, block, 0, st, p);
    case kNeighbours: return launch_chained(rotary_append_kernel<T, kNeighbours>, grid, block, 0, st, p);
    default: return launch_chained(rotary_append_kernel<T, kOddHalves>, grid, block, 0, st, p);
  }
}

}  // namespace

// ---- checks that the attention entries share
int check_head_rows(const mp_head_rows* r, int D, HeadRows* out) {
  if (!r || !r->data || D <= 0) return MP_ERR_INVALID_ARG;
  if (D % 8 || D > 128) return MP_ERR_UNSUPPORTED;
  if (r->token_stride < 0 || r->head_stride < 0) return MP_ERR_UNSUPPORTED;
  if (!aligned(r->data, 16) || r->token_stride % 8 || r->head_stride % 8) return MP_ERR_ALIGNMENT;
  *out = HeadRows{static_cast<const char*>(r->data), r->token_stride * 2, r->head_stride * 2};
  return MP_OK;
}

int check_cache(const mp_paged_cache* c, int D, CacheSide* k, CacheSide* v) {
  if (!c || !c->k || !c->v || c->pages <= 0 || c->kv_heads <= 0 || c->page_size <= 0 || D <= 0) return MP_ERR_INVALID_ARG;
  if (D % 8 || D > 128 || c->kv_heads > 65535) return MP_ERR_UNSUPPORTED;
  const long long strides[6] = {c->k_page_stride, c->k_head_stride, c->k_token_stride,
                                c->v_page_stride, c->v_head_stride, c->v_token_stride};
  for (long long s : strides) {
    if (s < 0) return MP_ERR_UNSUPPORTED;
    if (s % 8) return MP_ERR_ALIGNMENT;
  }
  if (!aligned(c->k, 16) || !aligned(c->v, 16)) return MP_ERR_ALIGNMENT;
  *k = CacheSide{static_cast<char*>(c->k), c->k_page_stride * 2, c->k_head_stride * 2, c->k_token_stride * 2};
  *v = CacheSide{static_cast<char*>(c->v), c->v_page_stride * 2, c->v_head_stride * 2, c->v_token_stride * 2};
  return MP_OK;
}

}  // namespace mp

extern "C" int mp_rotary_append_paged(int dtype, const mp_head_rows* q, const mp_head_rows* k, const mp_head_rows* v,
                                      const void* cos_sin_f32, int max_positions, int rotated, int interleaved,
                                      const void* positions_i32, const void* slots_i32, int T, int Hq, int D,
                                      const mp_paged_cache* cache, void* q_out, void* k_out, int* index_word,
                                      mp_stream_t stream) {
  using namespace mp;
  AppendParams p{};
  int rc;
  if ((rc = check_head_rows(q, D, &p.q)) || (rc = check_head_rows(k, D, &p.k)) || (rc = check_head_rows(v, D, &p.v)) ||
      (rc = check_cache(cache, D, &p.kc, &p.vc)))
    return rc;
  if (!positions_i32 || !slots_i32 || !q_out || !cos_sin_f32 || T <= 0 || Hq <= 0 || max_positions <= 0 || rotated <= 0)
    return MP_ERR_INVALID_ARG;
  if ((dtype != 0 && dtype != 1) || rotated > D || rotated % 2 || Hq > 65535) return MP_ERR_UNSUPPORTED;
  if (!aligned(q_out, 16) || !aligned(k_out, 16) || !aligned(cos_sin_f32, 16)) return MP_ERR_ALIGNMENT;
  const int mode = interleaved ? kNeighbours : rotated % 16 == 0 ? kHalves : kOddHalves;
  p.table = static_cast<const float*>(cos_sin_f32);
  p.positions = static_cast<const int*>(positions_i32);
  p.slots = static_cast<const int*>(slots_i32);
  p.q_out = static_cast<char*>(q_out);
  p.k_out = static_cast<char*>(k_out);
  p.index_word = index_word;
  p.q_heads = Hq;
  p.kv_heads = cache->kv_heads;
  p.head_bytes = D * 2;
  p.rotated = rotated;
  p.max_positions = max_positions;
  p.per_head = mode == kHalves ? D / 8 - rotated / 16 : D / 8;
  p.items = (Hq + p.kv_heads) * p.per_head + p.kv_heads * (D / 8);
  p.slot_count = static_cast<long long>(cache->pages) * cache->page_size;
  p.by_per_head = make_fast_div(p.per_head);
  p.by_pieces = make_fast_div(D / 8);
  p.by_page = make_fast_div(cache->page_size);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == 0 ? launch_append<__half>(p, mode, T, st) : launch_append<__nv_bfloat16>(p, mode, T, st);
}
