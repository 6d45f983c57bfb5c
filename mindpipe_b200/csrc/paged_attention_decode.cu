// Attention of one new token per sequence over a paged cache of keys and values.
//
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   s_j = scale q . k_j,   m = max_j s_j
//
// with a running m, sum and o, in one pass over the cache: 2 len Hkv D 16-bit values per sequence, which HBM bounds.  The
// query heads that share a head of keys are the columns, eight or sixteen, of the products S^T = K Q^T and O^T = V^T P^T, so
// keys and values are read once for all of them (once for every sixteen, where there are more; mma.sync: at HBM's rate an SM multiplies one 16 x 16 piece of the cache in about 10
// clocks, far below what even this path of the tensor cores takes; tcgen05's 128 rows would be 7/8 padding or more).
//
// All lengths are known on the device only (a captured launch serves every later step), so the work is cut there: the list of
// (sequence, head) items, each in steps of a few keys, is cut evenly over teams of four warps, two teams to an SM, so that
// one copies while the other joins.  A warp is a stream of its own: it copies its tiles of keys and values to its part of
// shared memory (cp.async: a lane's 16 bytes go where ldmatrix finds them without conflicts, and what is not to be read
// becomes zero; TMA's boxes of 128 bytes a row came at 6.0 TB/s where these come at 6.4), several ahead, also across the
// ends of sequences, and it keeps its own maximum, sum and output until the team joins at the item's end.  The warps of a
// team take neighbouring tiles (with a run of tiles for each warp, and no joins but at the run's ends, the cache's rate fell
// from 6.4 to 5.7 TB/s).  Where an item spans teams they
// leave (m, sum, o) in the workspace, and the one that arrives last joins them in the teams' order, so results do not depend
// on which one that was.  Of short sequences, where there are many, a team's warps take an item each, four heads at a time, and
// need not join (301 sequences of 1 to 700 tokens and five heads: 25 us with four warps to every item).
//
// What runs once a launch runs from cold instruction caches, some ten clocks an instruction, and a step's worth of keys is
// 1.5 us: the code in front of the first tile and at an item's end is kept short.
#include "attention.cuh"

namespace mp {
namespace {

using namespace attn;

constexpr int kStages = 3;
constexpr int kRows = 16;                                     // query heads per tile
constexpr int kItemCost = 2;           // what an item costs beside its steps, in steps
// Steps up to which an item is not cut: a join of teams takes 2-3 us.  (Sequences of 300 tokens and eight heads, with 1, 4, 8:
// 16 of them, 3 steps an item, 13.9, 8.4, 8.4 us; 19, 5 steps, 13.0, 13.0, 10.5; 64 21.9, 21.9, 19.1; 64 of 75 to 425
// tokens 20.8, 21.0, 21.7; no difference from 2000 tokens on.)
constexpr int kWholeSteps = 4;
// Weights are 2^(s - m + lift), rounded to the type before the product with V, since that is what the tensor cores multiply
// (results are off by 2.6e-4 of their norm in fp16 and 2.3e-3 in bf16, with 32-bit weights 2.1e-4 and 1.7e-3).  fp16 has no more than 24 bits below 1, and many
// weights beneath those would be lost together; multiplied by 2^15 they keep all their bits down to 2^-29.
template <typename T> constexpr float kLift = __is_same(T, __half) ? 15.0f : 0.0f;
// Tiles of a sequence up to which a warp takes an item alone, if there are many items.  (301 sequences with five heads, of 60,
// 130, 250 tokens on average, with 4, 8, 16 tiles: 15.2, 14.6, 14.6 us; 19.3, 21.5, 23.9; 27.8, 27.5, 33.4.  256 with eight
// heads, of 100 tokens: 31.3, 30.1, 29.0.)
constexpr int kSoloTiles = 8;

// A team's two parts of items that it shares: the one it begins within (0) and the one it ends within (1).
template <int DP>
struct PartialTile {
  float m[kRows], sum[kRows];
  float o[kRows][DP];
};
template <int DP> constexpr int kWarpsOf = DP == 64 ? 16 : 8; // of a block, one block to an SM
constexpr int kFour = 4;                                      // warps of a team where there are more items than blocks
constexpr size_t kCounterBytes = 4096;
static_assert(kSmCount * kWarpsOf<64> / kFour * sizeof(int) <= kCounterBytes, "");
template <int DP> constexpr size_t kPartialBytes = sizeof(PartialTile<DP>) * kSmCount * kWarpsOf<DP> / kFour * 2;
constexpr size_t kWorkspaceBytes = kCounterBytes + (kPartialBytes<64> > kPartialBytes<128> ? kPartialBytes<64> : kPartialBytes<128>);

struct DecodeParams {
  HeadRows q;
  CacheSide kc, vc;
  const int* page_table;
  const int* seq_lens;
  char* out;
  int* counters;               // one per team: arrivals at the item that the team ends within
  void* partials;
  int* index_word;
  int batch, q_heads, kv_heads, dim;
  int group, row_tiles, items;         // query heads per head of keys, tiles of rows they take, items of a sequence
  int solo_tiles;                      // tiles up to which a warp takes an item of a sequence alone
  int table_pages, pages;
  int capacity;                        // tokens that a row of the table has room for
  float scale_log2;
  FastDiv by_page;
};

// DP: head size rounded up.  HALF: at most eight rows are in use.  EIGHTS: pages of a multiple of eight tokens.  WHOLE: the
// block is one team.
template <typename T, int DP, bool HALF, bool EIGHTS, bool WHOLE>
struct Decode {
  static constexpr int kTeamWarps = WHOLE ? kWarpsOf<DP> : kFour, kTeam = 32 * kTeamWarps;
  static constexpr int kTeams = kWarpsOf<DP> / kTeamWarps, kThreads = kTeam * kTeams;
  static constexpr int kBoxes = DP / 64;                      // of 64 columns, rows of 128 bytes
  static constexpr int kKeys = 16;                            // per tile: 8 KB of keys and values, or 4
  static constexpr int kSideBytes = kKeys * 128 * kBoxes;
  static constexpr int kTileBytes = 2 * kSideBytes;
  static constexpr int kRingBytes = kTeamWarps * kTeams * kStages * kTileBytes;
  // eight rows of every warp's output, maximum and sum; rows four banks apart, so that a warp's stores meet no conflict
  static constexpr int kJoinRow = DP + 4;
  static constexpr int kJoinBytes = kTeamWarps * 8 * kJoinRow * 4;
  static constexpr int kSmem = kRingBytes + kTeams * kJoinBytes;
};

// An item, or four whose warps take one each, and the steps of it that are in turn.
struct Cursor {
  int seq, unit, len, step, stop;      // stop < 0: the run is over
  bool solo;
};
// Runs of a list of n units over `count` takers: the first n % count have one more.
struct Cut {
  unsigned each, more;
  __device__ __forceinline__ Cut(unsigned n, unsigned count) : each(n / count), more(n - n / count * count) {}
  __device__ __forceinline__ unsigned begin(unsigned i) const { return i * each + min(i, more); }
  __device__ __forceinline__ unsigned taker(unsigned at) const {
    const unsigned low = more * (each + 1);
    return at < low ? at / (each + 1) : more + (at - low) / each;
  }
};

// An 8 x 8 matrix of 16-bit values, two of a row to a lane, with rows and columns exchanged.
__device__ __forceinline__ uint32_t transpose(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <typename T, int DP, bool HALF, bool EIGHTS, bool WHOLE>
__global__ void __launch_bounds__(Decode<T, DP, HALF, EIGHTS, WHOLE>::kThreads, 1) paged_decode_kernel(const DecodeParams p) {
  using C = Decode<T, DP, HALF, EIGHTS, WHOLE>;
  constexpr int kTeams = C::kTeams, kThreads = C::kThreads, kTeamWarps = C::kTeamWarps, kTeam = C::kTeam;
  using Partial = PartialTile<DP>;
  Partial* const partials = static_cast<Partial*>(p.partials);
  extern __shared__ __align__(128) char smem[];
  __shared__ unsigned s_warp[kThreads / 32];
  __shared__ int s_place[kTeams][2][3];        // of a team: where its run begins and ends -- sequence, item, step
  __shared__ int s_last[kTeams];
  unsigned* s_scan = reinterpret_cast<unsigned*>(smem + C::kRingBytes);       // (where joins are, later)
  const int warp = tc::uniform_warp(), lane = threadIdx.x & 31, team = warp / kTeamWarps, member = warp % kTeamWarps;
  // the runs of the list go to the blocks' first teams, then to their second ones
  const int runs = gridDim.x * kTeams, run = blockIdx.x + team * gridDim.x;
  chain_wait();
  chain_release();

  // ---- the list's length and where runs begin.  A thread has a slice of the batch.
  auto length_of = [&](int seq) {
    int n = __ldg(p.seq_lens + seq);
    if (static_cast<unsigned>(n) > static_cast<unsigned>(p.capacity)) {
      if (p.index_word) *p.index_word = kBadIndex;
      n = n < 0 ? 0 : p.capacity;
    }
    return n;
  };
  auto tiles_of = [&](int len) { return max(1, (len + C::kKeys - 1) / C::kKeys); };
  auto is_solo = [&](int tiles) { return tiles <= p.solo_tiles; };
  auto steps_of = [&](int tiles) { return is_solo(tiles) ? tiles : (tiles + kTeamWarps - 1) / kTeamWarps; };
  auto units_of = [&](int tiles) { return is_solo(tiles) ? (p.items + kTeamWarps - 1) / kTeamWarps : p.items; };
  const int slice = (p.batch + kThreads - 1) / kThreads;
  unsigned sum_cost = 0;
  float about = 0.0f;
#pragma unroll 1
  for (int s = threadIdx.x * slice, n = 0; n < slice && s < p.batch; ++s, ++n) {
    const int tiles = tiles_of(length_of(s));
    sum_cost += static_cast<unsigned>(steps_of(tiles) + kItemCost) * units_of(tiles);
    about += static_cast<float>(steps_of(tiles) + kItemCost) * static_cast<float>(units_of(tiles));
  }
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned other = __shfl_up_sync(0xffffffffu, sum_cost, d);
    if (lane >= d) sum_cost += other;
  }
  s_scan[threadIdx.x] = sum_cost;
  if (lane == 31) s_warp[warp] = sum_cost;
  // Sums have 32 bits: a slice with 2^23 steps over all its items is refused, and nothing is written.  With teams of four that
  // is half a billion tokens times items: 67 million tokens of eight heads of keys (137 GB of them with 128 values).
  if (__syncthreads_or(about > 8388607.0f)) {
    if (p.index_word) *p.index_word = kBadIndex;
    return;
  }
  unsigned total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) total += s_warp[w];
  const Cut cut(total, runs);
  if (member == 0 && lane < 2) {
    unsigned rest = cut.begin(run + lane);
    const bool behind = rest >= total;                         // behind the last item
    if (behind) rest = total - 1;
    int w = 0;
    while (rest >= s_warp[w]) rest -= s_warp[w++];
    int t = 0;                                                 // the first thread of the warp whose sum is above `rest`
#pragma unroll
    for (int d = 16; d; d >>= 1)
      if (s_scan[w * 32 + t + d - 1] <= rest) t += d;
    if (t) rest -= s_scan[w * 32 + t - 1];
    int seq = (w * 32 + t) * slice;
    unsigned cost;
    int tiles;
    for (;; ++seq) {
      tiles = tiles_of(length_of(seq));
      cost = steps_of(tiles) + kItemCost;
      if (rest < cost * units_of(tiles)) break;
      rest -= cost * units_of(tiles);
    }
    int unit = static_cast<int>(rest / cost), step = 0;
    rest -= unit * cost;
    if (behind) ++unit;
    else if (!is_solo(tiles) && cost > kWholeSteps + kItemCost) step = max(0, static_cast<int>(rest) - kItemCost);
    else if (2 * rest >= cost) ++unit;                         // the place moves to where an item begins
    s_place[team][lane][0] = seq;
    s_place[team][lane][1] = unit;
    s_place[team][lane][2] = step;
  }
  __syncthreads();
  const int end_seq = s_place[team][1][0], end_unit = s_place[team][1][1], end_step = s_place[team][1][2];

  // from the place the cursor is at to what is there, or next
  auto settle = [&](Cursor& c) {
    c.stop = -1;
#pragma unroll 1
    while (c.seq <= end_seq && c.seq < p.batch) {
      c.len = length_of(c.seq);
      const int tiles = tiles_of(c.len);
      if (c.unit < units_of(tiles)) {
        if (c.seq == end_seq && c.unit > end_unit) return;
        const int stop = c.seq == end_seq && c.unit == end_unit ? end_step : steps_of(tiles);
        if (c.step < stop) c.stop = stop;
        c.solo = is_solo(tiles);
        return;
      }
      c.unit = 0;
      ++c.seq;
    }
  };
  auto advance = [&](Cursor& c) {
    ++c.unit;
    c.step = 0;
    settle(c);
  };
  auto item_of = [&](const Cursor& c) { return c.solo ? c.unit * kTeamWarps + member : c.unit; };       // p.items or more: none
  auto tile_of = [&](const Cursor& c) { return c.solo ? c.step : c.step * kTeamWarps + member; };
  auto keys_of = [&](const Cursor& c) { return item_of(c) < p.items ? min(C::kKeys, c.len - tile_of(c) * C::kKeys) : 0; };
  auto head_of = [&](int item) { return p.row_tiles == 1 ? item : item / p.row_tiles; };
  Cursor next{s_place[team][0][0], s_place[team][0][1], 0, s_place[team][0][2], -1, false};
  settle(next);

  // ---- copies of this warp's next tile
  const uint32_t ring = tc::smem_u32(smem) + warp * (kStages * C::kTileBytes);
  Cursor load = next;
  int load_stage = 0;
  // A tile that is to be copied: looks at the page table take as long as a copy, so they are made two turns ahead.
  struct Ahead {
    int seq, head, key0, keys;                 // keys < 0: there is none
    int page, offset;                          // EIGHTS: of this lane's eight rows
  };
  auto look_up = [&]() {
    Ahead t;
    t.keys = -1;
    if (load.stop < 0) return t;
    t.seq = load.seq;
    t.head = head_of(item_of(load));
    t.key0 = tile_of(load) * C::kKeys;
    t.keys = max(keys_of(load), 0);
    t.page = t.offset = 0;
    if (EIGHTS && lane * 8 < t.keys) {
      const int key = t.key0 + lane * 8, slot = fast_div(key, p.by_page);
      t.offset = key - slot * static_cast<int>(p.by_page.d);
      t.page = __ldg(p.page_table + static_cast<long long>(t.seq) * p.table_pages + slot);
    }
    if (++load.step >= load.stop) advance(load);
    return t;
  };
  Ahead first_up = look_up(), second_up = look_up();
  constexpr int kPieces = C::kBoxes * 8, kRowsPerCopy = 32 / kPieces;        // of 16 bytes to a row; rows that a warp copies at a time
  const int lane_row = lane / kPieces, lane_piece = lane % kPieces;
  const long long k_lane = lane_row * p.kc.token_stride + lane_piece * 16, v_lane = lane_row * p.vc.token_stride + lane_piece * 16;
  const bool in_head = lane_piece * 8 < p.dim;
  auto issue = [&]() {
    const Ahead t = first_up;
    first_up = second_up;
    second_up = look_up();
    if (t.keys >= 0) {
      const int keys = t.keys;
      // rows behind the sequence's end are not read and become zero: their weights are, and 0 x NaN would be NaN
      const uint32_t dst = ring + load_stage * C::kTileBytes + (lane_piece >> 3) * C::kKeys * 128 + lane_row * 128;
      const char* k_head = p.kc.data + t.head * p.kc.head_stride;
      const char* v_head = p.vc.data + t.head * p.vc.head_stride;
      auto copy = [&](int row0, const char* k_src, const char* v_src, bool there) {
        const bool valid = there && row0 + lane_row < keys && in_head;
        const uint32_t at = dst + row0 * 128 + ((((lane_piece & 7) ^ ((row0 + lane_row) & 7))) << 4);
        copy16_async(at, valid ? k_src : p.kc.data, valid);
        copy16_async(at + C::kSideBytes, valid ? v_src : p.vc.data, valid);
      };
      if (EIGHTS) {
        const bool bad = lane * 8 < keys && static_cast<unsigned>(t.page) >= static_cast<unsigned>(p.pages);
        if (bad && p.index_word) *p.index_word = kBadIndex;
        const int good_page = bad ? -1 : t.page;
#pragma unroll
        for (int e = 0; e < C::kKeys / 8; ++e) {
          const int at_page = __shfl_sync(0xffffffffu, good_page, e), at_row = __shfl_sync(0xffffffffu, t.offset, e);
          const char* k_src = k_head + at_page * p.kc.page_stride + at_row * p.kc.token_stride + k_lane;
          const char* v_src = v_head + at_page * p.vc.page_stride + at_row * p.vc.token_stride + v_lane;
#pragma unroll
          for (int r = 0; r < 8; r += kRowsPerCopy)
            copy(e * 8 + r, k_src + r * p.kc.token_stride, v_src + r * p.vc.token_stride, at_page >= 0);
        }
      } else {
        const int* table = p.page_table + static_cast<long long>(t.seq) * p.table_pages;
#pragma unroll
        for (int r = 0; r < C::kKeys; r += kRowsPerCopy) {
          int at_page = -1, at_row = 0;
          if (r + lane_row < keys) {
            const int key = t.key0 + r + lane_row, slot = fast_div(key, p.by_page);
            at_row = key - slot * static_cast<int>(p.by_page.d);
            at_page = __ldg(table + slot);
            if (static_cast<unsigned>(at_page) >= static_cast<unsigned>(p.pages)) {
              if (p.index_word) *p.index_word = kBadIndex;
              at_page = -1;
            }
          }
          copy(r, k_head + at_page * p.kc.page_stride + at_row * p.kc.token_stride + lane_piece * 16,
               v_head + at_page * p.vc.page_stride + at_row * p.vc.token_stride + lane_piece * 16, at_page >= 0);
        }
      }
      if (++load_stage == kStages) load_stage = 0;
    }
    copies_commit();
  };

  constexpr int kNQ = HALF ? 1 : 2;                            // eights of query rows
  constexpr int kMT = DP / 16;                                 // sixteens of the output's columns, and of the products' depth
  const int col0 = (lane & 3) * 2, row0 = lane >> 2;
  int stage = 0;
  uint32_t qf[kMT][kNQ][2], q_next[kMT][kNQ][2];
  // o[i][q][c]: column 16 i + row0 (+ 8 where c > 1) of query 8 q + col0 + (c & 1); m and sum: of those two queries
  float o[kMT][kNQ][4], m[kNQ][2], sum[kNQ][2];
  auto row_tile = [&](int item) { return item - head_of(item) * p.row_tiles; };
  auto rows_of = [&](int item) { return item < p.items ? min(kRows, p.group - row_tile(item) * kRows) : 0; };
  auto first_row = [&](int item) { return head_of(item) * p.group + row_tile(item) * kRows; };
  // Queries as the first product's right operand; the next item's are fetched while one is run.
  auto fetch_q = [&](const Cursor& c) {
    if (c.stop < 0) return;
    const int item = item_of(c), rows = rows_of(item);
    const char* q = p.q.data + c.seq * p.q.token_stride + first_row(item) * p.q.head_stride;
#pragma unroll
    for (int k = 0; k < kMT; ++k)
#pragma unroll
      for (int j = 0; j < kNQ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = j * 8 + row0, col = k * 16 + e * 8 + col0;
          q_next[k][j][e] = r >= rows || col >= p.dim ? 0u : __ldg(reinterpret_cast<const unsigned int*>(q + r * p.q.head_stride + col * 2));
        }
  };
  auto row_of = [&](const Cursor& c, int item, int row) {
    return p.out + (static_cast<long long>(c.seq) * p.q_heads + first_row(item) + row) * p.dim * 2;
  };
  // An empty sequence gives zeros; one whose scores are all minus infinity has a sum of 0 too, and gives 0 x infinity, NaN.
  auto inverse = [&](const Cursor& c, float sum) { return c.len == 0 ? 0.0f : 1.0f / sum; };
  auto store = [&](const Cursor& c, int row, int col, float4 v, float sum) {
    const float inv = inverse(c, sum);
    *reinterpret_cast<uint2*>(row_of(c, c.unit, row) + col * 2) = make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
  };
  auto team_sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(kTeam) : "memory"); };

  // ---- The turns of the loop: the first ones only copy; at an item's end it is joined and the next one begun; else a tile.
  float* join = reinterpret_cast<float*>(smem + C::kRingBytes + team * C::kJoinBytes);
  const int thread = threadIdx.x % kTeam;
  fetch_q(next);
  Cursor now{0, 0, 0, 0, 0, false};
  int first_step = 0, ahead = kStages - 1;
  bool running = false;
#pragma unroll 1
  for (;;) {
    if (ahead == 0 && now.step >= now.stop) {
      if (running) {
#pragma unroll
        for (int q = 0; q < kNQ; ++q)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) sum[q][e] += __shfl_xor_sync(0xffffffffu, sum[q][e], d);
      }
      if (running && now.solo) {
        const int item = item_of(now), rows = rows_of(item);
#pragma unroll
        for (int q = 0; q < kNQ; ++q) {
          const float inv0 = inverse(now, sum[q][0]), inv1 = inverse(now, sum[q][1]);
          char* dst = row_of(now, item, q * 8 + row0);
          // (all exchanges in front of the stores, which not all lanes have)
          uint32_t v[kMT][2];
#pragma unroll
          for (int i = 0; i < kMT; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)        // eight columns by eight queries, to a query a lane's four
              v[i][e] = transpose(pack2<T>(o[i][q][2 * e] * inv0, o[i][q][2 * e + 1] * inv1));
          if (q * 8 + row0 < rows) {
#pragma unroll
            for (int i = 0; i < kMT; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (i * 16 + e * 8 < p.dim) *reinterpret_cast<uint32_t*>(dst + (i * 16 + e * 8 + col0) * 2) = v[i][e];
          }
          __syncwarp();
        }
      } else if (running) {
        const int rows = rows_of(now.unit), all = steps_of(tiles_of(now.len));
        const bool enters = first_step > 0, leaves = now.stop < all;
        Partial* part = partials + (run * 2 + (enters ? 0 : 1));
#pragma unroll
        for (int h = 0; h < kNQ; ++h) {
          team_sync();                         // what was there has been read
          float* own = join + (member * 8 + col0) * C::kJoinRow;
#pragma unroll
          for (int i = 0; i < kMT; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) own[(c & 1) * C::kJoinRow + i * 16 + (c >> 1) * 8 + row0] = o[i][h][c];
          if (row0 < 2) *reinterpret_cast<float2*>(own + row0 * C::kJoinRow + DP) = make_float2(row0 ? m[h][1] : m[h][0], row0 ? sum[h][1] : sum[h][0]);
          team_sync();
#pragma unroll 1
          for (int i = thread; i < 8 * DP / 4; i += kTeam) {
            const int r = i / (DP / 4), col = (i - r * (DP / 4)) * 4, row = r + 8 * h;
            if (row >= rows) break;
            float2 of[kTeamWarps];             // maximum and sum
            float top = kNegInf, row_sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kTeamWarps; ++w) {
              of[w] = *reinterpret_cast<const float2*>(join + (w * 8 + r) * C::kJoinRow + DP);
              top = fmaxf(top, of[w].x);
            }
            const float base = top == kNegInf ? 0.0f : top;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kTeamWarps; ++w) {
              const float f = exp2_fast(of[w].x - base);
              const float4 x = *reinterpret_cast<const float4*>(join + (w * 8 + r) * C::kJoinRow + col);
              acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
              row_sum += of[w].y * f;
            }
            if (!enters && !leaves) {
              if (col < p.dim) store(now, row, col, acc, row_sum);
            } else {
              __stcg(reinterpret_cast<float4*>(&part->o[row][col]), acc);
              if (col == 0) {
                __stcg(&part->m[row], top);
                __stcg(&part->sum[row], row_sum);
              }
            }
          }
        }
        if (enters || leaves) {
          // ---- an item that spans teams: whoever arrives last joins the parts
          const unsigned first_unit = enters ? cut.begin(run) - first_step : cut.begin(run + 1) - now.stop;
          const int first = static_cast<int>(cut.taker(first_unit)), last = static_cast<int>(cut.taker(first_unit + all - 1));
          team_sync();
          if (thread == 0) {
            __threadfence();
            s_last[team] = atomicAdd(p.counters + first, 1) == last - first;
            if (s_last[team]) p.counters[first] = 0;
            __threadfence();
          }
          team_sync();
          if (s_last[team]) {
#pragma unroll 1
            for (int i = thread; i < rows * (DP / 4); i += kTeam) {
              const int row = i / (DP / 4), col = (i - row * (DP / 4)) * 4;
              if (col >= p.dim) continue;
              float top = kNegInf, row_sum = 0.0f;
              float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              constexpr int kBatch = 4;        // parts that are fetched at a time
#pragma unroll 1
              for (int t0 = first; t0 <= last; t0 += kBatch) {
                float pm[kBatch], ps[kBatch];
                float4 po[kBatch];
#pragma unroll
                for (int e = 0; e < kBatch; ++e) {
                  const int t = min(t0 + e, last);
                  const Partial& x = partials[t * 2 + (t == first)];
                  pm[e] = t0 + e <= last ? __ldcg(&x.m[row]) : kNegInf;
                  ps[e] = __ldcg(&x.sum[row]);
                  po[e] = __ldcg(reinterpret_cast<const float4*>(&x.o[row][col]));
                }
                float higher = top;
#pragma unroll
                for (int e = 0; e < kBatch; ++e) higher = fmaxf(higher, pm[e]);
                const float base = higher == kNegInf ? 0.0f : higher, keep = exp2_fast(top - base);
                top = higher;
                row_sum *= keep;
                acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
#pragma unroll
                for (int e = 0; e < kBatch; ++e) {
                  if (t0 + e > last) break;
                  const float f = exp2_fast(pm[e] - base);
                  row_sum += ps[e] * f;
                  acc.x += po[e].x * f; acc.y += po[e].y * f; acc.z += po[e].z * f; acc.w += po[e].w * f;
                }
              }
              store(now, row, col, acc, row_sum);
            }
          }
        }
      }
      if (next.stop < 0) break;
      now = next;
      first_step = now.step;
      running = true;
#pragma unroll
      for (int k = 0; k < kMT; ++k)
#pragma unroll
        for (int q = 0; q < kNQ; ++q) {
          qf[k][q][0] = q_next[k][q][0];
          qf[k][q][1] = q_next[k][q][1];
          o[k][q][0] = o[k][q][1] = o[k][q][2] = o[k][q][3] = 0.0f;
        }
#pragma unroll
      for (int q = 0; q < kNQ; ++q) {
        m[q][0] = m[q][1] = kNegInf;
        sum[q][0] = sum[q][1] = 0.0f;
      }
      advance(next);
      fetch_q(next);
    }
    issue();
    if (ahead) {
      --ahead;
      continue;
    }
    const int keys = keys_of(now);
    const uint32_t tile_k = ring + stage * C::kTileBytes, tile_v = tile_k + C::kSideBytes;
    copies_wait<kStages - 1>();
    __syncwarp();
    if (++stage == kStages) stage = 0;
    ++now.step;
    if (keys <= 0) continue;
    float s[kNQ][4], odd[kNQ][4];              // products of even and odd sixteens of the head: two shorter chains
#pragma unroll
    for (int q = 0; q < kNQ; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[q][e] = odd[q][e] = 0.0f;
#pragma unroll
    for (int k = 0; k < kMT; ++k) {
      uint32_t a[4];
      ldmatrix_x4(a, tile_k + (k >> 2) * C::kKeys * 128 + (lane & 15) * 128 + ((((k & 3) * 2 + (lane >> 4)) ^ (lane & 7)) << 4));
#pragma unroll
      for (int q = 0; q < kNQ; ++q) mma_16816<T>(k & 1 ? odd[q] : s[q], a, qf[k][q][0], qf[k][q][1]);
    }
    float top[kNQ][2];
    bool grown = false;
#pragma unroll
    for (int q = 0; q < kNQ; ++q) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[q][e] = row0 + (e >> 1) * 8 < keys ? (s[q][e] + odd[q][e]) * p.scale_log2 : kNegInf;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[q][e] = fmaxf(s[q][e], s[q][2 + e]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top[q][e] = fmaxf(top[q][e], __shfl_xor_sync(0xffffffffu, top[q][e], d));
        grown = grown || top[q][e] > m[q][e];
      }
    }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int q = 0; q < kNQ; ++q) {
        float keep[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float now_top = fmaxf(m[q][e], top[q][e]);
          keep[e] = now_top == kNegInf ? 1.0f : exp2_fast(m[q][e] - now_top);
          m[q][e] = now_top;
          sum[q][e] *= keep[e];
        }
#pragma unroll
        for (int i = 0; i < kMT; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[i][q][c] *= keep[c & 1];
      }
    }
    uint32_t pf[kNQ][2];
#pragma unroll
    for (int q = 0; q < kNQ; ++q) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {            // (nothing but minus infinity so far: no difference of infinities)
        w[e] = exp2_fast(s[q][e] - (m[q][e & 1] == kNegInf ? 0.0f : m[q][e & 1] - kLift<T>));
        sum[q][e & 1] += w[e];
      }
      pf[q][0] = transpose(pack2<T>(w[0], w[1]));
      pf[q][1] = transpose(pack2<T>(w[2], w[3]));
    }
#pragma unroll
    for (int i = 0; i < kMT; ++i) {
      uint32_t a[4];
      ldmatrix_x4_trans(a, tile_v + (i >> 2) * C::kKeys * 128 + ((lane & 7) + (lane >> 4) * 8) * 128 +
                               ((((i & 3) * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4));
#pragma unroll
      for (int q = 0; q < kNQ; ++q) mma_16816<T>(o[i][q], a, pf[q][0], pf[q][1]);
    }
    __syncwarp();              // the next copies overwrite this tile
  }
  copies_wait<0>();
}

template <typename T, int DP, bool HALF, bool EIGHTS, bool WHOLE>
int launch_decode(DecodeParams p, cudaStream_t st) {
  using C = Decode<T, DP, HALF, EIGHTS, WHOLE>;
  static thread_local int configured_device = -1;
  int device = 0;
  MP_CUDA_TRY(cudaGetDevice(&device));
  if (configured_device != device) {
    MP_CUDA_TRY(cudaFuncSetAttribute(paged_decode_kernel<T, DP, HALF, EIGHTS, WHOLE>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    configured_device = device;
  }
  const long long items = static_cast<long long>(p.batch) * p.items;
  // with an item to a team and more, warps take those of short sequences alone
  p.solo_tiles = items >= kSmCount * C::kTeams ? kSoloTiles : 1;
  // no more teams than there can be whole items and steps of what is cut; a block for every team of those
  const long long step = C::kKeys * C::kTeamWarps, steps = (p.capacity + step - 1) / step;
  const long long teams = items * (steps <= kWholeSteps ? 1 : steps);
  const int grid = static_cast<int>(teams < kSmCount ? teams : kSmCount);
  return launch_chained(paged_decode_kernel<T, DP, HALF, EIGHTS, WHOLE>, dim3(grid), dim3(C::kThreads), C::kSmem, st, p);
}

template <typename T, int DP, bool HALF, bool EIGHTS>
int dispatch_teams(const DecodeParams& p, cudaStream_t st) {
  // No more items than SMs: an SM's warps all go to one, which is then seldom cut.  (Eight heads; whole blocks, teams of four
  // warps: 1 sequence of 300 tokens 7.5, 8.0 us, 16 of them 8.4, 11.3, 18 (144 items) 8.7, 12.8; 1 and 18 of 8000 16.4, 21.6
  // and 97, 96.  Beyond: 24 of 2000 38.5, 38.7; 37 of 300 14.0, 12.4; 64 of 8000 329, 314.)
  return static_cast<long long>(p.batch) * p.items <= kSmCount ? launch_decode<T, DP, HALF, EIGHTS, true>(p, st)
                                                               : launch_decode<T, DP, HALF, EIGHTS, false>(p, st);
}
template <typename T, int DP, bool EIGHTS>
int dispatch_rows(const DecodeParams& p, cudaStream_t st) {
  return p.group <= 8 ? dispatch_teams<T, DP, true, EIGHTS>(p, st) : dispatch_teams<T, DP, false, EIGHTS>(p, st);
}
template <typename T, int DP>
int dispatch_pages(const DecodeParams& p, cudaStream_t st) {
  // (16 tokens to a page and eight heads, pages looked up by eight rows, by the row: 64 sequences of 2000 tokens 87, 111 us;
  // 1 of 300 7.5, 9.9)
  return p.by_page.d % 8 == 0 ? dispatch_rows<T, DP, true>(p, st) : dispatch_rows<T, DP, false>(p, st);
}
template <typename T>
int dispatch_decode(const DecodeParams& p, cudaStream_t st) {
  return p.dim <= 64 ? dispatch_pages<T, 64>(p, st) : dispatch_pages<T, 128>(p, st);
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
  if ((dtype != 0 && dtype != 1) || Hq % cache->kv_heads || Hq > 65535 || B > (1 << 30)) return MP_ERR_UNSUPPORTED;
  if (!aligned(out, 16) || !aligned(workspace, 16)) return MP_ERR_ALIGNMENT;
  if (!workspace || workspace_bytes < kWorkspaceBytes) return MP_ERR_WORKSPACE;
  p.page_table = static_cast<const int*>(page_table_i32);
  p.seq_lens = static_cast<const int*>(seq_lens_i32);
  p.out = static_cast<char*>(out);
  p.counters = static_cast<int*>(workspace);
  p.partials = static_cast<char*>(workspace) + kCounterBytes;
  p.index_word = index_word;
  p.batch = B;
  p.q_heads = Hq;
  p.kv_heads = cache->kv_heads;
  p.dim = D;
  p.group = Hq / cache->kv_heads;
  p.row_tiles = (p.group + kRows - 1) / kRows;
  p.table_pages = table_pages;
  p.pages = cache->pages;
  p.items = p.kv_heads * p.row_tiles;
  const long long room = static_cast<long long>(table_pages) * cache->page_size;
  p.capacity = static_cast<int>(room < 0x7fffff00LL ? room : 0x7fffff00LL);
  p.scale_log2 = scale * attn::kLog2e;
  p.by_page = make_fast_div(cache->page_size);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == 0 ? dispatch_decode<__half>(p, st) : dispatch_decode<__nv_bfloat16>(p, st);
}
