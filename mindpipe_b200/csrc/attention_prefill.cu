// Causal attention of whole prompts: packed sequences of different lengths, grouped heads.
//
//   o_i = sum_{j <= i} exp(s_ij - m_i) v_j / sum_{j <= i} exp(s_ij - m_i),   s_ij = scale q_i . k_j
//
// with a running maximum, sum and output over tiles of keys.
#include "attention.cuh"

namespace mp {
namespace {

using namespace attn;

constexpr int kRowsPerBlock = 64, kKeys = 64, kThreads = 128;

struct PrefillParams {
  HeadRows q, k, v;
  const int* cu_seqlens;
  char* out;
  int* index_word;
  int tokens, batch, q_heads, group, dim;
  float scale_log2;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) prefill_kernel(const PrefillParams p) {
  extern __shared__ __align__(128) char smem[];
  chain_wait();
  chain_release();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Tile numbers: sequence b has those from cu[b] / 64 + b on, which is room for all its tiles, so that the sequence of a
  // tile is found without the sum of the others'.
  const int number = blockIdx.x;
  int lo = 0, hi = p.batch;                     // first number of lo <= number < first number of hi
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (__ldg(p.cu_seqlens + mid) / kRowsPerBlock + mid <= number) lo = mid; else hi = mid;
  }
  const int begin = __ldg(p.cu_seqlens + lo), end = __ldg(p.cu_seqlens + lo + 1);
  if (begin < 0 || end < begin || end > p.tokens) {
    if (p.index_word) *p.index_word = kBadIndex;
    return;
  }
  const int row_begin = (number - begin / kRowsPerBlock - lo) * kRowsPerBlock, len = end - begin;
  if (row_begin < 0 || row_begin >= len) return;
  const int head = blockIdx.y, kv = head / p.group;
  const int row0 = row_begin + warp * 16 + (lane >> 2), col0 = (lane & 3) * 2;
  uint32_t qf[DP / 16][4];
  const char* q = p.q.data + begin * p.q.token_stride + head * p.q.head_stride;
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = row0 + (j & 1) * 8, c = k * 16 + col0 + (j >> 1) * 8;
      qf[k][j] = r >= len || c >= p.dim ? 0u : __ldg(reinterpret_cast<const unsigned int*>(q + r * p.q.token_stride + c * 2));
    }
  const char* k_rows = p.k.data + begin * p.k.token_stride + kv * p.k.head_stride;
  const char* v_rows = p.v.data + begin * p.v.token_stride + kv * p.v.head_stride;
  constexpr int kPieces = DP / 8, kSide = kKeys * DP * 2;
  const uint32_t base = tc::smem_u32(smem);
  auto load = [&](int tile) {
    const uint32_t dst = base + (tile & 1) * 2 * kSide;
    for (int i = threadIdx.x; i < kKeys * kPieces; i += kThreads) {
      const int row = i / kPieces, piece = i - row * kPieces, key = tile * kKeys + row;
      const bool valid = key < len && piece * 8 < p.dim;
      const long long r = valid ? key : 0;
      const int c = valid ? piece * 16 : 0;
      copy16_async(dst + piece_at<DP>(row, piece), k_rows + r * p.k.token_stride + c, valid);
      copy16_async(dst + kSide + piece_at<DP>(row, piece), v_rows + r * p.v.token_stride + c, valid);
    }
    copies_commit();
  };
  constexpr int kNT = DP / 8;
  float o[kNT][4];
#pragma unroll
  for (int n = 0; n < kNT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
  float m[2] = {kNegInf, kNegInf}, sum[2] = {0.0f, 0.0f};
  const int tiles = (min(row_begin + kRowsPerBlock, len) + kKeys - 1) / kKeys;
  load(0);
  for (int t = 0; t < tiles; ++t) {
    if (t + 1 < tiles) load(t + 1); else copies_commit();
    copies_wait<1>();
    __syncthreads();
    const uint32_t tile_k = base + (t & 1) * 2 * kSide, tile_v = tile_k + kSide;
    float s[kKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
      for (int n = 0; n < kKeys / 16; ++n) {
        uint32_t b[4];
        ldmatrix_x4(b, tile_k + piece_at<DP>(n * 16 + (lane & 7) + (lane >> 4) * 8, k * 2 + ((lane >> 3) & 1)));
        mma_16816<T>(s[2 * n], qf[k], b[0], b[1]);
        mma_16816<T>(s[2 * n + 1], qf[k], b[2], b[3]);
      }
    float keep[2], ref[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = kNegInf;
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float& v = s[n][2 * h + j];
          v = t * kKeys + n * 8 + col0 + j <= row0 + 8 * h ? v * p.scale_log2 : kNegInf;
          top = fmaxf(top, v);
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float now = fmaxf(m[h], top);
      ref[h] = now == kNegInf ? 0.0f : now;
      keep[h] = exp2_fast(m[h] - ref[h]);
      m[h] = now;
      sum[h] *= keep[h];
    }
    uint32_t pf[kKeys / 16][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float e0 = exp2_fast(s[n][2 * h] - ref[h]), e1 = exp2_fast(s[n][2 * h + 1] - ref[h]);
        sum[h] += e0 + e1;
        pf[n >> 1][(n & 1) * 2 + h] = pack2<T>(e0, e1);
      }
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[n][j] *= keep[j >> 1];
#pragma unroll
    for (int k = 0; k < kKeys / 16; ++k)
#pragma unroll
      for (int n = 0; n < kNT / 2; ++n) {
        uint32_t b[4];
        ldmatrix_x4_trans(b, tile_v + piece_at<DP>(k * 16 + (lane & 15), n * 2 + (lane >> 4)));
        mma_16816<T>(o[2 * n], pf[k], b[0], b[1]);
        mma_16816<T>(o[2 * n + 1], pf[k], b[2], b[3]);
      }
    __syncthreads();
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
    const float inv = 1.0f / sum[h];
    const int r = row0 + 8 * h;
    if (r >= len) continue;
    char* dst = p.out + ((static_cast<long long>(begin) + r) * p.q_heads + head) * p.dim * 2;
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      const int c = n * 8 + col0;
      if (c < p.dim) *reinterpret_cast<uint32_t*>(dst + c * 2) = pack2<T>(o[n][2 * h] * inv, o[n][2 * h + 1] * inv);
    }
  }
}

template <typename T, int DP>
int launch_prefill(const PrefillParams& p, cudaStream_t st) {
  const int smem = 4 * kKeys * DP * 2;
  static thread_local int configured_device = -1;
  int device = 0;
  MP_CUDA_TRY(cudaGetDevice(&device));
  if (configured_device != device) {
    MP_CUDA_TRY(cudaFuncSetAttribute(prefill_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    configured_device = device;
  }
  const dim3 grid(p.tokens / kRowsPerBlock + p.batch, p.q_heads);
  return launch_chained(prefill_kernel<T, DP>, grid, dim3(kThreads), smem, st, p);
}

}  // namespace
}  // namespace mp

extern "C" int mp_attention_prefill(int dtype, const mp_head_rows* q, const mp_head_rows* k, const mp_head_rows* v, int T,
                                    int Hq, int Hkv, int D, const void* cu_seqlens_i32, int B, float scale, void* out,
                                    int* index_word, int* error_word, mp_stream_t stream) {
  using namespace mp;
  PrefillParams p{};
  int rc;
  if ((rc = check_head_rows(q, D, &p.q)) || (rc = check_head_rows(k, D, &p.k)) || (rc = check_head_rows(v, D, &p.v))) return rc;
  if (!cu_seqlens_i32 || !out || T <= 0 || B <= 0 || Hq <= 0 || Hkv <= 0) return MP_ERR_INVALID_ARG;
  if ((dtype != 0 && dtype != 1) || Hq % Hkv || Hq > 65535) return MP_ERR_UNSUPPORTED;
  if (!aligned(out, 16)) return MP_ERR_ALIGNMENT;
  p.cu_seqlens = static_cast<const int*>(cu_seqlens_i32);
  p.out = static_cast<char*>(out);
  p.index_word = index_word;
  p.tokens = T;
  p.batch = B;
  p.q_heads = Hq;
  p.group = Hq / Hkv;
  p.dim = D;
  p.scale_log2 = scale * attn::kLog2e;
  (void)error_word;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (D <= 64) return dtype == 0 ? launch_prefill<__half, 64>(p, st) : launch_prefill<__nv_bfloat16, 64>(p, st);
  return dtype == 0 ? launch_prefill<__half, 128>(p, st) : launch_prefill<__nv_bfloat16, 128>(p, st);
}
