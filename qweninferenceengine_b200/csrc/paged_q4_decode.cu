// paged_q4_decode.cu -- decode attention over a 4-bit paged cache, one query token per
// sequence, and the weights that each cached slot was given:
//   out = sum_t softmax(scale q . K_t) V_t,  K_t, V_t = low + code step
#include "paged_q4.cuh"
#include "qwen_internal.h"

namespace qwen {
namespace {

constexpr int kWarps = 4;

// A CTA per (query head, sequence); a warp takes every fourth block of 16 slots: two
// lanes a slot for the scores, a lane D / 32 elements of the output.
template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32) k_attend_q4(const __grid_constant__ Q4AttnArgs a, float* lse) {
  constexpr int G = D / 32;
  __shared__ float qs[D], part[kWarps][D], ml[kWarps][2];
  const int s = blockIdx.y, head = blockIdx.x, h = head / (a.n_heads / (int)a.kv.n_kv_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t L = a.seq_len[s];
  if (L > q4_capacity(a.kv)) {
    if (threadIdx.x == 0) raise_error(a.err, kDevBadArgument);
    return;
  }
  for (int d = threadIdx.x; d < D; d += kWarps * 32)
    qs[d] = (float)reinterpret_cast<const T*>(a.q)[(long long)s * a.q_stride + head * D + d] * a.scale * kLog2e;
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[G] = {};
  for (uint32_t b = warp; b * 16 < L; b += kWarps) {
    const int slot = b * 16, page = q4_page(a.kv, a.err, s, slot >> a.page_shift);
    if (page < 0) continue;
    const int valid = min(16, (int)L - slot);
    const uint8_t* block = q4_block<D>(a.kv, page, h, slot & ((int)a.kv.page_size - 1));
    const int r = lane & 15;
    float score = 0.f;
    for (int g = lane >> 4; g < G; g += 2) {
      const uint4 w = *reinterpret_cast<const uint4*>(block + g * 256 + r * 16);
      const uint32_t p = *reinterpret_cast<const uint32_t*>(block + Q4Block<D>::kKeySteps + g * 64 + r * 4);
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x[8];
        expand_word<T>(ws[i], p, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) score += x[e] * qs[32 * g + 8 * i + e];
      }
    }
    score += __shfl_xor_sync(0xffffffffu, score, 16);
    if (r >= valid) score = -INFINITY;
    float top = score;
    for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float m2 = fmaxf(m, top), ref = m2 == -INFINITY ? 0.f : m2, f = m == -INFINITY ? 0.f : exp2f(m - ref);
    const float w = r < valid ? exp2f(score - ref) : 0.f;
    float sum = w;
    for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    m = m2;
    l = l * f + sum;
    for (int g = 0; g < G; ++g) o[g] *= f;
    for (int j = 0; j < valid; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      for (int g = 0; g < G; ++g) {
        const uint8_t byte = block[Q4Block<D>::kValues + g * 256 + j * 16 + lane / 2];
        const float2 p = unpack2(T{}, *reinterpret_cast<const uint32_t*>(block + Q4Block<D>::kValueSteps + g * 64 + j * 4));
        o[g] += wj * fmaf((float)(byte >> (4 * (lane & 1)) & 15), p.x, p.y);
      }
    }
  }
  if (lane == 0) {
    ml[warp][0] = m;
    ml[warp][1] = l;
  }
  for (int g = 0; g < G; ++g) part[warp][32 * g + lane] = o[g];
  __syncthreads();
  float M = -INFINITY, sum = 0.f;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ml[w][0]);
  float f[kWarps];
  for (int w = 0; w < kWarps; ++w) {
    f[w] = ml[w][0] == -INFINITY && ml[w][1] == 0.f ? 0.f : exp2f(ml[w][0] - (M == -INFINITY ? 0.f : M));
    if (isnan(ml[w][1])) f[w] = ml[w][1];
    sum += ml[w][1] * f[w];
  }
  for (int d = threadIdx.x; d < D; d += kWarps * 32) {
    float x = 0.f;
    for (int w = 0; w < kWarps; ++w) x += f[w] == 0.f ? 0.f : part[w][d] * f[w];
    const uint32_t y = pack2(T{}, sum == 0.f ? 0.f : x / sum, 0.f);
    a.out[(long long)s * a.out_stride + head * D + d] = (uint16_t)y;
  }
  if (threadIdx.x == 0 && lse)
    lse[(long long)s * a.n_heads + head] = sum == 0.f ? -INFINITY : (M + log2f(sum)) * kLn2;
}

// weights[s][h][slot] += sum over the query heads of kv head h of exp(scale q k - lse).
template <typename T, int D>
__global__ void __launch_bounds__(128) k_weigh_q4(const __grid_constant__ Q4AttnArgs a, const float* lse) {
  const int s = blockIdx.z, h = blockIdx.y, group = a.n_heads / (int)a.kv.n_kv_heads;
  const uint32_t L = a.seq_len[s];
  if (L > q4_capacity(a.kv)) return;
  for (uint32_t slot = blockIdx.x * 128 + threadIdx.x; slot < L; slot += gridDim.x * 128) {
    const int page = q4_page(a.kv, a.err, s, slot >> a.page_shift);
    if (page < 0) continue;
    const int in_page = slot & (a.kv.page_size - 1), r = in_page & 15;
    const uint8_t* block = q4_block<D>(a.kv, page, h, in_page);
    float total = 0.f;
    for (int j = 0; j < group; ++j) {
      const int head = h * group + j;
      const T* q = reinterpret_cast<const T*>(a.q) + (long long)s * a.q_stride + head * D;
      float score = 0.f;
      for (int g = 0; g < D / 32; ++g) {
        const uint4 w = *reinterpret_cast<const uint4*>(block + g * 256 + r * 16);
        const uint32_t p = *reinterpret_cast<const uint32_t*>(block + Q4Block<D>::kKeySteps + g * 64 + r * 4);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x[8];
          expand_word<T>(ws[i], p, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) score += x[e] * (float)q[32 * g + 8 * i + e];
        }
      }
      total += exp2f(score * a.scale * kLog2e - lse[(long long)s * a.n_heads + head] * kLog2e);
    }
    a.kv.weights[((long long)s * a.kv.n_kv_heads + h) * q4_capacity(a.kv) + slot] += total;
  }
}

template <typename T, int D>
int launch(const Q4AttnArgs& a, cudaStream_t st) {
  float* lse = a.lse ? a.lse : a.kv.weights ? static_cast<float*>(a.workspace) : nullptr;
  k_attend_q4<T, D><<<dim3(a.n_heads, a.kv.n_seq), kWarps * 32, 0, st>>>(a, lse);
  if (a.kv.weights) {
    const unsigned ctas = std::min(64u, (a.kv.max_pages * a.kv.page_size + 127) / 128);
    k_weigh_q4<T, D><<<dim3(ctas, a.kv.n_kv_heads, a.kv.n_seq), 128, 0, st>>>(a, lse);
  }
  return 0;
}

}  // namespace

size_t attention_q4_workspace(const qwen_paged_kv_q4& kv, int n_heads) {
  return (size_t)kv.n_seq * n_heads * sizeof(float);
}

int launch_attention_q4(const Q4AttnArgs& a, cudaStream_t st) {
  const bool d64 = a.kv.head_dim == 64;
  if (a.kv.dtype == QWEN_DTYPE_F16) return d64 ? launch<__half, 64>(a, st) : launch<__half, 128>(a, st);
  return d64 ? launch<__nv_bfloat16, 64>(a, st) : launch<__nv_bfloat16, 128>(a, st);
}

}  // namespace qwen
