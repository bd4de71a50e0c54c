// Low-rank adapters of many requests beside a shared projection:
//
//   out[m] = base[m] + s_i B_i (A_i x[m]),  i = ids[m]   (i outside [0, adapters): out[m] = base[m])
//
// No counterpart in the reference.  A_i x is summed in fp32 and kept in fp32
// between the two launches (t, in the workspace); out is rounded once.
#include "common.h"

namespace {

// t[m, r] = s_i A_i[r] . x[m], a wave per (m, r)
template <typename T>
__global__ __launch_bounds__(256) void lora_shrink_kernel(const T* __restrict__ x, int64_t x_stride,
                                                          const T* __restrict__ a, const int32_t* __restrict__ ids,
                                                          const float* __restrict__ scales, float* __restrict__ t,
                                                          int64_t K, int R, int adapters) {
  const int m = blockIdx.x, r = (int)blockIdx.y * 4 + ((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int i = ids[m];
  if (r >= R || i < 0 || i >= adapters) return;
  const T* row = a + ((int64_t)i * R + r) * K;
  const T* xr = x + m * x_stride;
  float s = 0.0f;
  for (int64_t k = lane; k < K; k += MK_WAVE) s += to_f32(xr[k]) * to_f32(row[k]);
  s = wave_sum(s);
  if (lane == 0) t[(int64_t)m * R + r] = scales ? s * scales[i] : s;
}

// a thread per output
template <typename T>
__global__ __launch_bounds__(256) void lora_expand_kernel(const T* __restrict__ base, int64_t base_stride,
                                                          const T* __restrict__ b, const int32_t* __restrict__ ids,
                                                          const float* __restrict__ t, T* __restrict__ out,
                                                          int64_t out_stride, int64_t N, int R, int adapters) {
  const int m = blockIdx.x;
  const int64_t n = blockIdx.y * (int64_t)256 + threadIdx.x;
  if (n >= N) return;
  const int i = ids[m];
  float s = to_f32(base[m * base_stride + n]);
  if (i >= 0 && i < adapters) {
    const T* row = b + ((int64_t)i * N + n) * R;
    float d = 0.0f;
    for (int r = 0; r < R; ++r) d += t[(int64_t)m * R + r] * to_f32(row[r]);
    s += d;
  }
  out[m * out_stride + n] = from_f32<T>(s);
}

}  // namespace

extern "C" {

size_t mk_lora_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t R, int64_t adapters) {
  if (M <= 0 || N <= 0 || K <= 0 || R <= 0 || adapters <= 0) return 0;
  return (size_t)M * R * sizeof(float);
}

int mk_lora_add(const void* x, int64_t x_stride, const void* base, int64_t base_stride, const void* a, const void* b,
                const int32_t* adapter_ids, const float* scales, void* out, int64_t out_stride, int64_t M, int64_t N,
                int64_t K, int64_t R, int64_t adapters, int dtype, void* workspace, size_t workspace_bytes,
                void* stream) {
  MK_REQUIRE(M >= 0 && N >= 0 && K > 0 && R > 0 && R <= 128 && adapters >= 0);
  MK_REQUIRE(M < (1LL << 24) && N < (1LL << 24) && K < (1LL << 31) && adapters < (1LL << 31));
  MK_REQUIRE(x_stride >= K && base_stride >= N && out_stride >= N);
  MK_REQUIRE(dtype == MK_DT_F16 || dtype == MK_DT_BF16);
  if (M == 0 || N == 0) return MK_OK;
  MK_REQUIRE(x && base && adapter_ids && out && (adapters == 0 || (a && b)));
  MK_REQUIRE(adapters == 0 || (workspace && workspace_bytes >= mk_lora_workspace_bytes(M, N, K, R, adapters) &&
                               mk_aligned(workspace, 16)));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  float* t = reinterpret_cast<float*>(workspace);
#define MK_LORA(T)                                                                                                   \
  do {                                                                                                               \
    if (adapters)                                                                                                    \
      lora_shrink_kernel<T><<<dim3((unsigned)M, (unsigned)((R + 3) / 4)), 256, 0, st>>>(                             \
          (const T*)x, x_stride, (const T*)a, adapter_ids, scales, t, K, (int)R, (int)adapters);                     \
    lora_expand_kernel<T><<<dim3((unsigned)M, (unsigned)((N + 255) / 256)), 256, 0, st>>>(                           \
        (const T*)base, base_stride, (const T*)b, adapter_ids, t, (T*)out, out_stride, N, (int)R, (int)adapters);    \
  } while (0)
  if (dtype == MK_DT_F16) MK_LORA(f16);
  else MK_LORA(bf16);
#undef MK_LORA
  MK_CHECK_LAUNCH();
  return MK_OK;
}

}  // extern "C"
