// Low-rank adapters of many requests beside a shared projection:
//
//   out[m] = base[m] + s_i B_i (A_i x[m]),  i = ids[m]   (i outside [0, adapters): out[m] = base[m])
//
// No counterpart in the reference.  Two launches: the first sums t = A_i x[m]
// in fp32 (per slice of K, in the workspace), the second joins the slices,
// multiplies by B_i and adds base, with one rounding.
//
// Both run on 16x16x32 matrix instructions over tiles of 16 rows, without any
// sorting of rows: for each adapter that a tile's rows name, the products of
// all 16 rows with it are formed and the rows that name it keep theirs, so a
// row's values touch no other row (an infinity or NaN stays where it is).
// Prompts, whose rows name one adapter a tile, do no product twice; a decode
// batch is bound by reading its adapters, whatever their order.
//
// The second product's operand t is 32 bits: it goes in as the sum of two
// values of the storage type (relative 2^-16 for bf16, 2^-21 for fp16), in fp16
// scaled by a power of two per row so that neither part leaves its range.
#include "common.h"

namespace {

template <typename T>
struct Frag;
template <>
struct Frag<f16> {
  typedef f16x8 v8;
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Frag<bf16> {
  typedef bf16x8 v8;
  static __device__ __forceinline__ f32x4 mfma(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// 8 values p[at .. at + 8), zeros from `end` on
template <typename T, bool VEC>
__device__ __forceinline__ typename Frag<T>::v8 load_frag(const T* p, int64_t at, int64_t end) {
  typename Frag<T>::v8 v;
  if constexpr (VEC) {  // whole 16-byte chunks
    u32x4 w = {0u, 0u, 0u, 0u};
    if (at < end) w = ldg128(p + at);
    v = bitcast<typename Frag<T>::v8>(w);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = at + e < end ? p[at + e] : from_f32<T>(0.0f);
  }
  return v;
}

// The adapters of a tile's 16 rows (lane & 15), each once and in the order of
// the rows: next() gives the number `skip` further on, -1 behind the last.
// Uniform over the wave.
struct TileAdapters {
  uint64_t rest;
  int id;
  __device__ __forceinline__ TileAdapters(int my) : rest(__ballot(my >= 0) & 0xffffull), id(my) {}
  __device__ __forceinline__ int next(int skip) {
    int a = -1;
    for (int k = 0; k <= skip; ++k) {
      if (rest == 0) return -1;
      a = __builtin_amdgcn_readlane(id, __builtin_ctzll(rest));
      rest &= ~__ballot(id == a);
    }
    return a;
  }
};

__device__ __forceinline__ int row_adapter(const int32_t* ids, int64_t m, int64_t M, int adapters) {
  const int i = m < M ? ids[m] : -1;
  return i < adapters ? i : -1;
}

// ---------------------------------------------------------------------------
// t = A x: a workgroup of 8 waves has a tile of rows, a slice of K, and every
// gridDim.z-th adapter of the tile; its waves take turns of 32 values of K and
// are summed through LDS.  The product is A (ranks down) times x (rows
// across): a lane ends with 4 ranks of one row.
// ---------------------------------------------------------------------------

constexpr int kShrinkWaves = 8;

template <typename T, int RT, bool VEC>
__global__ __launch_bounds__(64 * kShrinkWaves) void lora_shrink_kernel(
    const T* __restrict__ x, int64_t x_stride, const T* __restrict__ a, const int32_t* __restrict__ ids,
    float* __restrict__ t, int64_t M, int64_t K, int R, int adapters, int64_t k_slice) {
  constexpr int UN = VEC ? (RT >= 4 ? 2 : 4) : 1;  // turns whose loads are in flight together
  __shared__ f32x4 part[kShrinkWaves][RT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, grp = lane >> 4;
  const int64_t m = (int64_t)blockIdx.x * 16 + col;
  const int my = row_adapter(ids, m, M, adapters);
  const int64_t k0 = (int64_t)blockIdx.y * k_slice;
  const int64_t k1 = k0 + k_slice < K ? k0 + k_slice : K;
  const T* xr = x + (m < M ? m : M - 1) * x_stride;
  TileAdapters tile(my);
  for (int i = tile.next((int)blockIdx.z); i >= 0; i = tile.next((int)gridDim.z - 1)) {
    const T* ai = a + (int64_t)i * R * K;
    f32x4 acc[RT];
#pragma unroll
    for (int q = 0; q < RT; ++q) acc[q] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int64_t kb = k0 + 32 * wave; kb < k1; kb += 32 * kShrinkWaves * UN) {
      typename Frag<T>::v8 xf[UN], af[UN][RT];
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int64_t k = kb + 32 * kShrinkWaves * u + 8 * grp;
        xf[u] = load_frag<T, VEC>(xr, k, k1);
#pragma unroll
        for (int q = 0; q < RT; ++q) {
          const int r = 16 * q + col;
          af[u][q] = load_frag<T, VEC>(ai + (int64_t)(r < R ? r : 0) * K, k, r < R ? k1 : 0);
        }
      }
#pragma unroll
      for (int u = 0; u < UN; ++u)
#pragma unroll
        for (int q = 0; q < RT; ++q) acc[q] = Frag<T>::mfma(af[u][q], xf[u], acc[q]);
    }
    __syncthreads();  // the last adapter's sums are read
#pragma unroll
    for (int q = 0; q < RT; ++q) part[wave][q][lane] = acc[q];
    __syncthreads();
    for (int q = wave; q < RT; q += kShrinkWaves) {
      f32x4 s = part[0][q][lane];
#pragma unroll
      for (int w = 1; w < kShrinkWaves; ++w) s += part[w][q][lane];
      if (my == i)
        *reinterpret_cast<f32x4*>(t + ((int64_t)blockIdx.y * M + m) * (16 * RT) + 16 * q + 4 * grp) = s;
    }
  }
}

// ---------------------------------------------------------------------------
// out = base + s B t: a wave has 64 outputs of up to kRowTiles tiles of rows.
// The product is B (outputs down) times t (rows across).  The outputs of
// instruction j are 16 (r / 4) + 4 j + r % 4 for its rows r, so that a lane
// ends with 16 outputs side by side of one row: 32 bytes of base and out.
// ---------------------------------------------------------------------------

constexpr int kRowTiles = 4;

template <typename T, int RT, bool VEC>
__global__ __launch_bounds__(256) void lora_expand_kernel(
    const T* __restrict__ base, int64_t base_stride, const T* __restrict__ b, const int32_t* __restrict__ ids,
    const float* __restrict__ scales, const float* __restrict__ t, T* out, int64_t out_stride, int64_t M, int64_t N,
    int R, int adapters, int slices, int row_tiles, bool wide) {
  typedef typename Frag<T>::v8 v8;
  // up to 16 ranks: both parts of t in one instruction, over B twice
  constexpr int KS = RT == 1 ? 1 : (RT + 1) / 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, grp = lane >> 4;
  const int64_t n0 = ((int64_t)blockIdx.x * 4 + wave) * 64;
  if (n0 >= N) return;
  const int64_t n = n0 + 16 * grp;  // this lane's first output
  v8 bf[4][KS];
  int held = -1;  // the adapter in bf
  for (int rt = 0; rt < row_tiles; ++rt) {
    const int64_t m0 = ((int64_t)blockIdx.y * row_tiles + rt) * 16;
    if (m0 >= M) return;
    const int64_t m = m0 + col;
    const int my = row_adapter(ids, m, M, adapters);
    float keep[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) keep[e] = 0.0f;
    bool mine = my < 0 && blockIdx.z == 0 && base != out;
    TileAdapters tile(my);
    for (int i = tile.next((int)blockIdx.z); i >= 0; i = tile.next((int)gridDim.z - 1)) {
      if (i != held) {
        held = i;
        const T* bi = b + (int64_t)i * N * R;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t row = n0 + 16 * (col >> 2) + 4 * j + (col & 3);
#pragma unroll
          for (int s = 0; s < KS; ++s)
            bf[j][s] = load_frag<T, VEC>(bi + (row < N ? row : N - 1) * R, RT == 1 ? 8 * (grp & 1) : 32 * s + 8 * grp, R);
        }
      }
      // t of this lane's row, its slices joined
      float tv[KS][8];
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int at = RT == 1 ? 8 * (grp & 1) : 32 * s + 8 * grp;
#pragma unroll
        for (int e = 0; e < 8; ++e) tv[s][e] = 0.0f;
        if (my == i && at < 16 * RT) {
          const float* tr = t + m * (16 * RT) + at;
          for (int z = 0; z < slices; ++z, tr += M * (16 * RT)) {
            const f32x4 lo = *reinterpret_cast<const f32x4*>(tr), hi = *reinterpret_cast<const f32x4*>(tr + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              tv[s][e] += lo[e];
              tv[s][4 + e] += hi[e];
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(tv[s][e]));
      }
      float back = scales ? scales[i] : 1.0f;
      if constexpr (sizeof(T) == 2 && __is_same(T, f16)) {
        // the row's largest value to [2^13, 2^14)
        top = fmaxf(top, __shfl_xor(top, 16, MK_WAVE));
        top = fmaxf(top, __shfl_xor(top, 32, MK_WAVE));
        int e = 0;
        if (top > 0.0f && top < INFINITY) (void)frexpf(top, &e);
        else e = 14;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int q = 0; q < 8; ++q) tv[s][q] = ldexpf(tv[s][q], 14 - e);
        back = ldexpf(back, e - 14);
      }
      f32x4 acc[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        v8 hi, lo;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          hi[q] = from_f32<T>(tv[s][q]);
          const float left = tv[s][q] - to_f32(hi[q]);
          lo[q] = from_f32<T>(fabsf(tv[s][q]) < INFINITY ? left : 0.0f);
        }
        if constexpr (RT == 1) {
          const v8 both = grp < 2 ? hi : lo;
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = Frag<T>::mfma(bf[j][s], both, acc[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = Frag<T>::mfma(bf[j][s], hi, acc[j]);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = Frag<T>::mfma(bf[j][s], lo, acc[j]);
        }
      }
      if (my == i) {
        mine = true;
#pragma unroll
        for (int e = 0; e < 16; ++e) keep[e] = acc[e >> 2][e & 3] * back;
      }
    }
    if (!mine || m >= M) continue;
    const T* br = base + m * base_stride + n;
    T* orow = out + m * out_stride + n;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (wide && n + 8 * h < N) {  // whole 16-byte chunks
        const u32x4 w = ldg128(br + 8 * h);
        u32x4 o;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float y0 = to_f32(bitcast<T>((uint16_t)w[e >> 1])) + keep[8 * h + e];
          const float y1 = to_f32(bitcast<T>((uint16_t)(w[e >> 1] >> 16))) + keep[8 * h + e + 1];
          o[e >> 1] = (uint32_t)bitcast<uint16_t>(from_f32<T>(y0)) |
                      ((uint32_t)bitcast<uint16_t>(from_f32<T>(y1)) << 16);
        }
        if (my < 0) o = w;
        *reinterpret_cast<u32x4*>(orow + 8 * h) = o;
      } else if (!wide) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + 8 * h + e < N)
            orow[8 * h + e] = my < 0 ? br[8 * h + e] : from_f32<T>(to_f32(br[8 * h + e]) + keep[8 * h + e]);
      }
    }
  }
}

struct LoraPlan {
  int64_t tiles, k_slice;
  int slices, rank_tiles, adapters_at_once;
};

inline LoraPlan lora_plan(int64_t M, int64_t K, int64_t R, int64_t adapters) {
  LoraPlan p;
  p.tiles = (M + 15) / 16;
  p.rank_tiles = R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8;
  // decode batches: the adapters of a tile side by side; prompts: in turn
  const int64_t most = M < adapters ? M : adapters;
  p.adapters_at_once = M <= 64 ? (int)(most < 16 ? (most > 0 ? most : 1) : 16) : 1;
  // K in slices of four turns of a workgroup where there are few tiles
  const int64_t turn = 32 * kShrinkWaves;
  int64_t s = (K + 4 * turn - 1) / (4 * turn);
  const int64_t fill = (256 + p.tiles - 1) / p.tiles;
  if (s > fill) s = fill;
  p.k_slice = (K + s - 1) / s;
  p.k_slice = (p.k_slice + turn - 1) / turn * turn;
  p.slices = (int)((K + p.k_slice - 1) / p.k_slice);
  return p;
}

}  // namespace

extern "C" {

size_t mk_lora_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t R, int64_t adapters) {
  if (M <= 0 || N <= 0 || K <= 0 || R <= 0 || R > 128 || adapters <= 0) return 0;
  const LoraPlan p = lora_plan(M, K, R, adapters);
  return (size_t)p.slices * M * 16 * p.rank_tiles * sizeof(float);
}

int mk_lora_add(const void* x, int64_t x_stride, const void* base, int64_t base_stride, const void* a, const void* b,
                const int32_t* adapter_ids, const float* scales, void* out, int64_t out_stride, int64_t M, int64_t N,
                int64_t K, int64_t R, int64_t adapters, int dtype, void* workspace, size_t workspace_bytes,
                void* stream) {
  MK_REQUIRE(M >= 0 && N >= 0 && K > 0 && R > 0 && R <= 128 && adapters >= 0);
  MK_REQUIRE(M < (1LL << 20) && N < (1LL << 24) && K < (1LL << 31) && adapters < (1LL << 31));
  MK_REQUIRE(x_stride >= K && base_stride >= N && out_stride >= N && (out != base || out_stride == base_stride));
  MK_REQUIRE(dtype == MK_DT_F16 || dtype == MK_DT_BF16);
  if (M == 0 || N == 0) return MK_OK;
  MK_REQUIRE(x && base && adapter_ids && out && (adapters == 0 || (a && b)));
  MK_REQUIRE(adapters == 0 || (workspace && workspace_bytes >= mk_lora_workspace_bytes(M, N, K, R, adapters) &&
                               mk_aligned(workspace, 16)));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  float* t = reinterpret_cast<float*>(workspace);
  const LoraPlan p = lora_plan(M, K, R, adapters);
  const bool vec_a = K % 8 == 0 && x_stride % 8 == 0 && mk_aligned(x, 16) && mk_aligned(a, 16);
  const bool vec_b = R % 8 == 0 && mk_aligned(b, 16);
  const bool wide = N % 8 == 0 && base_stride % 8 == 0 && out_stride % 8 == 0 && mk_aligned(base, 16) &&
                    mk_aligned(out, 16);
  const int row_tiles = p.tiles >= kRowTiles ? kRowTiles : 1;
  const dim3 shrink((unsigned)p.tiles, (unsigned)p.slices, (unsigned)p.adapters_at_once);
  const dim3 expand((unsigned)((N + 255) / 256), (unsigned)((p.tiles + row_tiles - 1) / row_tiles),
                    (unsigned)p.adapters_at_once);
#define MK_SHRINK(T, RT, V)                                                                                      \
  lora_shrink_kernel<T, RT, V><<<shrink, 64 * kShrinkWaves, 0, st>>>((const T*)x, x_stride, (const T*)a, adapter_ids, \
                                                                     t, M, K, (int)R, (int)adapters, p.k_slice)
#define MK_EXPAND(T, RT, V)                                                                                       \
  lora_expand_kernel<T, RT, V><<<expand, 256, 0, st>>>((const T*)base, base_stride, (const T*)b, adapter_ids, scales, \
                                                       t, (T*)out, out_stride, M, N, (int)R, (int)adapters, p.slices, \
                                                       row_tiles, wide)
#define MK_LORA(T, RT)                  \
  do {                                  \
    if (adapters) {                     \
      if (vec_a) MK_SHRINK(T, RT, true); \
      else MK_SHRINK(T, RT, false);     \
    }                                   \
    if (vec_b) MK_EXPAND(T, RT, true);  \
    else MK_EXPAND(T, RT, false);       \
  } while (0)
#define MK_LORA_RANK(T)                         \
  do {                                          \
    if (p.rank_tiles == 1) MK_LORA(T, 1);       \
    else if (p.rank_tiles == 2) MK_LORA(T, 2);  \
    else if (p.rank_tiles == 4) MK_LORA(T, 4);  \
    else MK_LORA(T, 8);                         \
  } while (0)
  if (dtype == MK_DT_F16) MK_LORA_RANK(f16);
  else MK_LORA_RANK(bf16);
#undef MK_LORA_RANK
#undef MK_LORA
#undef MK_EXPAND
#undef MK_SHRINK
  MK_CHECK_LAUNCH();
  return MK_OK;
}

}  // extern "C"
