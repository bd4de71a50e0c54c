// Rotary positions in both layouts over all or the first part of each head
// (ops/rope_ops.py:61-75 has the interleaved layout over whole heads), and the
// norms of q and k heads with the rotation and the paged cache write in the
// same pass.
//
//   y_a = x_a c - x_b s,  y_b = x_a s + x_b c     (a, b) = (2i, 2i+1) or (i, i + R/2),  i < R/2
//   n = x * rsqrt(mean over the head of x^2 + eps) * w     before it, where weights are given
//
// c and s come from row p of the tables, p the token's position; values past R
// are copied.  fp32 throughout and one rounding into the storage type.
//
// Both are bound by memory: a head's D values are read and written once.  A
// unit of work is 16 values, two 16-byte chunks that hold the partners of
// each other's values (chunks u and u + R/16 in the half layout, 2u and
// 2u + 1 in the interleaved one), so a lane rotates without lane exchange and
// needs one run of 8 cos and 8 sin values; the lanes of a wave that hold the
// same unit of several heads read the same table bytes.  A head is D/16 lanes,
// and its sum of squares goes over those lanes by shuffles.
#include "common.h"
#include "paged_common.h"

namespace {

constexpr int kLayoutInterleaved = 0;
constexpr int kLayoutHalf = 1;

// first and second chunk (of 8 values) of unit u of a head with ru rotated units
template <int LAYOUT>
__device__ __forceinline__ void unit_chunks(int u, int ru, int* c0, int* c1) {
  const bool half = LAYOUT == kLayoutHalf && u < ru;
  *c0 = half ? u : 2 * u;
  *c1 = half ? u + ru : 2 * u + 1;
}

template <typename T>
__device__ __forceinline__ void unpack16(const u32x4& a, const u32x4& b, float (&v)[16]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = to_f32(bitcast<T>((uint16_t)(a[e >> 1] >> (16 * (e & 1)))));
    v[8 + e] = to_f32(bitcast<T>((uint16_t)(b[e >> 1] >> (16 * (e & 1)))));
  }
}

template <typename T>
__device__ __forceinline__ void pack16(const float (&v)[16], u32x4* a, u32x4* b) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    (*a)[e] = (uint32_t)bitcast<uint16_t>(from_f32<T>(v[2 * e])) |
              ((uint32_t)bitcast<uint16_t>(from_f32<T>(v[2 * e + 1])) << 16);
    (*b)[e] = (uint32_t)bitcast<uint16_t>(from_f32<T>(v[8 + 2 * e])) |
              ((uint32_t)bitcast<uint16_t>(from_f32<T>(v[8 + 2 * e + 1])) << 16);
  }
}

// the 8 pairs of a unit, with the 8 angles from cr and sr on
template <int LAYOUT>
__device__ __forceinline__ void rotate16(float (&v)[16], const float* cr, const float* sr) {
  float c[8], s[8];
  const u32x4 c0 = ldg128(cr), c1 = ldg128(cr + 4), s0 = ldg128(sr), s1 = ldg128(sr + 4);
  __builtin_memcpy(c, &c0, 16);
  __builtin_memcpy(c + 4, &c1, 16);
  __builtin_memcpy(s, &s0, 16);
  __builtin_memcpy(s + 4, &s1, 16);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int a = LAYOUT == kLayoutHalf ? i : 2 * i;
    const int b = LAYOUT == kLayoutHalf ? 8 + i : 2 * i + 1;
    float ya, yb;
    rope_pair(v[a], v[b], c[i], s[i], &ya, &yb);
    v[a] = ya;
    v[b] = yb;
  }
}

// value i of a rotated head, from its source values f(0 .. D-1)
template <int LAYOUT, typename F>
__device__ __forceinline__ float rotated_value(int i, int rd, const float* cr, const float* sr, F f) {
  if (i >= rd) return f(i);
  const int half = rd >> 1;
  const int j = LAYOUT == kLayoutHalf ? (i < half ? i : i - half) : i >> 1;
  const int a = LAYOUT == kLayoutHalf ? j : 2 * j;
  const int b = LAYOUT == kLayoutHalf ? j + half : 2 * j + 1;
  float ya, yb;
  rope_pair(f(a), f(b), cr[j], sr[j], &ya, &yb);
  return i == a ? ya : yb;
}

// where the token of row (b, s) stands: offset + s, pos[b] + s or pos[b, s];
// -1 (a row of zeros) for negative entries and positions outside the tables
constexpr int kPosOffset = 0, kPosFirst = 1, kPosEach = 2;
__device__ __forceinline__ int64_t row_position(const int32_t* pos, int mode, int64_t offset, int64_t b, int64_t s,
                                                int64_t S, int64_t rows) {
  int64_t p = offset + s;
  if (mode != kPosOffset) {
    p = pos[mode == kPosFirst ? b : b * S + s];
    if (p >= 0 && mode == kPosFirst) p += s;
  }
  return p < 0 || p >= rows ? -1 : p;
}

struct RopeDims {
  int64_t S, H, sb, ss, sh, rows, offset;  // strides of x in values; its last dimension is dense
  int D, rd, mode;
};

// a unit per thread; units < 2^31
template <typename T, int LAYOUT>
__global__ __launch_bounds__(256) void rope_vec_kernel(const T* __restrict__ x, const float* __restrict__ cos_t,
                                                       const float* __restrict__ sin_t,
                                                       const int32_t* __restrict__ pos, T* __restrict__ y,
                                                       uint32_t units, RopeDims d) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= units) return;
  const uint32_t upr = (uint32_t)d.D >> 4;
  const int ru = d.rd >> 4;
  const uint32_t row = i / upr, t = row / (uint32_t)d.H, b = t / (uint32_t)d.S;
  const int u = (int)(i - row * upr);
  const uint32_t h = row - t * (uint32_t)d.H, s = t - b * (uint32_t)d.S;
  int c0, c1;
  unit_chunks<LAYOUT>(u, ru, &c0, &c1);
  const T* xr = x + (int64_t)b * d.sb + (int64_t)s * d.ss + (int64_t)h * d.sh;
  const u32x4 x0 = ldg128(xr + 8 * c0), x1 = ldg128(xr + 8 * c1);
  const int64_t p = row_position(pos, d.mode, d.offset, b, s, d.S, d.rows);
  u32x4 y0 = {0u, 0u, 0u, 0u}, y1 = {0u, 0u, 0u, 0u};
  if (p >= 0) {
    y0 = x0;
    y1 = x1;
    if (u < ru) {
      float v[16];
      unpack16<T>(x0, x1, v);
      const size_t at = (size_t)p * (d.rd >> 1) + 8 * u;
      rotate16<LAYOUT>(v, cos_t + at, sin_t + at);
      pack16<T>(v, &y0, &y1);
    }
  }
  T* yr = y + (size_t)row * d.D;
  *reinterpret_cast<u32x4*>(yr + 8 * c0) = y0;
  *reinterpret_cast<u32x4*>(yr + 8 * c1) = y1;
}

// any sizes and alignment: a wave per head
template <typename T, int LAYOUT>
__global__ __launch_bounds__(256) void rope_any_kernel(const T* __restrict__ x, const float* __restrict__ cos_t,
                                                       const float* __restrict__ sin_t,
                                                       const int32_t* __restrict__ pos, T* __restrict__ y,
                                                       int64_t heads, RopeDims d) {
  const int lane = threadIdx.x & 63;
  for (int64_t row = blockIdx.x * 4ll + (threadIdx.x >> 6); row < heads; row += gridDim.x * 4ll) {
    const int64_t t = row / d.H, b = t / d.S;
    const int64_t h = row - t * d.H, s = t - b * d.S;
    const T* xr = x + b * d.sb + s * d.ss + h * d.sh;
    T* yr = y + row * d.D;
    const int64_t p = row_position(pos, d.mode, d.offset, b, s, d.S, d.rows);
    const float* cr = cos_t + (p < 0 ? 0 : p) * (d.rd >> 1);
    const float* sr = sin_t + (p < 0 ? 0 : p) * (d.rd >> 1);
    for (int i = lane; i < d.D; i += MK_WAVE) {
      if (p < 0) yr[i] = from_f32<T>(0.0f);
      else if (i >= d.rd) yr[i] = xr[i];
      else yr[i] = from_f32<T>(rotated_value<LAYOUT>(i, d.rd, cr, sr, [&](int j) { return to_f32(xr[j]); }));
    }
  }
}

// ---------------------------------------------------------------------------
// q and k norms, rotation and the cache write
// ---------------------------------------------------------------------------

struct QkDims {
  int64_t row_stride, page_size, max_blocks, num_pages, rows;  // row_stride of qkv in values
  int T, B, Hq, Hkv, D, rd, wdt;
  float eps;
};

__device__ __forceinline__ float norm_weight(const void* w, int wdt, int i) {
  if (wdt == MK_DT_F16) return to_f32(reinterpret_cast<const f16*>(w)[i]);
  if (wdt == MK_DT_BF16) return to_f32(reinterpret_cast<const bf16*>(w)[i]);
  return reinterpret_cast<const float*>(w)[i];
}

// norm weights of a unit's two chunks, 16-byte loads
__device__ __forceinline__ void norm_weights16(const void* w, int wdt, int c0, int c1, float (&v)[16]) {
  if (wdt == MK_DT_F32) {
    const float* p = reinterpret_cast<const float*>(w);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 a = ldg128(p + 8 * (h ? c1 : c0)), b = ldg128(p + 8 * (h ? c1 : c0) + 4);
      __builtin_memcpy(v + 8 * h, &a, 16);
      __builtin_memcpy(v + 8 * h + 4, &b, 16);
    }
    return;
  }
  const u32x4 a = ldg128(reinterpret_cast<const uint16_t*>(w) + 8 * c0);
  const u32x4 b = ldg128(reinterpret_cast<const uint16_t*>(w) + 8 * c1);
  if (wdt == MK_DT_F16) unpack16<f16>(a, b, v);
  else unpack16<bf16>(a, b, v);
}

// cache row (page * page_size + offset) of token t, -1 where it has none
__device__ __forceinline__ int64_t token_slot(const int32_t* pos, const int32_t* seq, const int32_t* bt,
                                              const QkDims& d, int t) {
  const int64_t p = pos[t];
  const int64_t b = seq ? seq[t] : t;
  if (p < 0 || b < 0 || b >= d.B) return -1;
  const int64_t blk = p / d.page_size;
  if (blk >= d.max_blocks) return -1;
  const int64_t page = bt[b * d.max_blocks + blk];
  return page < 0 || page >= d.num_pages ? -1 : page * d.page_size + (p - blk * d.page_size);
}

// The slot that token t writes, -1 for none.  With one token a sequence (seq
// NULL) the later of two tokens of one slot wins, as in mk_paged_kv_update:
// the workgroup looks through the later tokens.  Every thread takes part.
__device__ __forceinline__ int64_t token_write_slot(const int32_t* pos, const int32_t* seq, const int32_t* bt,
                                                    const QkDims& d, int t) {
  const int64_t slot = token_slot(pos, seq, bt, d, t);
  if (seq) return slot;
  int taken = 0;
  for (int r = t + 1 + (int)threadIdx.x; r < d.T; r += (int)blockDim.x)
    taken |= token_slot(pos, seq, bt, d, r) == slot;
  return __syncthreads_or(taken) ? -1 : slot;
}

// A workgroup has 128 lanes of one token's heads (q heads, then k, then v),
// 1 << lgl lanes a head, of which D / 16 hold a unit each.
template <typename T, int LAYOUT>
__global__ __launch_bounds__(128) void qk_norm_rope_vec_kernel(
    const T* __restrict__ qkv, const void* __restrict__ qw, const void* __restrict__ kw,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t, const int32_t* __restrict__ pos,
    const int32_t* __restrict__ seq, const int32_t* __restrict__ bt, T* __restrict__ Kp, T* __restrict__ Vp,
    T* __restrict__ q_out, int lgl, QkDims d) {
  const int t = blockIdx.x;
  const int at = (int)blockIdx.y * 128 + (int)threadIdx.x;
  const int head = at >> lgl, u = at & ((1 << lgl) - 1);
  const int ru = d.rd >> 4;
  const bool has = head < d.Hq + 2 * d.Hkv && u < (d.D >> 4);
  const bool is_q = head < d.Hq, is_v = head >= d.Hq + d.Hkv;
  int c0, c1;
  unit_chunks<LAYOUT>(u, is_v ? 0 : ru, &c0, &c1);
  u32x4 x0 = {0u, 0u, 0u, 0u}, x1 = {0u, 0u, 0u, 0u};
  if (has) {
    const T* xr = qkv + t * d.row_stride + (int64_t)head * d.D;
    x0 = ldg128(xr + 8 * c0);
    x1 = ldg128(xr + 8 * c1);
  }
  const int64_t p = pos[t];
  const bool live = p >= 0 && p < d.rows && (!seq || (seq[t] >= 0 && seq[t] < d.B));
  int64_t slot = -1;
  // (the last lane's head says whether the workgroup has any to write to the cache)
  if (live && (((int)blockIdx.y * 128 + 127) >> lgl) >= d.Hq) slot = token_write_slot(pos, seq, bt, d, t);
  if (live && !is_v) {
    float v[16];
    unpack16<T>(x0, x1, v);
    const void* w = is_q ? qw : kw;
    if (qw != nullptr) {
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) ss += v[e] * v[e];
      for (int o = 0; o < lgl; ++o) ss += __shfl_xor(ss, 1 << o, MK_WAVE);
      const float inv = rsqrtf(ss / (float)d.D + d.eps);
      if (has) {
        float wv[16];
        norm_weights16(w, d.wdt, c0, c1, wv);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = v[e] * inv * wv[e];
      }
    }
    if (has && u < ru) {
      const size_t a = (size_t)p * (d.rd >> 1) + 8 * u;
      rotate16<LAYOUT>(v, cos_t + a, sin_t + a);
    }
    if (qw != nullptr || u < ru) pack16<T>(v, &x0, &x1);
  }
  if (!has) return;
  T* out;
  if (is_q) {
    if (!live) x0 = x1 = u32x4{0u, 0u, 0u, 0u};
    out = q_out + ((size_t)t * d.Hq + head) * d.D;
  } else {
    if (slot < 0) return;
    out = (is_v ? Vp : Kp) + ((size_t)slot * d.Hkv + (head - d.Hq - (is_v ? d.Hkv : 0))) * d.D;
  }
  *reinterpret_cast<u32x4*>(out + 8 * c0) = x0;
  *reinterpret_cast<u32x4*>(out + 8 * c1) = x1;
}

// any sizes and alignment: a wave per head, four heads of a token a workgroup
template <typename T, int LAYOUT>
__global__ __launch_bounds__(256) void qk_norm_rope_any_kernel(
    const T* __restrict__ qkv, const void* __restrict__ qw, const void* __restrict__ kw,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t, const int32_t* __restrict__ pos,
    const int32_t* __restrict__ seq, const int32_t* __restrict__ bt, T* __restrict__ Kp, T* __restrict__ Vp,
    T* __restrict__ q_out, QkDims d) {
  const int t = blockIdx.x, lane = threadIdx.x & 63;
  const int head = (int)blockIdx.y * 4 + ((int)threadIdx.x >> 6);
  const int64_t p = pos[t];
  const bool live = p >= 0 && p < d.rows && (!seq || (seq[t] >= 0 && seq[t] < d.B));
  int64_t slot = -1;
  if (live && (int)blockIdx.y * 4 + 3 >= d.Hq) slot = token_write_slot(pos, seq, bt, d, t);
  if (head >= d.Hq + 2 * d.Hkv) return;
  const bool is_q = head < d.Hq, is_v = head >= d.Hq + d.Hkv;
  const T* xr = qkv + t * d.row_stride + (int64_t)head * d.D;
  T* out = nullptr;
  if (is_q) out = q_out + ((size_t)t * d.Hq + head) * d.D;
  else if (slot >= 0) out = (is_v ? Vp : Kp) + ((size_t)slot * d.Hkv + (head - d.Hq - (is_v ? d.Hkv : 0))) * d.D;
  if (!out) return;
  if (!live || is_v) {
    for (int i = lane; i < d.D; i += MK_WAVE) out[i] = live ? xr[i] : from_f32<T>(0.0f);
    return;
  }
  const void* w = is_q ? qw : kw;
  float inv = 1.0f;
  if (w) {
    float ss = 0.0f;
    for (int i = lane; i < d.D; i += MK_WAVE) {
      const float v = to_f32(xr[i]);
      ss += v * v;
    }
    inv = rsqrtf(wave_sum(ss) / (float)d.D + d.eps);
  }
  const float* cr = cos_t + (size_t)p * (d.rd >> 1);
  const float* sr = sin_t + (size_t)p * (d.rd >> 1);
  auto value = [&](int i) {
    const float v = to_f32(xr[i]);
    return w ? v * inv * norm_weight(w, d.wdt, i) : v;
  };
  for (int i = lane; i < d.D; i += MK_WAVE) out[i] = from_f32<T>(rotated_value<LAYOUT>(i, d.rd, cr, sr, value));
}

// a call of the kernel for the storage type and the layout
#define MK_ROPE_LAUNCH(KERNEL)                                                        \
  do {                                                                                \
    if (dtype == MK_DT_F16 && layout == kLayoutHalf) KERNEL(f16, kLayoutHalf);        \
    else if (dtype == MK_DT_F16) KERNEL(f16, kLayoutInterleaved);                     \
    else if (layout == kLayoutHalf) KERNEL(bf16, kLayoutHalf);                        \
    else KERNEL(bf16, kLayoutInterleaved);                                            \
  } while (0)

}  // namespace

extern "C" {

int mk_apply_rope(const void* x, const float* cos_t, const float* sin_t, const int32_t* positions, void* y, int64_t B,
                  int64_t S, int64_t H, int64_t D, int64_t stride_b, int64_t stride_s, int64_t stride_h,
                  int64_t rotary_dim, int64_t position_offset, int per_token, int64_t cos_rows, int layout, int dtype,
                  void* stream) {
  MK_REQUIRE(x && y && cos_t && sin_t && B >= 0 && S >= 0 && H >= 0 && D > 0 && D < (1 << 20));
  MK_REQUIRE(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= D && cos_rows > 0);
  MK_REQUIRE(position_offset >= 0 && stride_b >= 0 && stride_s >= 0 && stride_h >= 0);
  MK_REQUIRE(layout == kLayoutInterleaved || layout == kLayoutHalf);
  MK_REQUIRE(dtype == MK_DT_F16 || dtype == MK_DT_BF16);
  MK_REQUIRE(B < (1LL << 31) && S < (1LL << 31) && H < (1LL << 20) && B * S < (1LL << 40));
  if (B == 0 || S == 0 || H == 0) return MK_OK;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t heads = B * S * H;
  const RopeDims d = {S, H, stride_b, stride_s, stride_h, cos_rows, position_offset, (int)D, (int)rotary_dim,
                      positions ? (per_token ? kPosEach : kPosFirst) : kPosOffset};
  // whole units, 16-byte chunks at 16-byte addresses, unit numbers in 32 bits
  const bool vec = D % 16 == 0 && rotary_dim % 16 == 0 && stride_b % 8 == 0 && stride_s % 8 == 0 &&
                   stride_h % 8 == 0 && heads < (1LL << 31) / (D / 16) && mk_aligned(x, 16) && mk_aligned(y, 16) &&
                   mk_aligned(cos_t, 16) && mk_aligned(sin_t, 16);
  if (vec) {
    const uint32_t units = (uint32_t)(heads * (D / 16));
#define MK_RV(T, L)                                                                                             \
  rope_vec_kernel<T, L><<<(units + 255) / 256, 256, 0, st>>>((const T*)x, cos_t, sin_t, positions, (T*)y, units, d)
    MK_ROPE_LAUNCH(MK_RV);
#undef MK_RV
  } else {
    const int64_t want = (heads + 3) / 4;
    const unsigned blocks = (unsigned)(want < 65536 ? want : 65536);
#define MK_RA(T, L) \
  rope_any_kernel<T, L><<<blocks, 256, 0, st>>>((const T*)x, cos_t, sin_t, positions, (T*)y, heads, d)
    MK_ROPE_LAUNCH(MK_RA);
#undef MK_RA
  }
  MK_CHECK_LAUNCH();
  return MK_OK;
}

int mk_qk_norm_rope_paged_update(const void* qkv, int64_t row_stride, const void* q_weight, const void* k_weight,
                                 float eps, const float* cos_t, const float* sin_t, const int32_t* positions,
                                 const int32_t* sequences, const int32_t* block_table, void* K_pages, void* V_pages,
                                 void* q_out, int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                 int64_t rotary_dim, int64_t page_size, int64_t max_blocks, int64_t num_pages,
                                 int64_t cos_rows, int layout, int weight_dtype, int dtype, void* stream) {
  MK_REQUIRE(qkv && cos_t && sin_t && positions && block_table && K_pages && V_pages && q_out);
  MK_REQUIRE(!q_weight == !k_weight);
  MK_REQUIRE(T >= 0 && B >= 0 && Hq > 0 && Hkv > 0 && D > 0 && Hq < (1 << 20) && Hkv < (1 << 20) && D < (1 << 20));
  MK_REQUIRE(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= D && cos_rows > 0);
  MK_REQUIRE(page_size > 0 && max_blocks > 0 && num_pages > 0 && page_size < (1LL << 31));
  MK_REQUIRE(max_blocks < (1LL << 31) && num_pages < (1LL << 31) && B < (1LL << 31));
  MK_REQUIRE(row_stride >= (Hq + 2 * Hkv) * D);
  MK_REQUIRE(sequences ? T < (1LL << 24) : T < 65536 && T == B);
  MK_REQUIRE(layout == kLayoutInterleaved || layout == kLayoutHalf);
  MK_REQUIRE(dtype == MK_DT_F16 || dtype == MK_DT_BF16);
  MK_REQUIRE(weight_dtype == MK_DT_F16 || weight_dtype == MK_DT_BF16 || weight_dtype == MK_DT_F32);
  if (T == 0) return MK_OK;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const QkDims d = {row_stride, page_size, max_blocks, num_pages, cos_rows, (int)T, (int)B, (int)Hq, (int)Hkv,
                    (int)D, (int)rotary_dim, weight_dtype, eps};
  const int64_t heads = Hq + 2 * Hkv;
  // a head's units on at most one wave's lanes
  const bool vec = D % 16 == 0 && D <= 16 * MK_WAVE && rotary_dim % 16 == 0 && row_stride % 8 == 0 &&
                   mk_aligned(qkv, 16) && mk_aligned(q_out, 16) && mk_aligned(K_pages, 16) &&
                   mk_aligned(V_pages, 16) && mk_aligned(cos_t, 16) && mk_aligned(sin_t, 16) &&
                   mk_aligned(q_weight, 16) && mk_aligned(k_weight, 16);
  int lgl = 0;
  while (vec && (16 << lgl) < D) ++lgl;
  const int64_t gy = vec ? ((heads << lgl) + 127) / 128 : (heads + 3) / 4;
  MK_REQUIRE(gy < 65536);
  const dim3 grid((unsigned)T, (unsigned)gy);
#define MK_QV(TT, L)                                                                                              \
  qk_norm_rope_vec_kernel<TT, L><<<grid, 128, 0, st>>>((const TT*)qkv, q_weight, k_weight, cos_t, sin_t, positions, \
                                                       sequences, block_table, (TT*)K_pages, (TT*)V_pages,         \
                                                       (TT*)q_out, lgl, d)
#define MK_QA(TT, L)                                                                                              \
  qk_norm_rope_any_kernel<TT, L><<<grid, 256, 0, st>>>((const TT*)qkv, q_weight, k_weight, cos_t, sin_t, positions, \
                                                       sequences, block_table, (TT*)K_pages, (TT*)V_pages,         \
                                                       (TT*)q_out, d)
  if (vec) MK_ROPE_LAUNCH(MK_QV);
  else MK_ROPE_LAUNCH(MK_QA);
#undef MK_QV
#undef MK_QA
  MK_CHECK_LAUNCH();
  return MK_OK;
}

}  // extern "C"
