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
// unit of work is 16 values, two pieces of 8 that hold the partners of each
// other's values: 8 values and those R/2 further in the half layout, 16 in a
// row in the interleaved one and past R.  So a lane rotates without lane
// exchange and needs 8 cos and 8 sin values; the lanes of a wave that hold the
// same unit of several heads read the same table bytes.  The lanes of a head
// have its sum of squares by shuffles.
//
// WHOLE kernels have D and R in whole units and every address on 16 bytes.
// The others take any sizes and alignment: the last piece of a region starts 8
// values before the region's end, over values that an earlier piece has too
// (both write the same bits), loads are 16 bytes from any address, and only a
// region of under 8 values goes value by value.
//
// 4 x 2047 tokens of 32 heads of 128, bf16: 27 us with R = 64 or 128 (5.1 TB/s,
// what a copy of that size reaches), 30 us with R = 120 (94 us value by value,
// a wave a head).  Norms, rotation and cache write of 8191 tokens of 32 + 2 x 8
// such heads: 43 us (4.8 TB/s), with R = 120 62 us, for 9 of a head's 16 lanes
// have a unit (252 us value by value).  A single token's take 2 and 3 us: they
// are the launch.
#include "common.h"
#include "paged_common.h"

namespace {

constexpr int kLayoutInterleaved = 0;
constexpr int kLayoutHalf = 1;

struct Piece {
  int at, n, skip;  // n <= 8 values from `at` on; the first `skip` are an earlier piece's too
};

// the piece that starts at `at` in the region [lo, hi), moved back into it
__device__ __forceinline__ Piece piece_in(int at, int lo, int hi) {
  const int start = hi - lo < 8 ? lo : at < hi - 8 ? at : hi - 8;
  return {start, hi - lo < 8 ? hi - lo : 8, at - start};
}

// both pieces of unit u of a head of D values, rd of them rotated
template <int LAYOUT, bool WHOLE>
__device__ __forceinline__ void unit_pieces(int u, int rd, int D, Piece* a, Piece* b) {
  const int ru = WHOLE ? rd >> 4 : (rd + 15) >> 4;
  const bool half = LAYOUT == kLayoutHalf && u < ru;
  if constexpr (WHOLE) {
    *a = {half ? 8 * u : 16 * u, 8, 0};
    *b = {half ? 8 * u + (rd >> 1) : 16 * u + 8, 8, 0};
  } else if (half) {
    *a = *b = piece_in(8 * u, 0, rd >> 1);
    b->at += rd >> 1;
  } else {
    const int lo = u < ru ? 0 : rd, hi = u < ru ? rd : D, at = u < ru ? 16 * u : rd + 16 * (u - ru);
    *a = piece_in(at, lo, hi);
    *b = piece_in(at + 8, lo, hi);
  }
}

template <bool WHOLE>
__device__ __forceinline__ u32x4 load_piece(const uint16_t* p, int n) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if constexpr (WHOLE) return ldg128(p);
  else if (n == 8) __builtin_memcpy(&v, p, 16);
  else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) v[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
  }
  return v;
}

template <bool WHOLE>
__device__ __forceinline__ void store_piece(uint16_t* p, int n, const u32x4& v) {
  if constexpr (WHOLE) *reinterpret_cast<u32x4*>(p) = v;
  else if (n == 8) __builtin_memcpy(p, &v, 16);
  else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) p[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
  }
}

// N fp32 values, n of them there (0 where the others are)
template <bool WHOLE, int N>
__device__ __forceinline__ void load_floats(const float* p, int n, float* v) {
  if constexpr (WHOLE) {
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      const u32x4 a = ldg128(p + e);
      __builtin_memcpy(v + e, &a, 16);
    }
  } else if (n == N) {
    __builtin_memcpy(v, p, 4 * N);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = e < n ? p[e] : 0.0f;
  }
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

// the 8 pairs of a rotated unit by the angles of the rows cr and sr
template <int LAYOUT, bool WHOLE>
__device__ __forceinline__ void rotate16(float (&v)[16], const Piece& pa, const Piece& pb, const float* cr,
                                         const float* sr) {
  float c[8], s[8];
  if constexpr (LAYOUT == kLayoutHalf) {
    load_floats<WHOLE, 8>(cr + pa.at, pa.n, c);
    load_floats<WHOLE, 8>(sr + pa.at, pa.n, s);
  } else {
    load_floats<WHOLE, 4>(cr + (pa.at >> 1), pa.n >> 1, c);
    load_floats<WHOLE, 4>(cr + (pb.at >> 1), pb.n >> 1, c + 4);
    load_floats<WHOLE, 4>(sr + (pa.at >> 1), pa.n >> 1, s);
    load_floats<WHOLE, 4>(sr + (pb.at >> 1), pb.n >> 1, s + 4);
  }
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

// where the token of row (b, s) stands: offset + s, pos[b] + offset + s or pos[b, s];
// -1 (a row of zeros) for negative entries and positions outside the tables
constexpr int kPosOffset = 0, kPosFirst = 1, kPosEach = 2;
__device__ __forceinline__ int64_t row_position(const int32_t* pos, int mode, int64_t offset, int64_t b, int64_t s,
                                                int64_t S, int64_t rows) {
  int64_t p = offset + s;
  if (mode != kPosOffset) {
    p = pos[mode == kPosFirst ? b : b * S + s];
    if (p >= 0 && mode == kPosFirst) p += offset + s;
  }
  return p < 0 || p >= rows ? -1 : p;
}

struct RopeDims {
  int64_t S, sb, ss, sh, rows, offset;  // strides of x in values; its last dimension is dense
  int H, D, rd, mode;
};

// a unit per thread, upr of them a head
template <typename T, int LAYOUT, bool WHOLE>
__global__ __launch_bounds__(256) void rope_kernel(const T* __restrict__ x, const float* __restrict__ cos_t,
                                                   const float* __restrict__ sin_t, const int32_t* __restrict__ pos,
                                                   T* __restrict__ y, uint32_t units, uint32_t upr, RopeDims d) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= units) return;
  const uint32_t row = i / upr, t = row / (uint32_t)d.H, b = t / (uint32_t)d.S;
  const int u = (int)(i - row * upr);
  const uint32_t h = row - t * (uint32_t)d.H, s = t - b * (uint32_t)d.S;
  Piece pa, pb;
  unit_pieces<LAYOUT, WHOLE>(u, d.rd, d.D, &pa, &pb);
  const uint16_t* xr = reinterpret_cast<const uint16_t*>(x) + (int64_t)b * d.sb + (int64_t)s * d.ss + (int64_t)h * d.sh;
  const u32x4 x0 = load_piece<WHOLE>(xr + pa.at, pa.n), x1 = load_piece<WHOLE>(xr + pb.at, pb.n);
  const int64_t p = row_position(pos, d.mode, d.offset, b, s, d.S, d.rows);
  u32x4 y0 = {0u, 0u, 0u, 0u}, y1 = {0u, 0u, 0u, 0u};
  if (p >= 0) {
    y0 = x0;
    y1 = x1;
    if (16 * u < d.rd) {
      float v[16];
      unpack16<T>(x0, x1, v);
      rotate16<LAYOUT, WHOLE>(v, pa, pb, cos_t + (size_t)p * (d.rd >> 1), sin_t + (size_t)p * (d.rd >> 1));
      pack16<T>(v, &y0, &y1);
    }
  }
  uint16_t* yr = reinterpret_cast<uint16_t*>(y) + (size_t)row * d.D;
  store_piece<WHOLE>(yr + pa.at, pa.n, y0);
  store_piece<WHOLE>(yr + pb.at, pb.n, y1);
}

// ---------------------------------------------------------------------------
// q and k norms, rotation and the cache write
// ---------------------------------------------------------------------------

struct QkDims {
  int64_t row_stride, page_size, max_blocks, num_pages, rows;  // row_stride of qkv in values
  int T, B, Hq, Hkv, D, rd, wdt;
  float eps;
};

// norm weights of a unit's two pieces
template <bool WHOLE>
__device__ __forceinline__ void norm_weights16(const void* w, int wdt, const Piece& pa, const Piece& pb,
                                               float (&v)[16]) {
  if (wdt == MK_DT_F32) {
    load_floats<WHOLE, 8>(reinterpret_cast<const float*>(w) + pa.at, pa.n, v);
    load_floats<WHOLE, 8>(reinterpret_cast<const float*>(w) + pb.at, pb.n, v + 8);
    return;
  }
  const u32x4 a = load_piece<WHOLE>(reinterpret_cast<const uint16_t*>(w) + pa.at, pa.n);
  const u32x4 b = load_piece<WHOLE>(reinterpret_cast<const uint16_t*>(w) + pb.at, pb.n);
  if (wdt == MK_DT_F16) unpack16<f16>(a, b, v);
  else unpack16<bf16>(a, b, v);
}

// cache row (page * page_size + offset) of token t, -1 where it has none: an
// empty row (no position in the tables, no sequence) has none either
__device__ __forceinline__ int64_t token_slot(const int32_t* pos, const int32_t* seq, const int32_t* bt,
                                              const QkDims& d, int t) {
  const int64_t p = pos[t];
  const int64_t b = seq ? seq[t] : t;
  if (p < 0 || p >= d.rows || b < 0 || b >= d.B) return -1;
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
// 1 << lgl <= 64 lanes a head, each with its units u, u + (1 << lgl), ...  The
// first one stays in registers between the sum of squares and the rotation;
// with over 64 units in a head the others are read twice.
template <typename T, int LAYOUT, bool WHOLE>
__global__ __launch_bounds__(128) void qk_norm_rope_kernel(
    const T* __restrict__ qkv, const void* __restrict__ qw, const void* __restrict__ kw,
    const float* __restrict__ cos_t, const float* __restrict__ sin_t, const int32_t* __restrict__ pos,
    const int32_t* __restrict__ seq, const int32_t* __restrict__ bt, T* __restrict__ Kp, T* __restrict__ Vp,
    T* __restrict__ q_out, int lgl, QkDims d) {
  const int t = blockIdx.x;
  const int at = (int)blockIdx.y * 128 + (int)threadIdx.x;
  const int head = at >> lgl, u0 = at & ((1 << lgl) - 1);
  const bool is_q = head < d.Hq, is_v = head >= d.Hq + d.Hkv;
  const int rd = is_v ? 0 : d.rd;
  const int units = WHOLE ? d.D >> 4 : ((rd + 15) >> 4) + ((d.D - rd + 15) >> 4);
  const bool has = head < d.Hq + 2 * d.Hkv && u0 < units;
  const uint16_t* xr = reinterpret_cast<const uint16_t*>(qkv) + t * d.row_stride + (int64_t)head * d.D;
  Piece pa, pb;
  unit_pieces<LAYOUT, WHOLE>(u0, rd, d.D, &pa, &pb);
  u32x4 x0 = {0u, 0u, 0u, 0u}, x1 = {0u, 0u, 0u, 0u};
  if (has) {
    x0 = load_piece<WHOLE>(xr + pa.at, pa.n);
    x1 = load_piece<WHOLE>(xr + pb.at, pb.n);
  }
  const int64_t p = pos[t];
  const bool live = p >= 0 && p < d.rows && (!seq || (seq[t] >= 0 && seq[t] < d.B));
  int64_t slot = -1;
  // (the last lane's head says whether the workgroup has any to write to the cache)
  if (live && (((int)blockIdx.y * 128 + 127) >> lgl) >= d.Hq) slot = token_write_slot(pos, seq, bt, d, t);
  const bool norm = qw != nullptr && live && !is_v;
  float inv = 1.0f;
  if (norm) {
    float v[16], ss = 0.0f;
    auto add = [&]() {  // the values of x0 and x1 that no earlier unit has (those past a piece's end are 0)
      unpack16<T>(x0, x1, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (WHOLE || e >= pa.skip) ss += v[e] * v[e];
        if (WHOLE || e >= pb.skip) ss += v[8 + e] * v[8 + e];
      }
    };
    add();
    if (units > MK_WAVE) {
      for (int u = u0 + MK_WAVE; has && u < units; u += MK_WAVE) {
        unit_pieces<LAYOUT, WHOLE>(u, rd, d.D, &pa, &pb);
        x0 = load_piece<WHOLE>(xr + pa.at, pa.n);
        x1 = load_piece<WHOLE>(xr + pb.at, pb.n);
        add();
      }
      if (has) {
        unit_pieces<LAYOUT, WHOLE>(u0, rd, d.D, &pa, &pb);
        x0 = load_piece<WHOLE>(xr + pa.at, pa.n);
        x1 = load_piece<WHOLE>(xr + pb.at, pb.n);
      }
    }
    for (int o = 0; o < lgl; ++o) ss += __shfl_xor(ss, 1 << o, MK_WAVE);
    inv = rsqrtf(ss / (float)d.D + d.eps);
  }
  if (!has || (!is_q && slot < 0)) return;
  uint16_t* out = reinterpret_cast<uint16_t*>(is_q ? q_out : is_v ? Vp : Kp);
  if (is_q) out += ((size_t)t * d.Hq + head) * d.D;
  else out += ((size_t)slot * d.Hkv + (head - d.Hq - (is_v ? d.Hkv : 0))) * d.D;
  for (int u = u0;;) {
    if (!live) x0 = x1 = u32x4{0u, 0u, 0u, 0u};
    else if (norm || 16 * u < rd) {
      float v[16];
      unpack16<T>(x0, x1, v);
      if (norm) {
        float wv[16];
        norm_weights16<WHOLE>(is_q ? qw : kw, d.wdt, pa, pb, wv);
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = v[e] * inv * wv[e];
      }
      if (16 * u < rd)
        rotate16<LAYOUT, WHOLE>(v, pa, pb, cos_t + (size_t)p * (d.rd >> 1), sin_t + (size_t)p * (d.rd >> 1));
      pack16<T>(v, &x0, &x1);
    }
    store_piece<WHOLE>(out + pa.at, pa.n, x0);
    store_piece<WHOLE>(out + pb.at, pb.n, x1);
    u += MK_WAVE;
    if (u >= units) return;
    unit_pieces<LAYOUT, WHOLE>(u, rd, d.D, &pa, &pb);
    x0 = load_piece<WHOLE>(xr + pa.at, pa.n);
    x1 = load_piece<WHOLE>(xr + pb.at, pb.n);
  }
}

// units of a head
int64_t units_of(int64_t D, int64_t rd) { return (rd + 15) / 16 + (D - rd + 15) / 16; }

// a call of the kernel for the storage type, the layout and whole or other units
#define MK_ROPE_LAUNCH(KERNEL, W)                                                     \
  do {                                                                                \
    if (dtype == MK_DT_F16 && layout == kLayoutHalf) KERNEL(f16, kLayoutHalf, W);     \
    else if (dtype == MK_DT_F16) KERNEL(f16, kLayoutInterleaved, W);                  \
    else if (layout == kLayoutHalf) KERNEL(bf16, kLayoutHalf, W);                     \
    else KERNEL(bf16, kLayoutInterleaved, W);                                         \
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
  const int64_t upr = units_of(D, rotary_dim), token = H * upr;
  MK_REQUIRE(token < (1LL << 31));
  // whole units, 16-byte pieces at 16-byte addresses
  const bool whole = D % 16 == 0 && rotary_dim % 16 == 0 && stride_b % 8 == 0 && stride_s % 8 == 0 &&
                     stride_h % 8 == 0 && mk_aligned(x, 16) && mk_aligned(y, 16) && mk_aligned(cos_t, 16) &&
                     mk_aligned(sin_t, 16);
  // unit numbers fit in 31 bits: a launch for whole sequences or, of longer ones, for some rows of one
  const int64_t most = ((1LL << 31) - 1) / token;
  const int64_t nb = S <= most ? most / S : 1, ns = S <= most ? S : most;
  for (int64_t b0 = 0; b0 < B; b0 += nb) {
    for (int64_t s0 = 0; s0 < S; s0 += ns) {
      const int64_t b = B - b0 < nb ? B - b0 : nb, s = S - s0 < ns ? S - s0 : ns;
      const RopeDims d = {s, stride_b, stride_s, stride_h, cos_rows, (positions ? 0 : position_offset) + s0, (int)H,
                          (int)D, (int)rotary_dim, positions ? (per_token ? kPosEach : kPosFirst) : kPosOffset};
      const uint16_t* xs = (const uint16_t*)x + b0 * stride_b + s0 * stride_s;
      uint16_t* ys = (uint16_t*)y + (b0 * S + s0) * H * D;
      const int32_t* ps = positions ? positions + (per_token ? b0 * S + s0 : b0) : nullptr;
      const uint32_t units = (uint32_t)(b * s * token);
#define MK_R(T, L, W)                                                                                       \
  rope_kernel<T, L, W><<<(units + 255) / 256, 256, 0, st>>>((const T*)xs, cos_t, sin_t, ps, (T*)ys, units, \
                                                            (uint32_t)upr, d)
      if (whole) MK_ROPE_LAUNCH(MK_R, true);
      else MK_ROPE_LAUNCH(MK_R, false);
#undef MK_R
      MK_CHECK_LAUNCH();
    }
  }
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
  const bool whole = D % 16 == 0 && rotary_dim % 16 == 0 && row_stride % 8 == 0 && mk_aligned(qkv, 16) &&
                     mk_aligned(q_out, 16) && mk_aligned(K_pages, 16) && mk_aligned(V_pages, 16) &&
                     mk_aligned(cos_t, 16) && mk_aligned(sin_t, 16) && mk_aligned(q_weight, 16) &&
                     mk_aligned(k_weight, 16);
  int lgl = 0;
  while ((1 << lgl) < MK_WAVE && (1 << lgl) < units_of(D, rotary_dim)) ++lgl;
  const int64_t gy = ((heads << lgl) + 127) / 128;
  MK_REQUIRE(gy < 65536);
  const dim3 grid((unsigned)T, (unsigned)gy);
#define MK_Q(TT, L, W)                                                                                              \
  qk_norm_rope_kernel<TT, L, W><<<grid, 128, 0, st>>>((const TT*)qkv, q_weight, k_weight, cos_t, sin_t, positions, \
                                                      sequences, block_table, (TT*)K_pages, (TT*)V_pages,          \
                                                      (TT*)q_out, lgl, d)
  if (whole) MK_ROPE_LAUNCH(MK_Q, true);
  else MK_ROPE_LAUNCH(MK_Q, false);
#undef MK_Q
  MK_CHECK_LAUNCH();
  return MK_OK;
}

}  // extern "C"
