// Low-rank adapters of many requests beside a shared projection:
//
//   out[m] = base[m] + s_i B_i (A_i x[m]),  i = ids[m]   (i outside [0, adapters): out[m] = base[m])
//
// No counterpart in the reference.  The rows of one adapter, up to 64 of them,
// are a group.  One launch sums t = A_i x[m] of a group's rows in fp32 (in
// slices of K, kept in the workspace), the next joins the slices, multiplies
// by B_i and adds base, with one rounding.  Up to 64 rows, or 256 of few
// adapters, a wave finds its group by itself; beyond, a launch before them
// lists the groups.  So every adapter's matrices are read once for 64 rows,
// whatever the rows' order.  A single row of few ranks takes one launch.
//
// Few rows are bound by trips to memory one after another (32 rows, K 4096, N
// 6144, rank 16: 4.2 and 5.1 us for 3.7 MB), many by the streams of x, base and
// out: 4093 rows, K 4096, N 14336, rank 64: 7, 18 and 60 us for 280 MB, which a
// copy moves in 52.
//
// Both products run on 16x16x32 matrix instructions with the rows as columns:
// a row's values touch no other row (an infinity or NaN stays where it is),
// and which rows share a group changes no result.
//
// The second product's operand t is 32 bits: it goes in as the sum of two
// values of the storage type (relative 2^-16 for bf16, 2^-21 for fp16), in fp16
// scaled by a power of two per row so that neither part leaves its range: fp16's
// smallest step is then 2^-38 of the row's largest value of t, and ranks below
// that are lost.  Matrix instructions take both operands in one type, B is read
// in the storage type, and the result's rounding (2^-8, 2^-11) is far above both.
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

// two values in one conversion
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (__is_same(T, bf16)) {
    return bitcast<uint32_t>(__builtin_convertvector((f32x2){a, b}, bf16x2));
  } else {
    return bitcast<uint32_t>(f16x2{(f16)a, (f16)b});
  }
}

// 16 and 8 bytes from and to any address of a value
__device__ __forceinline__ u32x4 load16(const void* p) {
  u32x4 v;
  __builtin_memcpy(&v, (const uint16_t*)p, 16);
  return v;
}
typedef u32x2 __attribute__((aligned(2))) u32x2_any;
__device__ __forceinline__ u32x2 load8(const void* p) {
  u32x2 v;
  __builtin_memcpy(&v, (const uint16_t*)p, 8);
  return v;
}

// Rows along which a fragment of 8 values is read: of whole fragments; with a
// rest; of fewer than 8 values.
enum Len { kFew, kRest, kWhole };
inline Len len_of(int64_t n) { return n < 8 ? kFew : n % 8 ? kRest : kWhole; }

// 8 values p[at .. at + 8) of a row that ends at `end`, zeros behind it and
// where `ok` is false.  No branch but with under 8 values in all, so that loads
// stay in flight beside it: a fragment with the end in it is read from 8 before
// the end and moved down.
template <typename T, Len LEN>
__device__ __forceinline__ typename Frag<T>::v8 load_frag(const T* p, int64_t at, int64_t end, bool ok = true) {
  typename Frag<T>::v8 v;
  if constexpr (LEN == kWhole) {
    ok = ok && at < end;
    u32x4 w = load16(p + (at < end ? at : 0));
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = ok ? w[e] : 0u;
    v = bitcast<typename Frag<T>::v8>(w);
  } else if constexpr (LEN == kRest) {
    const int64_t from = at < end - 8 ? at : end - 8;
    const u32x4 w = load16(p + from);
    const int s = at - from < 8 ? 16 * (int)(at - from) : 128;  // bits
    const uint64_t lo = w[0] | (uint64_t)w[1] << 32, hi = w[2] | (uint64_t)w[3] << 32;
    uint64_t x = s < 64 ? lo >> s | (hi << 1) << (63 - s) : hi >> (s & 63), y = s < 64 ? hi >> s : 0;
    x = ok && s < 128 ? x : 0;
    y = ok ? y : 0;
    v = bitcast<typename Frag<T>::v8>(u32x4{(uint32_t)x, (uint32_t)(x >> 32), (uint32_t)y, (uint32_t)(y >> 32)});
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = ok && at + e < end ? p[at + e] : from_f32<T>(0.0f);
  }
  return v;
}

// ---------------------------------------------------------------------------
// groups: up to 64 rows of one adapter
// ---------------------------------------------------------------------------

constexpr int kGroupRows = 64;
// What a wave groups by itself beyond 64 rows.  Against a launch that lists the
// groups, K and N 4096, rank 16, us a call: 100 rows of 5 adapters 11.2 / 14.0,
// of 8 11.3 / 13.9, of 15 16.4 / 14.1; 256 rows 13.0 / 15.5, 14.1 / 15.6, 19.2
// / 15.7.
constexpr int kWaveRows = 256, kWaveAdapters = 8;
constexpr int kMaxAdapters = 4096;

struct Groups {
  const int32_t* ids;
  const int32_t* rows;      // [groups, 64], -1 behind a group's rows; NULL: the waves look for them
  const int32_t* adapters;  // [groups + 1]: the adapter of each (-1: none), in front of them their number
  int64_t M;
  int count;  // of adapters
};

// Group g of 65 to 256 rows, by a wave: adapters in the order of their first
// rows, the rows of each in order.
__device__ __forceinline__ int sort_out(const Groups& gs, int g, int* adapter, int* row) {
  constexpr int J = kWaveRows / 64;
  const int lane = threadIdx.x & 63;
  const uint64_t below = (1ull << lane) - 1;
  int id[J];
  uint64_t rest[J], have[J];
#pragma unroll
  for (int j = 0; j < J; ++j) id[j] = lane + 64 * j < gs.M ? gs.ids[lane + 64 * j] : -1;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if (id[j] < 0 || id[j] >= gs.count) id[j] = -1;
    rest[j] = __ballot(lane + 64 * j < gs.M);
  }
  for (;;) {
    bool any = false;
    int n = 0;
#pragma unroll
    for (int j = J - 1; j >= 0; --j)
      if (rest[j]) {
        *adapter = __builtin_amdgcn_readlane(id[j], __builtin_ctzll(rest[j]));
        any = true;
      }
    if (!any) return 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      have[j] = __ballot(id[j] == *adapter) & rest[j];
      rest[j] &= ~have[j];
      n += __builtin_popcountll(have[j]);
    }
    const int groups = (n + kGroupRows - 1) / kGroupRows;
    if (g < groups) break;
    g -= groups;
  }
  // the rows from 64 g on of those, the i-th to lane i; every lane sends, the others to the lanes that take nothing
  int before = -kGroupRows * g;
  *row = -1;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int rank = before + __builtin_popcountll(have[j] & below);
    const bool in = (have[j] >> lane) & 1 && rank >= 0 && rank < kGroupRows;
    const uint64_t members = __ballot(in);
    const int first = before > 0 ? before : 0, k = __builtin_popcountll(members);
    const int to = in ? rank : (first + k + __builtin_popcountll(~members & below)) & 63;
    const int got = __builtin_amdgcn_ds_permute(4 * to, lane + 64 * j);
    if (lane >= first && lane < first + k) *row = got;
    before += __builtin_popcountll(have[j]);
  }
  return before < kGroupRows ? before : kGroupRows;
}

// Group g: its adapter (-1: rows without one), its rows (row i in lane i, -1
// behind them), their number (0: there is no such group).  Uniform but `row`.
__device__ __forceinline__ int find_group(const Groups& gs, int g, int* adapter, int* row) {
  if (gs.rows) {
    if (g >= gs.adapters[0]) return 0;
    *adapter = gs.adapters[1 + g];
    *row = gs.rows[(int64_t)g * kGroupRows + (threadIdx.x & 63)];
    return __builtin_popcountll(__ballot(*row >= 0));
  }
  if (gs.M > kGroupRows) return sort_out(gs, g, adapter, row);
  const int lane = threadIdx.x & 63;
  int id = lane < gs.M ? gs.ids[lane] : -1;
  if (id < 0 || id >= gs.count) id = -1;
  uint64_t rest = __ballot(lane < gs.M), have = 0;
  for (int k = 0; k <= g; ++k) {
    if (rest == 0) return 0;
    *adapter = __builtin_amdgcn_readlane(id, __builtin_ctzll(rest));
    have = __ballot(id == *adapter) & rest;
    rest &= ~have;
  }
  // lane i of the group's rows sends its number to lane i; the others to lanes behind them
  const int n = __builtin_popcountll(have);
  const uint64_t below = (1ull << lane) - 1;
  const bool in = (have >> lane) & 1;
  const int to = in ? __builtin_popcountll(have & below) : n + __builtin_popcountll(~have & below);
  *row = __builtin_amdgcn_ds_permute(4 * to, in ? lane : -1);
  return n;
}

// The groups of more rows, by one workgroup.  Rows of an adapter take
// places in the order in which the threads get there: which rows share a group
// changes no result.
__global__ __launch_bounds__(1024) void lora_group_kernel(const int32_t* __restrict__ ids, int32_t* __restrict__ rows,
                                                          int32_t* __restrict__ adapters, int64_t M, int count) {
  __shared__ int number[kMaxAdapters + 1];  // rows of each adapter; `count`: of none
  __shared__ int first[kMaxAdapters + 1];   // its first group
  __shared__ int sums[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i <= count; i += 1024) number[i] = 0;
  __syncthreads();
  // a row's place: one addition for the rows of a wave that share the first's adapter
  auto take = [&](int bin, bool live) {
    const uint64_t all = __ballot(live);
    if (all == 0) return 0;
    const int head = __builtin_ctzll(all);
    const int lead = __builtin_amdgcn_readlane(bin, head);
    const uint64_t same = __ballot(live && bin == lead);
    int at = 0;
    if (lane == head) at = atomicAdd(&number[lead], (int)__builtin_popcountll(same));
    at = __builtin_amdgcn_readlane(at, head) + (int)__builtin_popcountll(same & ((1ull << lane) - 1));
    if (live && bin != lead) at = atomicAdd(&number[bin], 1);
    return at;
  };
  constexpr int ROWS = 8;  // of a thread, their ids on the way together
  int bin[ROWS], at[ROWS];
  auto read = [&](int64_t m0) {
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      const int64_t m = m0 + 1024 * u + tid;
      bin[u] = ids[m < M ? m : 0];
    }
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      if (bin[u] < 0 || bin[u] >= count) bin[u] = count;
      const int64_t m = m0 + 1024 * u;
      if (m < M) at[u] = take(bin[u], m + tid < M);  // (uniform)
    }
  };
  for (int64_t m0 = 0; m0 < M; m0 += 1024 * ROWS) read(m0);
  __syncthreads();
  // groups of each adapter, their sum up to it; a thread has a run of adapters
  const int per = (count + 1 + 1023) / 1024, lo = tid * per, hi = min(lo + per, count + 1);
  int mine = 0;
  for (int i = lo; i < hi; ++i) mine += (number[i] + kGroupRows - 1) / kGroupRows;
  int s = mine;
#pragma unroll
  for (int o = 1; o < MK_WAVE; o <<= 1) {
    const int up = __shfl_up(s, o, MK_WAVE);
    if (lane >= o) s += up;
  }
  if (lane == 63) sums[wave] = s;
  __syncthreads();
  int before = s - mine, total = 0;
  for (int w = 0; w < 16; ++w) {
    if (w < wave) before += sums[w];
    total += sums[w];
  }
  if (tid == 0) adapters[0] = total;
  for (int i = lo; i < hi; ++i) {
    first[i] = before;
    const int n = number[i], groups = (n + kGroupRows - 1) / kGroupRows;
    for (int g = 0; g < groups; ++g) adapters[1 + before + g] = i < count ? i : -1;
    for (int r = n; r < groups * kGroupRows; ++r) rows[(int64_t)before * kGroupRows + r] = -1;
    before += groups;
    number[i] = 0;
  }
  __syncthreads();
  for (int64_t m0 = 0; m0 < M; m0 += 1024 * ROWS) {
    if (M > 1024 * ROWS) read(m0);  // (else the places are those from before)
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
      const int64_t m = m0 + 1024 * u + tid;
      if (m < M) rows[(int64_t)first[bin[u]] * kGroupRows + at[u]] = (int32_t)m;
    }
  }
}

// ---------------------------------------------------------------------------
// t = A x: a workgroup of 8 waves has a group, or half of one, and a slice of
// K; its waves take turns of 32 values of K and are summed through LDS.  The
// product is A (ranks down) times x (rows across): a lane ends with 4 ranks of
// a row.  The order in which a row's values are added depends on no other row
// and not on its place among them.  It does depend on the slices of K, which go
// by K and by how many rows and stacked adapters the call has (lora_plan), and a
// call of a single row may take lora_one_kernel, whose order is another one.
// ---------------------------------------------------------------------------

constexpr int kShrinkWaves = 8;

// put(i, row, r, s): ranks r .. r + 3 of the group's row number i
template <typename T, int RT, int MT, Len LEN, typename Put>
__device__ __forceinline__ void shrink_rows(const T* x, int64_t x_stride, const T* ai, int64_t K, int R, int64_t k0,
                                            int64_t k1, int rowlist, f32x4 (&part)[kShrinkWaves][RT][64], Put put) {
  constexpr bool AHEAD = LEN != kFew && RT * MT <= 16;  // (more would not fit the registers)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, grp = lane >> 4;
  const int any = __builtin_amdgcn_readfirstlane(rowlist);
  int row[MT];
  const T* xr[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    row[i] = __shfl(rowlist, 16 * i + col, MK_WAVE);
    xr[i] = x + (int64_t)(row[i] < 0 ? any : row[i]) * x_stride;
  }
  f32x4 acc[RT][MT];
#pragma unroll
  for (int q = 0; q < RT; ++q)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[q][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Turn {
    typename Frag<T>::v8 x[MT], a[RT];
  };
  auto load = [&](int64_t kb) {
    Turn f;
    const int64_t k = kb + 8 * grp;
#pragma unroll
    for (int i = 0; i < MT; ++i) f.x[i] = load_frag<T, LEN>(xr[i], k, k1);
#pragma unroll
    for (int q = 0; q < RT; ++q) {
      const int r = 16 * q + col;
      f.a[q] = load_frag<T, LEN>(ai + (int64_t)(r < R ? r : 0) * K, k, k1, r < R);
    }
    return f;
  };
  auto multiply = [&](const Turn& f) {
#pragma unroll
    for (int q = 0; q < RT; ++q)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[q][i] = Frag<T>::mfma(f.a[q], f.x[i], acc[q][i]);
  };
  constexpr int64_t step = 32 * kShrinkWaves;
  int64_t kb = k0 + 32 * wave;
  if constexpr (AHEAD) {  // the next turn is on its way while one is multiplied
    if (kb < k1) {
      Turn cur = load(kb);
      for (kb += step; kb < k1; kb += step) {
        const Turn next = load(kb);
        multiply(cur);
        cur = next;
      }
      multiply(cur);
    }
  } else {
    for (; kb < k1; kb += step) multiply(load(kb));
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    if (i) __syncthreads();  // the last rows' sums are read
#pragma unroll
    for (int q = 0; q < RT; ++q) part[wave][q][lane] = acc[q][i];
    __syncthreads();
    for (int q = wave; q < RT; q += kShrinkWaves) {
      f32x4 s = part[0][q][lane];
#pragma unroll
      for (int w = 1; w < kShrinkWaves; ++w) s += part[w][q][lane];
      put(16 * i + col, row[i], 16 * q + 4 * grp, s);
    }
  }
}

template <typename T, int RT, Len LEN, typename Put>
__device__ __forceinline__ void shrink_group(const T* x, int64_t x_stride, const T* ai, int64_t K, int R, int64_t k0,
                                             int64_t k1, int n, int rowlist, f32x4 (&part)[kShrinkWaves][RT][64],
                                             Put put) {
  if constexpr (LEN != kFew) {
    if (n <= 16) shrink_rows<T, RT, 1, LEN>(x, x_stride, ai, K, R, k0, k1, rowlist, part, put);
    else if (n <= 32) shrink_rows<T, RT, 2, LEN>(x, x_stride, ai, K, R, k0, k1, rowlist, part, put);
    else shrink_rows<T, RT, 4, LEN>(x, x_stride, ai, K, R, k0, k1, rowlist, part, put);
  } else {  // values one by one: 16 rows at a time leave the registers for them
    for (int i = 0; i < n; i += 16) {
      const int at = ((int)threadIdx.x & 63) + i;
      const int row = __shfl(rowlist, at & 63, MK_WAVE);
      if (i) __syncthreads();  // the last rows' sums are read
      shrink_rows<T, RT, 1, LEN>(x, x_stride, ai, K, R, k0, k1, at < 64 ? row : -1, part,
                                 [&](int j, int m, int r, const f32x4& s) { put(i + j, m, r, s); });
    }
  }
}

template <typename T, int RT, Len LEN>
__global__ __launch_bounds__(64 * kShrinkWaves) void lora_shrink_kernel(Groups gs, const T* __restrict__ x,
                                                                        int64_t x_stride, const T* __restrict__ a,
                                                                        float* __restrict__ t, int64_t K, int R,
                                                                        int64_t k_slice, int rows) {
  __shared__ f32x4 part[kShrinkWaves][RT][64];
  int adapter, rowlist;
  const int parts = kGroupRows / rows, r0 = (int)blockIdx.x % parts * rows;
  int n = find_group(gs, (int)blockIdx.x / parts, &adapter, &rowlist);
  if (n <= r0 || adapter < 0) return;
  if (r0 > 0 || n > rows) {
    n = n - r0 < rows ? n - r0 : rows;
    const int lane = (int)threadIdx.x & 63, row = __shfl(rowlist, (r0 + lane) & 63, MK_WAVE);
    rowlist = lane < n ? row : -1;
  }
  const int64_t k0 = (int64_t)blockIdx.y * k_slice;
  const int64_t k1 = k0 + k_slice < K ? k0 + k_slice : K;
  const T* ai = a + (int64_t)adapter * R * K;
  t += (int64_t)blockIdx.y * gs.M * (16 * RT);
  shrink_group<T, RT, LEN>(x, x_stride, ai, K, R, k0, k1, n, rowlist, part,
                           [&](int, int m, int r, f32x4 s) {
#pragma unroll
                             for (int e = 0; e < 4; ++e) s[e] = r + e < R ? s[e] : 0.0f;  // (0 x infinity behind R)
                             if (m >= 0) *reinterpret_cast<f32x4*>(t + (int64_t)m * (16 * RT) + r) = s;
                           });
}

// ---------------------------------------------------------------------------
// out = base + s B t: a workgroup of 4 waves has a group and `blocks` times
// 256 outputs.  It puts both parts of t of its rows into LDS; then each wave
// takes 64 outputs at a time.  The product is t (rows down) times B (outputs
// across).  Instruction j has the outputs 4 c + j for its columns c, so that a
// lane ends with 4 outputs side by side of 4 rows, and an access of 8 bytes a
// lane covers 128 bytes each of 4 rows.  Bound by the base and out streams, for
// which the 128 bytes count: copying 4093 rows x 14336 in 64-byte pieces takes
// 57 us, in these 47.
// ---------------------------------------------------------------------------

template <typename T, int RT>
struct ExpandRows {
  typedef typename Frag<T>::v8 v8;
  static constexpr int RP = 16 * RT;               // ranks, whole tiles
  static constexpr int KS = RT == 1 ? 1 : RT / 2;  // up to 16 ranks: both parts in one instruction, over B twice
  static constexpr int CH = RP / 8;                // chunks of 8 ranks
  T parts[kGroupRows][2 * RP + 8];                 // both parts of t; 16 bytes that spread the rows over the banks
  f32x4 backs[kGroupRows / 4];
  int64_t at_base[kGroupRows], at_out[kGroupRows];  // where the rows begin: products of 64 bits are slow

  // chunk c of row i, by CH lanes side by side, a power of two
  __device__ __forceinline__ void put(int i, int c, float (&v)[8], float back, bool live) {
    if constexpr (__is_same(T, f16)) {  // the row's largest finite value to [2^13, 2^14)
      float top = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fabsf(v[e]) < INFINITY ? fmaxf(top, fabsf(v[e])) : top;
#pragma unroll
      for (int o = 1; o < CH; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, MK_WAVE));
      int e = 14;
      if (top > 0.0f) (void)frexpf(top, &e);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = ldexpf(v[q], 14 - e);
      back = ldexpf(back, e - 14);
    }
    v8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      hi[e] = from_f32<T>(v[e]);
      const float left = v[e] - to_f32(hi[e]);
      lo[e] = from_f32<T>(fabsf(v[e]) < INFINITY ? left : 0.0f);
    }
    if (!live) return;
    *reinterpret_cast<v8*>(&parts[i][8 * c]) = hi;
    *reinterpret_cast<v8*>(&parts[i][RP + 8 * c]) = lo;
    if (c == 0) reinterpret_cast<float*>(backs)[i] = back;
  }
};

// B's fragments of 64 outputs from n0 on
template <typename T, int RT, Len LEN>
__device__ __forceinline__ void load_b(const T* bi, int64_t n0, int64_t N, int R,
                                       typename Frag<T>::v8 (&bf)[4][ExpandRows<T, RT>::KS]) {
  const int col = threadIdx.x & 15, grp = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t r = n0 + 4 * col + j;
#pragma unroll
    for (int s = 0; s < ExpandRows<T, RT>::KS; ++s)
      bf[j][s] = load_frag<T, LEN>(bi + (r < N ? r : N - 1) * R, RT == 1 ? 8 * (grp & 1) : 32 * s + 8 * grp, R);
  }
}

// Rows without an adapter: outputs c0 .. c1 of them copied, by a workgroup, 4
// side by side a thread and those of 4 places of the rows on their way together
// (a row at a time is 64 trips to memory one after another).
template <typename T>
__device__ __forceinline__ void copy_rows(const T* base, int64_t base_stride, T* out, int64_t out_stride, int64_t c0,
                                          int64_t c1, int n, int rowlist) {
  constexpr int UN = 4;
  const int width = (int)(c1 - c0), chunks = (width + 3) / 4, all = n * chunks;
  for (int at0 = 0; at0 < all; at0 += UN * (int)blockDim.x) {
    u32x2 w[UN];
    const T* br[UN];
    T* orow[UN];
    int left[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int at = at0 + u * (int)blockDim.x + (int)threadIdx.x, i = at / chunks, c = at - i * chunks;
      const int64_t m = __shfl(rowlist, i & 63, MK_WAVE);  // (every lane: the source has to be active)
      br[u] = base + m * base_stride + c0 + 4 * c;
      orow[u] = out + m * out_stride + c0 + 4 * c;
      left[u] = at < all ? width - 4 * c : 0;
      if (left[u] >= 4) w[u] = load8(br[u]);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      if (left[u] >= 4) *reinterpret_cast<u32x2_any*>(orow[u]) = w[u];
      else for (int e = 0; e < left[u]; ++e) orow[u][e] = br[u][e];
    }
  }
}

// 64 outputs from n0 on of a group's n rows, by a wave
template <typename T, int RT>
__device__ __forceinline__ void expand_rows(const ExpandRows<T, RT>& l, const T* base, T* out, int64_t N, int64_t n0,
                                            int n, const typename Frag<T>::v8 (&bf)[4][ExpandRows<T, RT>::KS]) {
  typedef ExpandRows<T, RT> L;
  typedef typename L::v8 v8;
  const int col = threadIdx.x & 15, grp = (threadIdx.x & 63) >> 4;
  const int64_t nn = n0 + 4 * col;  // this lane's first output
  auto product = [&](int rt, f32x4 (&acc)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const T* pr = l.parts[16 * rt + col];
#pragma unroll
    for (int s = 0; s < L::KS; ++s) {
      if constexpr (RT == 1) {  // chunks 0 and 1 of the first part, then of the second
        const v8 both = *reinterpret_cast<const v8*>(pr + 8 * grp);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = Frag<T>::mfma(both, bf[j][s], acc[j]);
      } else {
        const v8 hi = *reinterpret_cast<const v8*>(pr + 32 * s + 8 * grp);
        const v8 lo = *reinterpret_cast<const v8*>(pr + L::RP + 32 * s + 8 * grp);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = Frag<T>::mfma(hi, bf[j][s], acc[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = Frag<T>::mfma(lo, bf[j][s], acc[j]);
      }
    }
  };
  const T* bn = base + nn;
  T* on = out + nn;
  // outputs 4 side by side: the sums of row i of 4 on base's values
  auto join = [&](const f32x4 (&acc)[4], float back, int i, u32x2 w) {
    u32x2 o;
#pragma unroll
    for (int j = 0; j < 4; j += 2)
      o[j >> 1] = pack2<T>(fmaf(acc[j][i], back, to_f32(bitcast<T>((uint16_t)w[j >> 1]))),
                           fmaf(acc[j + 1][i], back, to_f32(bitcast<T>((uint16_t)(w[j >> 1] >> 16)))));
    return o;
  };
  int rt = 0;
  if (n0 + 64 <= N && n >= 16) {
    // whole tiles, without a branch: base of the next 16 rows is on its way while these are computed
    const int whole = n / 16;
    u32x2 w[4], next[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = load8(bn + l.at_base[4 * grp + i]);
    for (; rt < whole; ++rt) {
      const int then = 16 * (rt + 1 < whole ? rt + 1 : rt) + 4 * grp;
#pragma unroll
      for (int i = 0; i < 4; ++i) next[i] = load8(bn + l.at_base[then + i]);
      f32x4 acc[4];
      product(rt, acc);
      const f32x4 back = l.backs[4 * rt + grp];
#pragma unroll
      for (int i = 0; i < 4; ++i)  // (streamed: 4093 rows x 14336 in 88.8 us, 90.6 by way of the L2)
        __builtin_nontemporal_store(join(acc, back[i], i, w[i]),
                                    reinterpret_cast<u32x2_any*>(on + l.at_out[16 * rt + 4 * grp + i]));
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = next[i];
    }
  }
  const bool four = nn + 4 <= N;
  for (; 16 * rt < n; ++rt) {
    u32x2 w[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * rt + 4 * grp + i;
      if (four) w[i] = load8(bn + l.at_base[r < n ? r : 0]);
    }
    f32x4 acc[4];
    product(rt, acc);
    const f32x4 back = l.backs[4 * rt + grp];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 16 * rt + 4 * grp + i;
      if (r >= n) continue;
      if (four) {
        *reinterpret_cast<u32x2_any*>(on + l.at_out[r]) = join(acc, back[i], i, w[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (nn + j < N) on[l.at_out[r] + j] = from_f32<T>(fmaf(acc[j][i], back[i], to_f32(bn[l.at_base[r] + j])));
      }
    }
  }
}

template <typename T, int RT, Len LEN>
__global__ __launch_bounds__(256) void lora_expand_kernel(Groups gs, const T* base, int64_t base_stride,
                                                          const T* __restrict__ b, const float* __restrict__ scales,
                                                          const float* __restrict__ t, T* out, int64_t out_stride,
                                                          int64_t N, int R, int slices, int blocks) {
  typedef ExpandRows<T, RT> L;
  __shared__ L l;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int adapter, rowlist;
  const int n = find_group(gs, (int)blockIdx.y, &adapter, &rowlist);
  if (n == 0 || (adapter < 0 && base == out)) return;
  if (adapter < 0) {
    const int64_t c0 = (int64_t)blockIdx.x * blocks * 256;
    copy_rows(base, base_stride, out, out_stride, c0, c0 + 256 * blocks < N ? c0 + 256 * blocks : N, n, rowlist);
    return;
  }
  if (wave == 0) {
    l.at_base[lane] = rowlist * base_stride;
    l.at_out[lane] = rowlist * out_stride;
  }
  const T* bi = b + (int64_t)adapter * N * R;
  typename L::v8 bf[4][L::KS];
  int64_t n0 = ((int64_t)blockIdx.x * blocks * 4 + wave) * 64;
  load_b<T, RT, LEN>(bi, n0, N, R, bf);  // on the way while t is joined
  const float scale = scales ? scales[adapter] : 1.0f;
  const int chunks = ((n + 15) & ~15) * L::CH;
  for (int at0 = 0; at0 < chunks; at0 += 256) {
    const int at = at0 + (int)threadIdx.x, i = at / L::CH, c = at % L::CH;
    const int row = __shfl(rowlist, i & 63, MK_WAVE);  // (every lane: the source has to be active)
    const int m = at < chunks ? row : -1;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (m >= 0) {
      const float* tr = t + (int64_t)m * L::RP + 8 * c;
      const int64_t step = gs.M * L::RP;
      for (int z = 0; z < slices; z += 4) {  // four slices on their way together
        f32x4 lo[4], hi[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          lo[u] = hi[u] = f32x4{0.f, 0.f, 0.f, 0.f};
          if (z + u < slices) {
            lo[u] = *reinterpret_cast<const f32x4*>(tr + (z + u) * step);
            hi[u] = *reinterpret_cast<const f32x4*>(tr + (z + u) * step + 4);
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] += lo[u][e];
            v[4 + e] += hi[u][e];
          }
      }
    }
    l.put(i, c, v, scale, at < chunks);
  }
  lds_barrier();  // (the loads of B stay in flight)
  for (int blk = 0; blk < blocks; ++blk, n0 += 256) {
    if (n0 >= N) return;
    if (blk) load_b<T, RT, LEN>(bi, n0, N, R, bf);
    expand_rows<T, RT>(l, base, out, N, n0, n, bf);
  }
}

// ---------------------------------------------------------------------------
// Both in one launch, for a single row of few ranks and a short K: a workgroup
// of 8 waves has 512 outputs and forms t by itself, reading all of A: a wave
// has every 8th rank, and reads a kilobyte of a row at a time.  That costs the
// workgroup K ranks x 2 bytes from the L2, and saves a launch and the way
// through memory.  One launch against two, us a call in a graph (the host's time
// falls from 18 to 14 us): K 4096, rank 16: 5.2 / 6.9; K 4096, rank 32: 6.6 /
// 7.4; K 14336, rank 16: 8.8 / 8.3; K 8192, rank 32: 9.0 / 8.3; K 14336, rank
// 32: 14.3 / 9.3.  (Two rows at K 4096, rank 16 would take 10.2 / 7.6: the
// matrix cores are the better way for more.)
// ---------------------------------------------------------------------------

constexpr int kOneWaves = 8;

template <typename T, int RT, Len LA, Len LB>
__global__ __launch_bounds__(64 * kOneWaves) void lora_one_kernel(const int32_t* __restrict__ ids, int adapters,
                                                                  const T* __restrict__ x, const T* base,
                                                                  const T* __restrict__ a, const T* __restrict__ b,
                                                                  const float* __restrict__ scales, T* out, int64_t N,
                                                                  int64_t K, int R) {
  typedef ExpandRows<T, RT> L;
  constexpr int RW = L::RP / kOneWaves;  // ranks of a wave
  constexpr int UN = RT == 1 ? 4 : 2;    // kilobytes of each row in flight
  __shared__ L l;
  __shared__ float t[L::RP];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int adapter = ids[0];
  if (adapter < 0 || adapter >= adapters) {
    const int64_t c0 = (int64_t)blockIdx.x * 64 * kOneWaves;
    if (base != out) copy_rows(base, 0, out, 0, c0, c0 + 64 * kOneWaves < N ? c0 + 64 * kOneWaves : N, 1, 0);
    return;
  }
  if (wave == 0) l.at_base[lane] = l.at_out[lane] = 0;
  const int64_t n0 = ((int64_t)blockIdx.x * kOneWaves + wave) * 64;
  typename L::v8 bf[4][L::KS];
  load_b<T, RT, LB>(b + (int64_t)adapter * N * R, n0, N, R, bf);  // on the way while t is formed
  const T* ar[RW];
  float acc[RW];
#pragma unroll
  for (int q = 0; q < RW; ++q) {
    const int r = wave + kOneWaves * q;
    ar[q] = a + ((int64_t)adapter * R + (r < R ? r : 0)) * K;
    acc[q] = 0.0f;
  }
  for (int64_t k0 = 8 * lane; k0 < K; k0 += 512 * UN) {
    typename L::v8 av[UN][RW], xv[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
#pragma unroll
      for (int q = 0; q < RW; ++q) av[u][q] = load_frag<T, LA>(ar[q], k0 + 512 * u, K);
      xv[u] = load_frag<T, LA>(x, k0 + 512 * u, K);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int q = 0; q < RW; ++q) acc[q] = fmaf(to_f32((T)av[u][q][e]), to_f32((T)xv[u][e]), acc[q]);
  }
#pragma unroll
  for (int q = 0; q < RW; ++q) {
    const float s = wave_sum(acc[q]);
    const int r = wave + kOneWaves * q;
    if (lane == 0) t[r] = r < R ? s : 0.0f;
  }
  lds_barrier();
  {
    const int i = (int)threadIdx.x / L::CH, c = (int)threadIdx.x % L::CH;  // 16 rows, zeros behind the first
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (i == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = t[8 * c + e];
    }
    l.put(i & 15, c, v, scales ? scales[adapter] : 1.0f, i < 16);
  }
  lds_barrier();
  if (n0 < N) expand_rows<T, RT>(l, base, out, N, n0, 1, bf);
}

struct LoraPlan {
  int64_t groups, k_slice, order_ints;  // most groups that there can be
  int slices, rank_tiles, blocks, rows;  // rows of a workgroup of the first product
  bool one;   // one launch, no workspace
  bool list;  // a launch that lists the groups
};

inline LoraPlan lora_plan(int64_t M, int64_t N, int64_t K, int64_t R, int64_t adapters) {
  LoraPlan p;
  p.rank_tiles = R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8;
  const int64_t kinds = adapters + 1 < M ? adapters + 1 : M;  // adapters that rows can name, and none
  // One launch saves an eager call 4 us of host time and a graph's replay 0.8 to
  // 1.7 us at K 4096; at the end of this range (K 14336 of rank 16, 8192 of 32) a
  // replay takes 0.5 to 0.7 us longer than with two launches.
  p.one = M == 1 && R <= 32 && K >= 8 && K * p.rank_tiles <= 16384;
  p.list = M > kWaveRows || (M > kGroupRows && adapters > kWaveAdapters);
  p.groups = M <= kGroupRows ? kinds : M / kGroupRows + kinds;
  p.order_ints = !p.list ? 0 : (p.groups * (kGroupRows + 1) + 1 + 3) / 4 * 4;
  // Half a group is more workgroups and reads A twice as often; N 4096, 32 / 64
  // rows of a workgroup, us a call: K 4096: 500 rows of rank 16 17.5 / 19.5, of
  // rank 128 31.4 / 35.1; 1000 rows 20.1 / 22.1, 35.4 / 39.1; 2000 rows 24.0 /
  // 24.9, 41.9 / 42.8; K 8192, 2000 rows of rank 128 43.2 / 37.4.
  p.rows = M > kGroupRows && M <= 1024 ? 32 : kGroupRows;
  // K in slices where there are few workgroups: of four turns, or of two while
  // there are no more than 8 of them.  Two / four / eight turns, us a call: 32
  // rows of K 4096, rank 64: 10.0 / 11.4 / 15.8, of rank 16: 8.0 / 8.2 / 9.6; 8
  // rows of K 14336, rank 16 (28, 14 and 7 slices to join): 9.5 / 8.8 / 9.1.
  const int64_t turn = 32 * kShrinkWaves;
  int64_t s = (K + 4 * turn - 1) / (4 * turn);
  const int64_t two = (K + 2 * turn - 1) / (2 * turn);
  if (s < 8) s = two < 8 ? two : 8;
  const int64_t full = (M + kGroupRows - 1) / kGroupRows;
  const int64_t fill = 256 / ((M + p.rows - 1) / p.rows + kinds);  // one round of a workgroup for each CU
  if (s > fill) s = fill > 1 ? fill : 1;
  p.k_slice = (K + s - 1) / s;
  p.k_slice = (p.k_slice + turn - 1) / turn * turn;
  p.slices = (int)((K + p.k_slice - 1) / p.k_slice);
  // Outputs of a workgroup, 512 against 256: joining t and finding the group
  // count less, and fewer workgroups fill the CUs less.  us a call: 8192 rows x
  // 14336, rank 128: 177 / 187; x 4096, rank 128: 120 / 118; 4093 rows x 14336,
  // rank 16: 70.2 / 67.2; 8192 x 8192, rank 32: 85.4 / 82.5.
  p.blocks = R > 64 && (N + 255) / 256 * full >= 4096 ? 2 : 1;
  return p;
}

}  // namespace

extern "C" {

size_t mk_lora_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t R, int64_t adapters) {
  if (M <= 0 || N <= 0 || K <= 0 || R <= 0 || R > 128 || adapters <= 0) return 0;
  const LoraPlan p = lora_plan(M, N, K, R, adapters);
  if (p.one) return 0;
  return ((size_t)p.order_ints + (size_t)p.slices * M * 16 * p.rank_tiles) * sizeof(float);
}

int mk_lora_add(const void* x, int64_t x_stride, const void* base, int64_t base_stride, const void* a, const void* b,
                const int32_t* adapter_ids, const float* scales, void* out, int64_t out_stride, int64_t M, int64_t N,
                int64_t K, int64_t R, int64_t adapters, int dtype, void* workspace, size_t workspace_bytes,
                void* stream) {
  MK_REQUIRE(M >= 0 && N >= 0 && K > 0 && R > 0 && R <= 128 && adapters > 0 && adapters <= kMaxAdapters);
  MK_REQUIRE(M < (1LL << 20) && N < (1LL << 24) && K < (1LL << 31));
  MK_REQUIRE(x_stride >= K && base_stride >= N && out_stride >= N && (out != base || out_stride == base_stride));
  MK_REQUIRE(dtype == MK_DT_F16 || dtype == MK_DT_BF16);
  if (M == 0 || N == 0) return MK_OK;
  MK_REQUIRE(x && base && adapter_ids && out && a && b && mk_aligned(workspace, 16));
  const size_t need = mk_lora_workspace_bytes(M, N, K, R, adapters);
  MK_REQUIRE(need == 0 || (workspace && workspace_bytes >= need));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const LoraPlan p = lora_plan(M, N, K, R, adapters);
  int32_t* order = reinterpret_cast<int32_t*>(workspace);
  float* t = reinterpret_cast<float*>(workspace) + p.order_ints;
  const Len len_a = len_of(K), len_b = len_of(R);
  Groups gs = {adapter_ids, nullptr, nullptr, M, (int)adapters};
  if (p.list) {
    gs.rows = order;
    gs.adapters = order + p.groups * kGroupRows;
    lora_group_kernel<<<1, 1024, 0, st>>>(adapter_ids, order, order + p.groups * kGroupRows, M, (int)adapters);
  }
#define MK_ONE(T, RT, LA, LB)                                                                                        \
  lora_one_kernel<T, RT, LA, LB><<<(unsigned)((N + 64 * kOneWaves - 1) / (64 * kOneWaves)), 64 * kOneWaves, 0, st>>>( \
      adapter_ids, (int)adapters, (const T*)x, (const T*)base, (const T*)a, (const T*)b, scales, (T*)out, N, K, (int)R)
#define MK_ONE_LEN(T, RT)                                                 \
  do {                                                                    \
    if (len_b == kFew && len_a == kRest) MK_ONE(T, RT, kRest, kFew);      \
    else if (len_b == kFew) MK_ONE(T, RT, kWhole, kFew);                  \
    else if (len_b == kRest && len_a == kRest) MK_ONE(T, RT, kRest, kRest); \
    else if (len_b == kRest) MK_ONE(T, RT, kWhole, kRest);                \
    else if (len_a == kRest) MK_ONE(T, RT, kRest, kWhole);                \
    else MK_ONE(T, RT, kWhole, kWhole);                                   \
  } while (0)
  if (p.one) {
    if (dtype == MK_DT_F16 && p.rank_tiles == 1) MK_ONE_LEN(f16, 1);
    else if (dtype == MK_DT_F16) MK_ONE_LEN(f16, 2);
    else if (p.rank_tiles == 1) MK_ONE_LEN(bf16, 1);
    else MK_ONE_LEN(bf16, 2);
    MK_CHECK_LAUNCH();
    return MK_OK;
  }
#undef MK_ONE_LEN
#undef MK_ONE
  const dim3 shrink((unsigned)(p.groups * (kGroupRows / p.rows)), (unsigned)p.slices);
  const dim3 expand((unsigned)((N + 256 * p.blocks - 1) / (256 * p.blocks)), (unsigned)p.groups);
#define MK_SHRINK(T, RT, L)                                                                                         \
  lora_shrink_kernel<T, RT, L><<<shrink, 64 * kShrinkWaves, 0, st>>>(gs, (const T*)x, x_stride, (const T*)a, t, K, \
                                                                     (int)R, p.k_slice, p.rows)
#define MK_EXPAND(T, RT, L)                                                                                      \
  lora_expand_kernel<T, RT, L><<<expand, 256, 0, st>>>(gs, (const T*)base, base_stride, (const T*)b, scales, t, \
                                                       (T*)out, out_stride, N, (int)R, p.slices, p.blocks)
#define MK_LORA(T, RT)                                  \
  do {                                                  \
    if (len_a == kWhole) MK_SHRINK(T, RT, kWhole);      \
    else if (len_a == kRest) MK_SHRINK(T, RT, kRest);   \
    else MK_SHRINK(T, RT, kFew);                        \
    if (len_b == kWhole) MK_EXPAND(T, RT, kWhole);      \
    else if (RT > 1 || len_b == kRest) MK_EXPAND(T, RT, kRest); \
    else MK_EXPAND(T, 1, kFew);                         \
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
