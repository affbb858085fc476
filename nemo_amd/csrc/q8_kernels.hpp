// q8_kernels.hpp -- feature rows held in 8 bits: quantise, read back, products on the bf16 matrix cores, clutter score
// Part of the single translation unit nemo_hip.hip (included from there, in order; not a stand-alone header).
//
// A row of C channels is C codes (e4m3, the format without infinities) and one scale byte per block of 128 channels:
//   amax = the largest |x_c| of the block's finite numbers,  e = max(-117, ceil(log2(amax / 448))),
//   code_c = e4m3(x_c 2^-e) to nearest even (NaN where x_c is not finite),  byte = e + 127.
// The scale is a power of two because nothing is lost by it that amax / 448 would keep, but for range at the small end
// (e4m3's step is relative), while x 2^-e and code 2^e become exact, the latter in bf16 too: 4 significant bits and fp32's range.
// -117: the smallest code, 2^-9, times 2^-117 is still a normal number.
//
// Products run on the bf16 matrix instructions, on the numbers that the codes stand for (v_cvt_scalef32_pk_bf16_fp8: exact from 2^-133 to
// 2^128, bf16's range with its subnormals; quantising writes nothing below 2^-126).
// The 8-bit matrix instructions have twice the rate, but add neighbouring products after cutting each at 2^-14 of the
// largest among them (measured; 1.4e-5 of the result where the bf16 ones are off by 5e-9): that is no fp32 sum.
#ifndef Q8_KERNELS_HPP
#define Q8_KERNELS_HPP

namespace {

constexpr int Q8_BLOCK = 128;  // channels per scale
constexpr uint32_t Q8_INF = 0x7f800000u;

typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef uint32_t u4va __attribute__((ext_vector_type(4)));

// e of a block from the bits of its (finite) amax: 448 = 1.75 * 2^8
__device__ __forceinline__ int q8_exponent(uint32_t amax) {
  const int e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, -117);
}
__device__ __forceinline__ float q8_pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 <= e <= 127
// the number a scale byte stands for (byte 0: 2^-127, byte 255: NaN; quantising writes neither)
__device__ __forceinline__ float q8_scale(uint32_t byte) {
  return __uint_as_float(byte << 23 | (byte - 1 >= 254 ? 0x00400000u : 0u));
}
__device__ __forceinline__ uint32_t q8_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// four numbers, already times 2^-e, to four codes
__device__ __forceinline__ uint32_t q8_pack(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
__device__ __forceinline__ void q8_unpack(uint32_t codes, float s, float *x) {
  auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
  auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  x[0] = lo[0] * s; x[1] = lo[1] * s; x[2] = hi[0] * s; x[3] = hi[1] * s;
}

// the three types a row is quantised from and read back to
// (at: number s of those that a 4-byte word holds; bits: a number as it is in memory; NAN_BITS: makes any infinity a NaN)
struct Q8F32 {
  typedef float T;
  static constexpr uint32_t NAN_BITS = 0x00400000u;
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
  static __device__ __forceinline__ float at(uint32_t w, int) { return __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t bits(float x) { return __float_as_uint(x); }
};
struct Q8BF16 {
  typedef __bf16 T;
  static constexpr uint32_t NAN_BITS = 0x0040u;
  static __device__ __forceinline__ float get(__bf16 x) { return (float)x; }
  static __device__ __forceinline__ __bf16 put(float x) { return (__bf16)x; }
  static __device__ __forceinline__ float at(uint32_t w, int s) { return __uint_as_float(s ? w & 0xffff0000u : w << 16); }
  static __device__ __forceinline__ uint32_t bits(__bf16 x) { return __builtin_bit_cast(uint16_t, x); }
};
struct Q8F16 {
  typedef _Float16 T;
  static constexpr uint32_t NAN_BITS = 0x0200u;
  static __device__ __forceinline__ float get(_Float16 x) { return (float)x; }
  static __device__ __forceinline__ _Float16 put(float x) { return (_Float16)x; }
  static __device__ __forceinline__ float at(uint32_t w, int s) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(s ? w >> 16 : w & 0xffffu)); }
  static __device__ __forceinline__ uint32_t bits(_Float16 x) { return __builtin_bit_cast(uint16_t, x); }
};

// Where image i of a call sits in the cache: slots[i], or i.  -1: nowhere (out of range).
__device__ __forceinline__ int q8_slot(const int32_t *slots, int i, int n_slots) {
  const int s = slots ? slots[i] : i;
  return s >= 0 && s < n_slots ? s : -1;
}
// Two images written to the same slot: the later one stays, as if they were written in order.  Whether a later image
// than i has slot s (whole workgroup).  Every workgroup reads the slots behind its image's: no matter at 512 images (of 16 pixels x 128, f32:
// 8.0 us, 7.6 without slots), much at many small ones (16384: 72 and 27 us, 262144: 8.7 and 0.49 ms).
__device__ __forceinline__ bool q8_overwritten(const int32_t *slots, int i, int n, int s) {
  if (!slots) return false;
  bool hit = false;
  for (int j = i + 1 + (int)threadIdx.x; j < n; j += (int)blockDim.x) hit |= slots[j] == s;
  return __syncthreads_or(hit) != 0;
}

// ---------------------------------------------------------------- quantise, channels contiguous
// x [n][rows][C] -> q [slot][rows][C], e [slot][rows][nb].  16 lanes own a block of 128 channels, 8 numbers a lane (fp32: 4
// in either half of the block, so that every load instruction reads whole cache lines), its maximum goes through four
// rotations inside the 16 lanes.  Bound by memory: 33 maps of 160 x 200 x 256 in bf16, 813 MB, 152 us = 5.3 TB/s (a large copy moves
// 4.7); with the loads of 2 bytes or not in flight together it took 350.
constexpr int Q8_QU = 4;  // blocks per 16 lanes: their loads are all in flight before the first is used
template <class TT>
__global__ __launch_bounds__(256) void q8_quantize_kernel(const typename TT::T *__restrict__ x, int n, int rows, int C, int nb, unsigned chunks,
                                                          const int32_t *__restrict__ slots, int n_slots, uint8_t *__restrict__ q,
                                                          uint8_t *__restrict__ e) {
  constexpr bool F32 = sizeof(typename TT::T) == 4;
  const int img = (int)(blockIdx.x / chunks);
  const unsigned chunk = blockIdx.x - (unsigned)img * chunks;
  const int slot = q8_slot(slots, img, n_slots);
  if (slot < 0 || q8_overwritten(slots, img, n, slot)) return;
  const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
  const size_t blocks = (size_t)rows * nb, b0 = (size_t)chunk * (16 * Q8_QU) + group;
  float v[Q8_QU][8];
#pragma unroll
  for (int u = 0; u < Q8_QU; ++u) {
    const size_t blk = b0 + 16 * u;
    const size_t row = nb == 1 ? blk : blk / nb;
    const int c0 = nb == 1 ? 0 : (int)(blk - row * nb) * Q8_BLOCK;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = c0 + (F32 ? 64 * h + 4 * lane : 8 * lane + 4 * h);
      typedef typename TT::T v4 __attribute__((ext_vector_type(4)));
      v4 p = {};
      if (blk < blocks && c < C) p = *(const v4 *)(x + ((size_t)img * rows + row) * C + c);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[u][4 * h + k] = TT::get(p[k]);
    }
  }
#pragma unroll
  for (int u = 0; u < Q8_QU; ++u) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, q8_abs_bits(v[u][k]));
    auto all16 = [](uint32_t a) {
      a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x128, 0xf, 0xf, false));
      a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x124, 0xf, 0xf, false));
      a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x122, 0xf, 0xf, false));
      return max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x121, 0xf, 0xf, false));
    };
    m = all16(m);
    if (__any(m >= Q8_INF)) {  // numbers that are not finite: rare, the whole wave takes the maximum again without them
      m = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t a = q8_abs_bits(v[u][k]);
        m = max(m, a < Q8_INF ? a : 0u);
        v[u][k] = a < Q8_INF ? v[u][k] : __uint_as_float(0x7fc00000u);
      }
      m = all16(m);
    }
    const int ex = q8_exponent(m);
    const float s = q8_pow2(-ex);
    const size_t blk = b0 + 16 * u;
    if (blk >= blocks) continue;
    const size_t row = nb == 1 ? blk : blk / nb;
    const int b = nb == 1 ? 0 : (int)(blk - row * nb);
    uint8_t *qp = q + ((size_t)slot * rows + row) * C + (size_t)b * Q8_BLOCK;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = F32 ? 64 * h + 4 * lane : 8 * lane + 4 * h;
      if (b * Q8_BLOCK + c < C) *(uint32_t *)(qp + c) = q8_pack(v[u][4 * h] * s, v[u][4 * h + 1] * s, v[u][4 * h + 2] * s, v[u][4 * h + 3] * s);
    }
    if (lane == 0) e[((size_t)slot * rows + row) * nb + b] = (uint8_t)(ex + 127);
  }
}

// ---------------------------------------------------------------- quantise, pixels contiguous
// x [n][C][rows] -> the same q and e (the layout a backbone leaves and a feature record holds).  A workgroup owns 64 PX pixels and one
// block of 128 channels, a wave 32 of the channels: a lane's numbers are of PX pixels (one 4-byte load a channel: PX = 1 for fp32, 2 for
// 16 bits, where loads of 2 bytes reached 2.3 TB/s), so the maximum needs one exchange between the waves; the codes go through LDS so that a
// pixel's 128 bytes leave as one line.  Bound by memory: 512 fp32 maps of 80 x 100 x 128, 2.63 GB, 497 us = 5.3 TB/s; one map of
// 32 x 84 x 128 takes 3.4 us, a launch.
template <class TT>
__global__ __launch_bounds__(256) void q8_quantize_t_kernel(const typename TT::T *__restrict__ x, int n, int rows, int C, int nb, unsigned tiles,
                                                            const int32_t *__restrict__ slots, int n_slots, uint8_t *__restrict__ q,
                                                            uint8_t *__restrict__ e) {
  typedef typename TT::T T;
  constexpr int PX = 4 / (int)sizeof(T), TP = 64 * PX;
  struct __attribute__((packed, aligned(sizeof(T)))) Word { uint32_t v; };
  __shared__ uint32_t top[4][TP];
  __shared__ __align__(16) uint8_t codes[TP][Q8_BLOCK + 16];
  const unsigned per = tiles * (unsigned)nb;
  const int img = (int)(blockIdx.x / per);
  const unsigned rest = blockIdx.x - (unsigned)img * per;
  const int b = (int)(rest / tiles), p0 = (int)(rest - (unsigned)b * tiles) * TP;
  const int slot = q8_slot(slots, img, n_slots);
  if (slot < 0 || q8_overwritten(slots, img, n, slot)) return;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int c0 = b * Q8_BLOCK + 32 * w;
  const T *xp = x + ((size_t)img * C + c0) * rows;
  uint32_t raw[32];  // PX numbers of channel c0 + k each, as they are in memory
#pragma unroll
  for (int k = 0; k < 32; ++k) raw[k] = 0;
#pragma unroll
  for (int k = 0; k < 32; k += 16) {
    if (c0 + k >= C) break;
    if (p0 + TP <= rows) {
#pragma unroll
      for (int j = k; j < k + 16; ++j) raw[j] = ((const Word *)(xp + (size_t)j * rows + (p0 + PX * lane)))->v;
    } else {
#pragma unroll
      for (int j = k; j < k + 16; ++j)
#pragma unroll
        for (int s = 0; s < PX; ++s) raw[j] |= TT::bits(xp[(size_t)j * rows + min(p0 + PX * lane + s, rows - 1)]) << (16 * s);
    }
  }
  uint32_t m[PX];
  bool odd = false;
#pragma unroll
  for (int s = 0; s < PX; ++s) {
    m[s] = 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) m[s] = max(m[s], q8_abs_bits(TT::at(raw[k], s)));
    odd |= m[s] >= Q8_INF;
  }
  if (__any(odd)) {  // numbers that are not finite: rare, the maxima are taken again without them
#pragma unroll
    for (int s = 0; s < PX; ++s) {
      m[s] = 0;
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        const uint32_t a = q8_abs_bits(TT::at(raw[k], s));
        m[s] = max(m[s], a < Q8_INF ? a : 0u);
        if (a >= Q8_INF) raw[k] |= TT::NAN_BITS << (16 * s);  // infinity to NaN
      }
    }
  }
#pragma unroll
  for (int s = 0; s < PX; ++s) top[w][PX * lane + s] = m[s];
  __syncthreads();
  int ex[PX];
#pragma unroll
  for (int s = 0; s < PX; ++s) {
    const int p = PX * lane + s;
    ex[s] = q8_exponent(max(max(top[0][p], top[1][p]), max(top[2][p], top[3][p])));
    const float f = q8_pow2(-ex[s]);
#pragma unroll
    for (int k = 0; k < 32; k += 16) {
      u4va c;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t *r = raw + k + 4 * j;
        c[j] = q8_pack(TT::at(r[0], s) * f, TT::at(r[1], s) * f, TT::at(r[2], s) * f, TT::at(r[3], s) * f);
      }
      *(u4va *)&codes[p][32 * w + k] = c;
    }
  }
  __syncthreads();
  const size_t row0 = (size_t)slot * rows + p0;
#pragma unroll
  for (int j = 0; j < 2 * PX; ++j) {
    const int i = (int)threadIdx.x + 256 * j, r = i >> 3, c = (i & 7) * 16;
    if (p0 + r < rows && b * Q8_BLOCK + c < C) *(u4va *)(q + (row0 + r) * C + (size_t)b * Q8_BLOCK + c) = *(const u4va *)&codes[r][c];
  }
  if (w == 0)
#pragma unroll
    for (int s = 0; s < PX; ++s)
      if (p0 + PX * lane + s < rows) e[(row0 + PX * lane + s) * nb + b] = (uint8_t)(ex[s] + 127);
}

// ---------------------------------------------------------------- read back, channels contiguous
// q [slot][rows][C], e -> x [n][rows][C]; a lane reads as many codes as make 16 bytes of numbers, Q8_DU times.  An image without a slot
// reads zeros.  Bound by memory: 512 maps of 80 x 100 x 128 to fp32, 2.63 GB, 473 us = 5.5 TB/s; one of them 3.8 us.
constexpr int Q8_DU = 4;
template <class TT>
__global__ __launch_bounds__(256) void q8_dequantize_kernel(const uint8_t *__restrict__ q, const uint8_t *__restrict__ e, int rows, int C, int nb,
                                                            unsigned chunks, const int32_t *__restrict__ slots, int n_slots,
                                                            typename TT::T *__restrict__ x) {
  constexpr int P = 16 / (int)sizeof(typename TT::T);
  typedef typename TT::T vp __attribute__((ext_vector_type(P)));
  typedef uint32_t cp __attribute__((ext_vector_type(P / 4)));
  const int img = (int)(blockIdx.x / chunks);
  const unsigned chunk = blockIdx.x - (unsigned)img * chunks;
  const int slot = q8_slot(slots, img, n_slots);
  const unsigned ppr = (unsigned)C / P;  // pieces per row
  const size_t pieces = (size_t)rows * ppr, base = (size_t)max(slot, 0) * rows;
#pragma unroll
  for (int u = 0; u < Q8_DU; ++u) {
    const size_t i = (size_t)chunk * (256 * Q8_DU) + 256 * u + threadIdx.x;
    if (i >= pieces) return;
    const size_t row = i / ppr;
    const unsigned c = (unsigned)(i - row * ppr);
    float f[P];
#pragma unroll
    for (int k = 0; k < P; ++k) f[k] = 0.0f;
    if (slot >= 0) {
      const cp codes = *(const cp *)(q + base * C + P * i);
      const float s = q8_scale(e[(base + row) * nb + c / (Q8_BLOCK / P)]);
#pragma unroll
      for (int k = 0; k < P / 4; ++k) q8_unpack(codes[k], s, f + 4 * k);
    }
    vp o;
#pragma unroll
    for (int k = 0; k < P; ++k) o[k] = TT::put(f[k]);
    *(vp *)(x + (size_t)img * rows * C + P * i) = o;
  }
}

// ---------------------------------------------------------------- read back, pixels contiguous
// q [slot][rows][C], e -> x [n][C][rows]: 256 pixels x 128 channels through LDS, whose rows of 33 words let the lanes of a wave read one word
// each of different pixels.  A lane writes PX numbers of a channel, the waves neighbouring pixels: 1 KB (fp32) or 512 bytes of a channel
// leave at about the same time, and the tiles of a channel follow each other on one XCD (workgroup b runs on XCD b % 8), because lines that
// are filled in parts cost the memory several times their bytes.  40 maps of 97 x 101 x 208, whose channels begin anywhere in a line: 102 us
// to fp32 (4.0 TB/s), 74 to bf16.
template <class TT>
__global__ __launch_bounds__(256) void q8_dequantize_t_kernel(const uint8_t *__restrict__ q, const uint8_t *__restrict__ e, int rows, int C, int nb,
                                                              unsigned tiles, unsigned n_blocks, const int32_t *__restrict__ slots, int n_slots,
                                                              typename TT::T *__restrict__ x) {
  typedef typename TT::T T;
  constexpr int PX = 4 / (int)sizeof(T), TP = 256, WP = 4 / PX;  // WP waves side by side, PX of them share the channels
  struct __attribute__((packed, aligned(sizeof(T)))) Word { T v[PX]; };
  __shared__ uint32_t codes[TP][Q8_BLOCK / 4 + 1];
  const unsigned share = (n_blocks + 7) / 8, id = (blockIdx.x & 7) * share + (blockIdx.x >> 3);
  if (id >= n_blocks) return;
  const unsigned per = tiles * (unsigned)nb;
  const int img = (int)(id / per);
  const unsigned rest = id - (unsigned)img * per;
  const int b = (int)(rest / tiles), p0 = (int)(rest - (unsigned)b * tiles) * TP;
  const int slot = q8_slot(slots, img, n_slots);
  const size_t row0 = (size_t)max(slot, 0) * rows + p0;
  u4va v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = (int)threadIdx.x + 256 * j, r = i >> 3, c = (i & 7) * 16;
    v[j] = u4va{0, 0, 0, 0};
    if (slot >= 0 && p0 + r < rows && b * Q8_BLOCK + c < C) v[j] = *(const u4va *)(q + (row0 + r) * C + (size_t)b * Q8_BLOCK + c);
  }
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), p = (w % WP) * 64 * PX + PX * lane;
  float s[PX];
#pragma unroll
  for (int k = 0; k < PX; ++k) s[k] = slot >= 0 && p0 + p + k < rows ? q8_scale(e[(row0 + p + k) * nb + b]) : 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = (int)threadIdx.x + 256 * j;
#pragma unroll
    for (int k = 0; k < 4; ++k) codes[i >> 3][(i & 7) * 4 + k] = v[j][k];
  }
  __syncthreads();
  if (p0 + p >= rows) return;
  const bool whole = p0 + p <= rows - PX;
  T *xp = x + ((size_t)img * C + b * Q8_BLOCK) * rows + p0 + p;
  constexpr int CH_W = Q8_BLOCK / PX;  // channels of a wave
#pragma unroll
  for (int j = 0; j < CH_W; j += 4) {
    const int c = CH_W * (w / WP) + j;
    if (b * Q8_BLOCK + c >= C) break;
    float f[PX][4];
#pragma unroll
    for (int k = 0; k < PX; ++k) q8_unpack(codes[p + k][c / 4], s[k], f[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      Word o;
#pragma unroll
      for (int m = 0; m < PX; ++m) o.v[m] = TT::put(f[m][k]);
      T *to = xp + (size_t)(c + k) * rows;
      if (whole) *(Word *)to = o;
      else *to = o.v[0];
    }
  }
}

// ---------------------------------------------------------------- products
// out[m][n] = sum over blocks of 2^(ea + eb) * sum of code products, accumulated in fp32 by the matrix cores.  Rows come in
// segments (rows row_off[s] .. row_off[s + 1] of a, or seg_rows each), a segment is multiplied with the rows of one bank
// (rows bank_off[g] .. bank_off[g + 1] of b, g = bank_of[s], or s, or 0 where there is one bank): a product of each group of rows with its own matrix, ragged both ways.
struct Q8Args {
  const uint8_t *a, *ae, *b, *be;
  const int32_t *row_off, *bank_off, *bank_of;
  int seg_rows;       // rows of every segment where row_off is null
  int n_seg, n_banks;
  int M, N;           // rows of a, rows of b: what the offsets are clamped to
  int K, nb;          // channels, blocks of 128
  int n_cols;         // row length of out
};
struct Q8Seg {
  int r0, r1;         // rows of a
  int n0, n1;         // rows of b; n0 > n1 never, r0 == r1: nothing to do
};
__device__ __forceinline__ void q8_seg_rows(const Q8Args &A, int s, int &r0, int &r1) {
  if (A.row_off) {
    r0 = min(max(A.row_off[s], 0), A.M);
    r1 = max(min(A.row_off[s + 1], A.M), r0);
  } else {
    r0 = s * A.seg_rows;
    r1 = r0 + A.seg_rows;
  }
}
// Tile `work` of all segments' tiles of TM rows in a row: its segment, and the rows it starts at (whole workgroup).
template <int WAVES>
__device__ __forceinline__ bool q8_find(const Q8Args &A, unsigned work, int TM, Q8Seg &S) {
  __shared__ int found[2], wsum[WAVES];
  int s, t;
  if (!A.row_off) {
    const unsigned per = ((unsigned)A.seg_rows + TM - 1) / TM;
    s = (int)(work / per);
    t = (int)(work - (unsigned)s * per);
    if (s >= A.n_seg) return false;
  } else {
    unsigned before = 0;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    s = -1;
    t = 0;
    for (int base = 0; base < A.n_seg; base += 64 * WAVES) {
      const int i = base + (int)threadIdx.x;
      int tiles = 0;
      if (i < A.n_seg) {
        int r0, r1;
        q8_seg_rows(A, i, r0, r1);
        tiles = (int)(((unsigned)(r1 - r0) + TM - 1) / TM);
      }
      int sum = tiles;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(sum, d);
        if (lane >= d) sum += o;
      }
      if (threadIdx.x == 0) found[0] = -1;
      if (lane == 63) wsum[w] = sum;
      __syncthreads();
      unsigned first = before + (unsigned)(sum - tiles);
      for (int k = 0; k < w; ++k) first += (unsigned)wsum[k];
      if (tiles > 0 && work >= first && work - first < (unsigned)tiles) {
        found[0] = i;
        found[1] = (int)(work - first);
      }
#pragma unroll
      for (int k = 0; k < WAVES; ++k) before += (unsigned)wsum[k];
      __syncthreads();
      s = __builtin_amdgcn_readfirstlane(found[0]);
      t = __builtin_amdgcn_readfirstlane(found[1]);
      if (s >= 0 || before > work) break;
      __syncthreads();
    }
    if (s < 0) return false;
  }
  int r0, r1;
  q8_seg_rows(A, s, r0, r1);
  S.r0 = r0 + t * TM;
  S.r1 = r1;
  const int g = A.bank_of ? A.bank_of[s] : A.n_banks == 1 ? 0 : s;
  if (g < 0 || g >= A.n_banks) return false;
  S.n0 = A.bank_off ? min(max(A.bank_off[g], 0), A.N) : 0;
  S.n1 = A.bank_off ? max(min(A.bank_off[g + 1], A.N), S.n0) : A.N;
  return true;
}

// Operands of v_mfma_f32_32x32x16_bf16: lane l holds row l % 32 and, of a block of 128 channels, the 16-byte chunks 2 u + l / 32, u = 0 .. 3.
// A chunk feeds two instructions, eight channels each; which channels meet in which instruction does not matter as long as it is the
// same for both operands (and it is the same in every kernel here: a product of up to 256 channels has the same bits whichever computes it).
__device__ __forceinline__ bf8v q8_numbers(uint32_t lo, uint32_t hi, float s) {
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, s, true);
  const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, s, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, s, true);
  return bf8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The wave's 64 lanes copy 16 bytes each from their own address to consecutive places of LDS, without going through registers; complete
// after q8_wait_copies() and a barrier.
__device__ __forceinline__ void q8_copy16(const uint8_t *from, uint8_t *lds) {
  __builtin_amdgcn_global_load_lds((const uint32_t GAS *)(uintptr_t)from, (__attribute__((address_space(3))) uint32_t *)lds, 16, 0, 0);
}
__device__ __forceinline__ void q8_wait_copies() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)
// Where chunk q (16 bytes) of a row lies in LDS: lines of 256 bytes hold two rows of 128 or one of 256, piece x of line l at place
// x ^ (l & 15).  The 16 lanes that are served together read the same chunk of 16 rows, one after another or two apart, and meet 16 different
// places in the 64 banks either way.
template <int NB>
__device__ __forceinline__ int q8_place(int row, int q) {
  const int l = NB == 1 ? row >> 1 : row, x = NB == 1 ? (row & 1) * 8 + q : q;
  return l * 256 + 16 * (x ^ (l & 15));
}
// and the row and chunk that lie at 16-byte place p
template <int NB>
__device__ __forceinline__ void q8_at(int p, int &row, int &q) {
  const int l = p >> 4, x = (p & 15) ^ (l & 15);
  row = NB == 1 ? 2 * l + (x >> 3) : l;
  q = NB == 1 ? x & 7 : x;
}
// What the wave's lanes wrote to LDS before, its lanes read after.
__device__ __forceinline__ void q8_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
struct Q8Frag { bf8v v[8]; };  // 32 rows of 128 channels
struct Q8Raw { u4va v[4]; };   // the same as codes
__device__ __forceinline__ Q8Raw q8_load(const uint8_t *row, int b, int h, int K) {
  Q8Raw x;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int k = b * Q8_BLOCK + 16 * (2 * u + h);
    x.v[u] = k < K ? *(const u4va *)(row + k) : u4va{0, 0, 0, 0};
  }
  return x;
}
__device__ __forceinline__ Q8Frag q8_frag(const Q8Raw &x, float s) {
  Q8Frag f;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    f.v[2 * u] = q8_numbers(x.v[u][0], x.v[u][1], s);
    f.v[2 * u + 1] = q8_numbers(x.v[u][2], x.v[u][3], s);
  }
  return f;
}
__device__ __forceinline__ f16v q8_mfma(const Q8Frag &x, const Q8Frag &y, f16v c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.v[i], y.v[i], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ f16v q8_zero() {
  f16v c;
#pragma unroll
  for (int r = 0; r < 16; ++r) c[r] = 0.0f;
  return c;
}

// Stores one 32 x 32 tile of products: lane l has column l % 32 of rows 8 (r / 4) + 4 (l / 32) + r % 4.  m0, m1, n0 and n1 are the same
// for the whole wave: a row's address is a scalar, a lane's place in it 32 bits (Q8_MAX_COLS).
template <class TT>
__device__ __forceinline__ void q8_store(typename TT::T *out, int ld, int m0, int m1, int n0, int n1, int i, int h, const f16v &acc) {
  typedef typename TT::T T;
  if (n0 + i >= n1) return;
  const uint32_t at = (uint32_t)(4 * h * ld + i) * (uint32_t)sizeof(T);
  char *base = (char *)(out + (size_t)m0 * ld + n0);
  auto to = [&](int r) { return (T GAS *)(uintptr_t)(base + (size_t)(8 * (r >> 2) + (r & 3)) * ld * sizeof(T) + at); };
  if (m0 + 32 <= m1) {
#pragma unroll
    for (int r = 0; r < 16; ++r) *to(r) = TT::put(acc[r]);
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (m0 + 8 * (r >> 2) + (r & 3) + 4 * h < m1) *to(r) = TT::put(acc[r]);
  }
}

// Few rows, or few columns: a wave owns 32 x 32 products.  Its 4 KB of either operand and block are read in order of addresses, a block
// ahead, and turned in LDS of its own (read by rows, a load instruction touches 32 lines for 32 bytes of each: 16 blocks of one tile took
// 18 us that way).  KS = 1: `across` of the 4 waves of a workgroup stand side by side, the others below them.  KS = 4, for long rows: they deal the blocks of the same tile
// among them, and their sums are added in the order of the waves.
// Bound by the launch and the way to memory and back: 1 x 1088 x 128 3.6 us, 1 x 128 x 2048 4.9 (12.4 before the waves shared
// the blocks), 12 groups of up to 40 rows x up to 1100 4.8.
template <class TT, int KS>
__global__ __launch_bounds__(256) void q8_product_few_kernel(Q8Args A, int across, typename TT::T *__restrict__ out) {
  __shared__ __align__(16) uint8_t turn[4][2][4096];
  Q8Seg S;
  if (!q8_find<4>(A, blockIdx.x, KS == 1 ? 128 / across : 32, S)) return;
  const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int cols = min(S.n1 - S.n0, A.n_cols);
  const int n0 = (KS == 1 ? (int)blockIdx.y * across + w % across : (int)blockIdx.y) * 32;
  if (KS == 1) S.r0 += 32 * (w / across);
  if (n0 >= cols || S.r0 >= S.r1) return;
  const uint8_t *pa[4], *pb[4];  // the lane's 16-byte pieces of a block
  int at[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    int row;
    q8_at<1>(64 * j + lane, row, at[j]);
    at[j] *= 16;
    pa[j] = A.a + (size_t)min(S.r0 + row, S.r1 - 1) * A.K + at[j];
    pb[j] = A.b + ((size_t)S.n0 + min(n0 + row, cols - 1)) * A.K + at[j];
  }
  const uint8_t *ea = A.ae + (size_t)min(S.r0 + i, S.r1 - 1) * A.nb, *eb = A.be + ((size_t)S.n0 + min(n0 + i, cols - 1)) * A.nb;
  u4va ga[4], gb[4];
  uint32_t sa = 0, sb = 0;
  auto fetch = [&](int b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = b * Q8_BLOCK + at[j] < A.K;
      ga[j] = in ? *(const u4va *)(pa[j] + b * Q8_BLOCK) : u4va{0, 0, 0, 0};
      gb[j] = in ? *(const u4va *)(pb[j] + b * Q8_BLOCK) : u4va{0, 0, 0, 0};
    }
    sa = ea[b];
    sb = eb[b];
  };
  f16v acc = q8_zero();
  int b = KS == 1 ? 0 : w;
  if (b < A.nb) fetch(b);
  for (; b < A.nb; b += KS) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      *(u4va *)&turn[w][0][16 * (64 * j + lane)] = ga[j];
      *(u4va *)&turn[w][1][16 * (64 * j + lane)] = gb[j];
    }
    const float fa = q8_scale(sa), fb = q8_scale(sb);
    q8_wave_sync();
    Q8Raw x, y;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      x.v[u] = *(const u4va *)&turn[w][0][q8_place<1>(i, 2 * u + h)];
      y.v[u] = *(const u4va *)&turn[w][1][q8_place<1>(i, 2 * u + h)];
    }
    if (b + KS < A.nb) fetch(b + KS);
    acc = q8_mfma(q8_frag(x, fa), q8_frag(y, fb), acc);
    q8_wave_sync();
  }
  if (KS == 1) {
    q8_store<TT>(out, A.n_cols, S.r0, S.r1, n0, cols, i, h, acc);
    return;
  }
  float *part = (float *)&turn[0][0][0];  // 4 KB of the wave's own 8
#pragma unroll
  for (int r = 0; r < 16; ++r) part[w * 2048 + r * 64 + lane] = acc[r];
  __syncthreads();
  if (n0 + i >= cols) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {  // wave w adds and stores rows 8 w .. 8 w + 7 of the tile
    const int at = (4 * w + k) * 64 + lane, m = S.r0 + 8 * w + 4 * h + k;
    const float sum = ((part[at] + part[2048 + at]) + part[2 * 2048 + at]) + part[3 * 2048 + at];
    if (m < S.r1) out[(size_t)m * A.n_cols + n0 + i] = TT::put(sum);
  }
}

// The bank's way to LDS, for the kernels that keep their rows of a in registers (8 waves, K <= 128 NB): SR rows at a time as codes, copied
// by the memory unit, which fills places (q8_place) in order of lanes.
template <int NB, bool TAIL, int SR, int BUFS>  // TAIL: K is less than 128 NB
struct Q8Bank {
  static constexpr int RB = Q8_BLOCK * NB;                  // bytes of a row in LDS
  static constexpr int PER = SR * RB / (512 * 16);          // 16-byte copies per thread and buffer
  static constexpr int NE = (SR * NB + 511) / 512;          // scales per thread and buffer
  static_assert(PER * 512 * 16 == SR * RB && SR % 32 == 0, "");
  uint8_t codes[BUFS][SR * RB];
  float scale[BUFS][SR * NB];
  // starts copying `room` rows (whole 8 KB) from row `first` of the bank's `rows` on; the scale bytes stay in e until put_scale
  __device__ __forceinline__ void copy(int buf, const uint8_t *bank, const uint8_t *bank_e, int K, int rows, int first, int room, int tid, uint32_t (&e)[NE]) {
    const int lane = tid & 63, w = tid >> 6;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (8192 * j >= room * RB) break;
      int r, q;
      q8_at<NB>((8 * j + w) * 64 + lane, r, q);
      const int row = min(first + r, rows - 1);             // rows past the end repeat the last one
      q8_copy16(bank + (TAIL ? (size_t)row * K + min(16 * q, K - 16) : (size_t)row * RB + 16 * q), &codes[buf][(8 * j + w) * 1024]);
    }
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      const int k = tid + 512 * j;
      e[j] = k < SR * NB ? bank_e[(size_t)min(first + k / NB, rows - 1) * NB + k % NB] : 0;
    }
  }
  __device__ __forceinline__ void put_scale(int buf, int tid, const uint32_t (&e)[NE]) {
#pragma unroll
    for (int j = 0; j < NE; ++j)
      if (tid + 512 * j < SR * NB) scale[buf][tid + 512 * j] = q8_scale(e[j]);
  }
  // rows n + i, i = 0 .. 31, of a buffer
  __device__ __forceinline__ Q8Frag get(int buf, int n, int b, int i, int h, int K) const {
    Q8Raw raw;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int q = 8 * b + 2 * u + h;
      raw.v[u] = *(const u4va *)&codes[buf][q8_place<NB>(n + i, q)];
      if (TAIL && 16 * q >= K) raw.v[u] = u4va{0, 0, 0, 0};
    }
    return q8_frag(raw, scale[buf][(n + i) * NB + b]);
  }
};

// Products leave in groups of NT tiles of 32 columns, tile t with columns NT i + t, so that a lane has NT neighbouring ones: 16 stores
// of 8 bytes a lane and whole lines a row, at any alignment of out's rows (the bf16 result's rows of an odd length begin in
// the middle of a word).
template <class TT, int NT> struct __attribute__((packed, aligned(sizeof(typename TT::T)))) Q8Out { typename TT::T v[NT]; };
template <class TT, int NT>
__device__ __forceinline__ void q8_store_group(typename TT::T *out, int ld, int m0, int m1, int n0, int n1, int i, int h, const f16v (&acc)[NT]) {
  typedef typename TT::T T;
  const uint32_t at = (uint32_t)(4 * h * ld + NT * i) * (uint32_t)sizeof(T);
  T *base = out + (size_t)m0 * ld + n0;
  if (m0 + 32 <= m1 && n0 + 32 * NT <= n1) {
    // A row's address stays a scalar and the lane's place 32 bits (Q8_MAX_COLS), so that the store instruction adds them (the empty asm keeps the compiler
    // from summing them in vector registers, an instruction and two registers a store).
    uint32_t place = at;
    asm("" : "+v"(place));
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      Q8Out<TT, NT> o;
#pragma unroll
      for (int t = 0; t < NT; ++t) o.v[t] = TT::put(acc[t][r]);
      uintptr_t row = (uintptr_t)(base + (size_t)(8 * (r >> 2) + (r & 3)) * ld);
      asm("" : "+s"(row));
      __builtin_memcpy((char GAS *)row + place, &o, sizeof(o));
    }
  } else {
    // The lanes whose columns all exist still store them together (262144 x 40: bf16 20.8 -> 16.0 us, f32 23 -> 20.0).
    const int left = n1 - n0 - NT * i, rows = m1 - m0 - 4 * h;
    auto to = [&](int r) { return (char GAS *)(uintptr_t)(base + (size_t)(8 * (r >> 2) + (r & 3)) * ld) + at; };
    if (left >= NT) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        Q8Out<TT, NT> o;
#pragma unroll
        for (int t = 0; t < NT; ++t) o.v[t] = TT::put(acc[t][r]);
        if (8 * (r >> 2) + (r & 3) < rows) __builtin_memcpy(to(r), &o, sizeof(o));
      }
    } else {  // one lane of either half, at most
#pragma unroll
      for (int t = 0; t < NT - 1; ++t) {
        if (t >= left) break;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (8 * (r >> 2) + (r & 3) < rows) ((T GAS *)to(r))[t] = TT::put(acc[t][r]);
      }
    }
  }
}

// Short rows (K <= 128).  What bounds these products is the result's way to memory (a row of 128 channels meets a row of the bank in 256
// operations, but leaves 4 bytes), so the work is cut for the stores: the 8 waves of a workgroup own neighbouring columns of the same
// rows, 64 each, whose bank rows stay in registers, and the rows pass by, up to 256 of them copied to LDS as codes before the
// first product.  A workgroup then writes 512 columns of 32 rows at about the same time, which fills whole lines also where out's rows
// begin in the middle of one, and waits for no store.  With wc < 8, 8 / wc waves share the columns and take the row tiles in turn; so do
// all 8 where a bank's last columns are few (262144 rows x 1088: bf16 136 -> 125 us, f32 227 -> 213; x 640 f32 152 -> 134; x 1095, whose lines
// are shared between the cuts, bf16 182 -> 186, f32 240 -> 242).  f32 reaches 5.2 TB/s of results where rows are whole lines and 4.7 where
// they are not (x 1095), bf16 4.5 and 3.1: a line that leaves in two parts costs about as much as two (these stores without the products
// reach 5.4 and 3.2 on the same rows in bf16, a linear fill of either result 6.9).  A mixed batch of 12 banks of 536 to 1095 rows into bf16 rows
// of 1095 takes 158-168 us for 421 MB, 155 without its products: an XCD has one contiguous eighth of all row tiles and cuts, which hold
// 0.77 to 1.25 of the mean of results there, and the rows begin inside lines; with 12 banks of 1024 it takes 128 us for 574 MB.
// Twice the columns a wave, so that a bf16 row leaves in the same 256 bytes as an f32 one, takes 216 registers and leaves one workgroup a compute
// unit: 200 us for 262144 x 1095, 250 for the mixed batch.
template <class TT, bool TAIL>
__global__ __launch_bounds__(512, 4) void q8_product_short_kernel(Q8Args A, int tiles, int cuts, int wc, int rt, typename TT::T *__restrict__ out) {
  constexpr int NB = 1, NT = 2;
  typedef Q8Bank<NB, TAIL, sizeof(typename TT::T) == 4 ? Q8_PR / 2 : Q8_PR, 1> Rows;
  __shared__ __align__(16) Rows L;
  __shared__ __align__(16) uint8_t turn[8][4096];
  // the column cuts of the same rows follow each other on one XCD (workgroup b runs on XCD b % 8): they share the lines between them
  const unsigned n = (unsigned)tiles * (unsigned)cuts, per = (n + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (id >= n) return;
  Q8Seg S;
  if (!q8_find<8>(A, id / cuts, 32 * rt, S)) return;
  const int tid = threadIdx.x, lane = tid & 63, i = lane & 31, h = lane >> 5, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cols = min(S.n1 - S.n0, A.n_cols), c0 = (int)(id % cuts) * wc * 32 * NT, m1 = min(S.r1, S.r0 + 32 * rt);
  if (c0 >= cols) return;
  while (wc > 1 && cols - c0 <= 16 * NT * wc) wc /= 2;  // a bank's last columns
  const int n0 = c0 + (w % wc) * 32 * NT;
  uint32_t e[Rows::NE];
  L.copy(0, A.a + (size_t)S.r0 * A.K, A.ae + (size_t)S.r0 * NB, A.K, m1 - S.r0, 0, 32 * rt, tid, e);
  // The wave's 32 NT bank rows, 8 KB, read in order of addresses and turned in LDS by halves: lanes i < 16 have their rows in the first
  // (read by rows, a load instruction would touch 32 lines for 32 bytes of each).
  u4va g[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int r = (64 * j + lane) / (8 * NB), q = (64 * j + lane) % (8 * NB);
    const size_t row = (size_t)S.n0 + min(n0 + r, cols - 1);
    g[j] = !TAIL || 16 * q < A.K ? *(const u4va *)(A.b + row * A.K + 16 * q) : u4va{0, 0, 0, 0};
  }
  uint32_t ey[NT][NB];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int b = 0; b < NB; ++b) ey[t][b] = A.be[((size_t)S.n0 + min(n0 + NT * i + t, cols - 1)) * NB + b];
  Q8Raw raw[NT][NB];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = (64 * j + lane) / (8 * NB), q = (64 * j + lane) % (8 * NB);
      *(u4va *)&turn[w][q8_place<NB>(r, q)] = g[4 * half + j];
    }
    q8_wave_sync();
    if ((i >> 4) == half) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int u = 0; u < 4; ++u) raw[t][b].v[u] = *(const u4va *)&turn[w][q8_place<NB>(NT * (i & 15) + t, 8 * b + 2 * u + h)];
    }
    q8_wave_sync();
  }
  Q8Frag y[NT][NB];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int b = 0; b < NB; ++b) y[t][b] = q8_frag(raw[t][b], q8_scale(ey[t][b]));
  L.put_scale(0, tid, e);
  q8_wait_copies();
  __syncthreads();
  if (n0 >= cols) return;
  for (int m = 32 * (w / wc); S.r0 + m < m1; m += 32 * (8 / wc)) {
    f16v acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = q8_zero();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const Q8Frag x = L.get(0, m, b, i, h, A.K);
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t] = q8_mfma(x, y[t][b], acc[t]);
    }
    q8_store_group<TT, NT>(out, A.n_cols, S.r0 + m, m1, n0, cols, i, h, acc);
  }
}

// Long rows (K > 128): tiles of 128 x 128, 4 waves of 64 x 64, 128 channels a step, whose codes the memory unit copies to LDS: a's, which
// come from far, two steps ahead into two buffers, b's, which the other tiles keep near, one step into one, 48 KB for three workgroups a compute
// unit.  A wave reads its 16 KB of a step into registers, and once all waves have, the next copies start under the widening (128
// instructions a wave) and the products (32, 1024 cycles).
// Bound by the copies, above all: 172032 x 128 x 2048 (443 MB, 90 GFLOP) takes 110-120 us = 4 TB/s and 0.8 PFLOP/s, 105 without its products, 80
// without its stores too (a's codes alone 58, 6 TB/s), but 118 without the reads from LDS and 117 without the widening; 8192 x 8192 x
// 2048 takes 246-256 us = 1.1 PFLOP/s, 194 and 159 in the same way.  For the former two buffers of both and two workgroups a compute unit took
// 155, one buffer copied before it is read into registers 135; one buffer copied after it the same as now, but 346 us for 262144 x 1088 x
// 256 (now 295) and 200 for 50000 x 2600 x 512 (now 186).
// The wave's codes of a step (x: 32 rows and the 32 behind them, y: the even and the odd of 64 rows) out of LDS.  The compiler would wait for
// every copy under way before a read of LDS that it sees; the wait for the reads stands in the same block.
__device__ __forceinline__ void q8_read_step(uint32_t ax, uint32_t ay, Q8Raw (&x)[2], Q8Raw (&y)[2]) {
  asm volatile(
      "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
      "ds_read_b128 %4, %8 offset:4096\n\tds_read_b128 %5, %9 offset:4096\n\tds_read_b128 %6, %10 offset:4096\n\tds_read_b128 %7, %11 offset:4096\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x[0].v[0]), "=&v"(x[0].v[1]), "=&v"(x[0].v[2]), "=&v"(x[0].v[3]), "=&v"(x[1].v[0]), "=&v"(x[1].v[1]), "=&v"(x[1].v[2]), "=&v"(x[1].v[3])
      : "v"(ax), "v"(ax ^ 32), "v"(ax ^ 64), "v"(ax ^ 96)
      : "memory");
  asm volatile(
      "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
      "ds_read_b128 %4, %12\n\tds_read_b128 %5, %13\n\tds_read_b128 %6, %14\n\tds_read_b128 %7, %15\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(y[0].v[0]), "=&v"(y[0].v[1]), "=&v"(y[0].v[2]), "=&v"(y[0].v[3]), "=&v"(y[1].v[0]), "=&v"(y[1].v[1]), "=&v"(y[1].v[2]), "=&v"(y[1].v[3])
      : "v"(ay), "v"(ay ^ 32), "v"(ay ^ 64), "v"(ay ^ 96), "v"(ay ^ 128), "v"(ay ^ 160), "v"(ay ^ 192), "v"(ay ^ 224)
      : "memory");
}
__device__ __forceinline__ void q8_barrier() {  // no wait for copies under way
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
template <class TT>
__global__ __launch_bounds__(256, 2) void q8_product_long_kernel(Q8Args A, int tiles, int cuts, typename TT::T *__restrict__ out) {
  constexpr int STEP = 128 * Q8_BLOCK;
  __shared__ __align__(256) uint8_t codes[3][STEP];  // a, a of the next step, b
  // Workgroups that follow each other on an XCD take 4 row tiles with one column tile, then with the next: what its L2 brings of b serves all 4
  // (30000 x 10300 x 512: 459 us a row tile at a time, 402 by 4, 406 by 8, 431 by 16; 60000 x 1100 x 256, whose column tiles share lines of
  // the result: 75.4, 75.1 and 78.7).
  constexpr unsigned GROUP = 4;
  const unsigned n = (unsigned)tiles * (unsigned)cuts, per = (n + 7) / 8, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (id >= n) return;
  const unsigned first = id / (GROUP * (unsigned)cuts) * GROUP, in = id - first * (unsigned)cuts, high = min(GROUP, (unsigned)tiles - first);
  const unsigned tile = first + in % high, cut = in / high;
  Q8Seg S;
  if (!q8_find<4>(A, tile, 128, S)) return;
  const int tid = threadIdx.x, lane = tid & 63, i = lane & 31, h = lane >> 5, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cols = min(S.n1 - S.n0, A.n_cols), n0 = (int)cut * 128, m1 = S.r1;
  if (n0 >= cols) return;
  // the thread's 16-byte pieces of a step, 32 rows apart: where their rows begin behind the tile's first (128 rows: 32 bits)
  const uint8_t *ta = A.a + (size_t)S.r0 * A.K, *tb = A.b + ((size_t)S.n0 + n0) * A.K;
  int r0, q;
  q8_at<1>(tid, r0, q);
  uint32_t pa = (uint32_t)r0 * (uint32_t)A.K, pb = pa;
  const uint32_t last_a = (uint32_t)min(m1 - 1 - S.r0, 127) * (uint32_t)A.K, last_b = (uint32_t)min(cols - 1 - n0, 127) * (uint32_t)A.K;
  const int mw = 64 * (w >> 1), nw = 64 * (w & 1);  // the wave's corner of the tile
  // its scales: rows i and i + 32 of a's, 2 i and 2 i + 1 of b's
  const uint8_t *tae = A.ae + (size_t)S.r0 * A.nb, *tbe = A.be + ((size_t)S.n0 + n0) * A.nb;
  uint32_t pea = (uint32_t)(mw + i) * (uint32_t)A.nb, peb = (uint32_t)(nw + 2 * i) * (uint32_t)A.nb;
  const uint32_t last_ea = (uint32_t)min(m1 - 1 - S.r0, 127) * (uint32_t)A.nb, last_eb = (uint32_t)min(cols - 1 - n0, 127) * (uint32_t)A.nb;
  uint32_t e[4];
  auto piece = [&](int b) { return (uint32_t)min(b * Q8_BLOCK + 16 * q, A.K - 16); };  // past the end of a row: its last piece, taken for zeros below
  auto copy_a = [&](int b) {
    const uint32_t k = piece(b);
    __builtin_amdgcn_sched_barrier(0);  // the wait above counts on these being the last
    asm("" : "+v"(pa));  // the four places are computed anew: kept, they would cost the third workgroup a compute unit
#pragma unroll
    for (int j = 0; j < 4; ++j) q8_copy16(ta + (min(pa + 32 * j * (uint32_t)A.K, last_a) + k), &codes[b & 1][4096 * j + 1024 * w]);
  };
  auto copy_b = [&](int b) {
    const uint32_t k = piece(b);
    asm("" : "+v"(pb), "+v"(pea), "+v"(peb));
#pragma unroll
    for (int j = 0; j < 4; ++j) q8_copy16(tb + (min(pb + 32 * j * (uint32_t)A.K, last_b) + k), &codes[2][4096 * j + 1024 * w]);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      e[s] = tae[min(pea + 32 * s * (uint32_t)A.nb, last_ea) + (uint32_t)b];
      e[2 + s] = tbe[min(peb + s * (uint32_t)A.nb, last_eb) + (uint32_t)b];
    }
  };
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)&codes[0][0];
  const uint32_t ax = lds + (uint32_t)q8_place<1>(mw + i, h), ay = lds + 2 * STEP + (uint32_t)q8_place<1>(nw + 2 * i, h);
  f16v acc[2][2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int t = 0; t < 2; ++t) acc[s][t] = q8_zero();
  auto step = [&](int b, auto more_a, auto more_b) {
    __builtin_amdgcn_s_waitcnt(decltype(more_b)::value ? 0x0f74 : 0x0f70);  // vmcnt(4): all but the copies of the next step's a; or (0)
    q8_barrier();
    asm volatile("" : "+v"(e[0]), "+v"(e[1]), "+v"(e[2]), "+v"(e[3]));  // what is made of them is not made before the wait
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = q8_scale(e[j]);
    Q8Raw x[2], y[2];
    q8_read_step(ax + (uint32_t)(b & 1) * STEP, ay, x, y);
    q8_barrier();  // the buffers have been read
    if (decltype(more_b)::value) copy_b(b + 1);
    if (decltype(more_a)::value) copy_a(b + 2);
    __builtin_amdgcn_sched_barrier(0);
    const int left = A.K - b * Q8_BLOCK;
    if (!decltype(more_b)::value && left < Q8_BLOCK) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (16 * (2 * u + h) >= left) x[0].v[u] = x[1].v[u] = y[0].v[u] = y[1].v[u] = u4va{0, 0, 0, 0};
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const bf8v x0 = q8_numbers(x[0].v[u][2 * g], x[0].v[u][2 * g + 1], f[0]), y0 = q8_numbers(y[0].v[u][2 * g], y[0].v[u][2 * g + 1], f[2]);
        acc[0][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x0, y0, acc[0][0], 0, 0, 0);
        const bf8v x1 = q8_numbers(x[1].v[u][2 * g], x[1].v[u][2 * g + 1], f[1]), y1 = q8_numbers(y[1].v[u][2 * g], y[1].v[u][2 * g + 1], f[3]);
        acc[1][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x1, y0, acc[1][0], 0, 0, 0);
        acc[0][1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x0, y1, acc[0][1], 0, 0, 0);
        acc[1][1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x1, y1, acc[1][1], 0, 0, 0);
      }
  };
  copy_a(0);
  copy_b(0);
  copy_a(1);  // K > 128: there are two steps
  int b = 0;
  for (; b + 2 < A.nb; ++b) step(b, std::true_type(), std::true_type());
  step(b, std::false_type(), std::true_type());
  step(b + 1, std::false_type(), std::false_type());
#pragma unroll
  for (int s = 0; s < 2; ++s)
    if (S.r0 + mw + 32 * s < m1 && n0 + nw < cols)
      q8_store_group<TT, 2>(out, A.n_cols, S.r0 + mw + 32 * s, m1, n0 + nw, cols, i, h, acc[s]);
}

// ---------------------------------------------------------------- clutter score
// The largest product of a pixel's row with the rows of its image's bank; NaN where one of them is, -infinity for an empty bank.  The
// bank is the first operand, so a lane's 16 results are of one pixel and the maximum stays in the lane: 8 three-way
// maxima (v_maximum3_f32, which keeps NaN) per 8 NB matrix instructions.
__device__ __forceinline__ float q8_max(float best, const f16v &acc) {
#pragma unroll
  for (int r = 0; r < 16; ++r) best = __builtin_elementwise_maximum(best, acc[r]);
  return best;
}
// 8 waves, each with the numbers of T x 32 pixels in registers: a row tile of the bank is read and widened once per wave and meets T
// tiles of pixels (per 32 matrix instructions of 32 cycles: 32 widening ones, 32 maxima, 4 KB out of LDS, at T = 4).  Bound by the matrix
// unit: 512 maps of 80 x 100 x 128 against 2560 vectors 1.73 ms = 1.55 PFLOP/s, a large bf16 library product reaches 1.3 to 1.6.  What
// measured no better: taking the maxima between the next tile's products with two accumulators and the codes a tile ahead (1.78 ms; it
// spills at D = 256), copying the next chunk after the last read of this one (1.77 ms).
template <int NB, int T>
__global__ __launch_bounds__(512, T * NB >= 2 ? 2 : 4) void q8_score_kernel(Q8Args A, float *__restrict__ out) {
  constexpr int K = Q8_BLOCK * NB;
  typedef Q8Bank<NB, false, 128, 2> Bank;  // a chunk of 128 rows is copied while the one before is multiplied: one barrier a chunk
  __shared__ __align__(16) Bank L;
  Q8Seg S;
  if (!q8_find<8>(A, blockIdx.x, 256 * T, S)) return;
  const int tid = threadIdx.x, lane = tid & 63, i = lane & 31, h = lane >> 5, w = tid >> 6;
  const int rows = S.n1 - S.n0, m0 = S.r0 + 32 * T * w;
  const uint8_t *bank = A.b + (size_t)S.n0 * K, *bank_e = A.be + (size_t)S.n0 * NB;
  float best[T];
#pragma unroll
  for (int t = 0; t < T; ++t) best[t] = -INFINITY;
  if (rows > 0) {
    uint32_t e[Bank::NE];
    L.copy(0, bank, bank_e, K, rows, 0, 128, tid, e);
    Q8Frag x[T][NB];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const size_t row = (size_t)min(m0 + 32 * t + i, S.r1 - 1);
#pragma unroll
      for (int b = 0; b < NB; ++b) x[t][b] = q8_frag(q8_load(A.a + row * K, b, h, K), q8_scale(A.ae[row * NB + b]));
    }
    L.put_scale(0, tid, e);
    q8_wait_copies();
    __syncthreads();
    const int chunks = (rows + 127) / 128;
    for (int c = 0; c < chunks; ++c) {
      if (c + 1 < chunks) L.copy((c + 1) & 1, bank, bank_e, K, rows, 128 * (c + 1), 128, tid, e);
      if (m0 < S.r1) {
        const int left = min(rows - 128 * c, 128);
        for (int n = 0; n < left; n += 32) {
          Q8Frag y[NB];
#pragma unroll
          for (int b = 0; b < NB; ++b) y[b] = L.get(c & 1, n, b, i, h, K);
#pragma unroll
          for (int t = 0; t < T; ++t) {
            f16v acc = q8_zero();
#pragma unroll
            for (int b = 0; b < NB; ++b) acc = q8_mfma(y[b], x[t][b], acc);
            best[t] = q8_max(best[t], acc);
          }
        }
      }
      if (c + 1 < chunks) L.put_scale((c + 1) & 1, tid, e);
      q8_wait_copies();
      __syncthreads();
    }
  }
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const float top = __builtin_elementwise_maximum(best[t], __shfl_xor(best[t], 32));
    const int m = m0 + 32 * t + i;
    if (h == 0 && m < S.r1) out[m] = top;
  }
}
// Few pixels: the 8 waves share 32 pixels and deal the bank's row tiles among them; the bank comes straight from memory, a tile ahead.
// Bound by the launch: one map of 80 x 100 against one vector 3.2 us.
template <int NB>
__global__ __launch_bounds__(512) void q8_score_few_kernel(Q8Args A, float *__restrict__ out) {
  constexpr int RB = Q8_BLOCK * NB;
  __shared__ float top[8][32];
  Q8Seg S;
  if (!q8_find<8>(A, blockIdx.x, 32, S)) return;
  const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5, w = threadIdx.x >> 6;
  const int rows = S.n1 - S.n0;
  float best = -INFINITY;
  if (32 * w < rows) {
    const size_t row = (size_t)min(S.r0 + i, S.r1 - 1);
    Q8Raw raw[NB];
    uint32_t e[NB];
    auto fetch = [&](int n) {
      const size_t rb = (size_t)S.n0 + min(n + i, rows - 1);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        raw[b] = q8_load(A.b + rb * RB, b, h, RB);
        e[b] = A.be[rb * NB + b];
      }
    };
    fetch(32 * w);
    Q8Frag x[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) x[b] = q8_frag(q8_load(A.a + row * RB, b, h, RB), q8_scale(A.ae[row * NB + b]));
    for (int n = 32 * w; n < rows; n += 256) {
      Q8Frag y[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) y[b] = q8_frag(raw[b], q8_scale(e[b]));
      if (n + 256 < rows) fetch(n + 256);
      f16v acc = q8_zero();
#pragma unroll
      for (int b = 0; b < NB; ++b) acc = q8_mfma(y[b], x[b], acc);
      best = q8_max(best, acc);
    }
  }
  best = __builtin_elementwise_maximum(best, __shfl_xor(best, 32));
  if (h == 0) top[w][i] = best;
  __syncthreads();
  if (threadIdx.x < 32 && S.r0 + (int)threadIdx.x < S.r1) {
    float m = top[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < 8; ++k) m = __builtin_elementwise_maximum(m, top[k][threadIdx.x]);
    out[S.r0 + threadIdx.x] = m;
  }
}

}  // namespace
#endif  // Q8_KERNELS_HPP
