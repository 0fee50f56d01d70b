// kv4.hip -- the 4-bit paged K/V cache: append (head norm + rotation + quantisation), attention that reads it, read-back,
// and their C entry points (include/fishmi.h).
//
// Number format.  32 consecutive dims share one power of two, a value is a 4-bit float (sign, 0 0.5 1 1.5 2 3 4 6): the
// matrix unit's own 4-bit type, so v_cvt_scalef32_pk_fp4_bf16 / v_cvt_scalef32_pk_bf16_fp4 pack and unpack two values
// per instruction, scale included.  The block's power is the smallest with max|x| <= 7 * 2^e: everything up to 6 * 2^e is
// off by at most half a grid step, and 6..7 by at most 1, the half step that the top interval 4..6 has anyway (on normal
// values 19.0 dB against 18.8 for a limit of 6 or 8).  Dequantised values are exact in bf16.
#include <float.h>
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "kv4_kernels.h"

namespace fmi {

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

constexpr int KV4_MIN_SCALE = 127 - 100;   // smallest block power 2^-100: every product below stays a normal number
constexpr int KV4_MAX_SCALE = 127 + 125;   // largest, 2^125: 6 * 2^125 is finite, 4 * 2^126 would not be
constexpr int KV4_NAN_SCALE = 255;

__device__ inline float kv4_scale(uint32_t b) { return __uint_as_float(b << 23); }

// 8 codes (one dword) -> 8 bf16 values; the conversion reads the exponent field of `scale` only, 255 there gives NaN
__device__ inline u32x4 kv4_unpack8(uint32_t codes, float scale) {
  u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  return r;
}
// two fp32 -> two bf16, round to nearest even
__device__ inline uint32_t kv4_pk_bf16(float lo, float hi) {
  const f32x2_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}
__device__ inline float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ inline float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// =====================================================================================
// append
// =====================================================================================

template <int MASK>
__device__ inline double xor_lane_d(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)xor_lane<MASK>((int)(uint32_t)u, lane), hi = (uint32_t)xor_lane<MASK>((int)(u >> 32), lane);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// 1 / sqrt(m) rounded to fp32: the fp32 estimate and two Newton steps in fp64 (error ~2^-52 before the rounding)
__device__ inline float kv4_rstd(double m) {
  if (!(m > 1e-30 && m < 1e30)) return (float)(1.0 / sqrt(m));
  double y = (double)__builtin_amdgcn_rsqf((float)m);
  const double h = 0.5 * m;
  y = y * (1.5 - h * y * y);
  y = y * (1.5 - h * y * y);
  return (float)y;
}

// A lane's 8 dims of a head: the norm weights and rotation factors that belong to them.  HALF: the rotation pairs dims rot / 2
// apart, so the other element of each pair is in another chunk, `xp`, which the lane reads and norms too.
template <int D, bool HALF>
struct Kv4Chunk {
  float wv[8], wp[8], cs[8], sn[8];

  __device__ inline void load_norm(const bf16_t* nw, int sub, int psub) {
    const u32x4 w0 = *reinterpret_cast<const u32x4*>(nw + sub * 8), w1 = *reinterpret_cast<const u32x4*>(nw + psub * 8);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wv[i] = i & 1 ? bf_hi(w0[i >> 1]) : bf_lo(w0[i >> 1]);
      if (HALF) wp[i] = i & 1 ? bf_hi(w1[i >> 1]) : bf_lo(w1[i >> 1]);
    }
  }
  // pos_tab: the position's rot / 2 (cos, sin).  Interleaved: cs / sn [i] of pair i (i < 4); half: of this lane's element i, the
  // sine negated for the first of a pair
  __device__ inline void load_rope(const bf16_t* pos_tab, int rot, int sub) {
    const int hr = rot / 2;
    const bool first = sub * 8 < hr;
    const bf16_t* tab = pos_tab + (HALF ? (first ? sub * 8 : sub * 8 - hr) * 2 : sub * 8);
    uint32_t t[8];
    *reinterpret_cast<u32x4*>(t) = *reinterpret_cast<const u32x4*>(tab);
    if (HALF) *reinterpret_cast<u32x4*>(t + 4) = *reinterpret_cast<const u32x4*>(tab + 8);
#pragma unroll
    for (int i = 0; i < (HALF ? 8 : 4); ++i) {
      cs[i] = bf_lo(t[i]);
      sn[i] = HALF && first ? -bf_hi(t[i]) : bf_hi(t[i]);
    }
  }
  // the D / 8 lanes of a head together
  __device__ inline void norm(u32x4& x, u32x4& xp, double eps, int lane) const {
    double ss = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double e0 = (double)bf_lo(x[i]), e1 = (double)bf_hi(x[i]);
      ss = fma(e0, e0, ss);
      ss = fma(e1, e1, ss);
    }
    ss += xor_lane_d<1>(ss, lane);
    ss += xor_lane_d<2>(ss, lane);
    if (D / 8 > 4) ss += xor_lane_d<4>(ss, lane);
    if (D / 8 > 8) ss += xor_lane_d<8>(ss, lane);
    const float rstd = kv4_rstd(ss * (1.0 / D) + eps);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = kv4_pk_bf16(bf_lo(x[i]) * rstd * wv[2 * i], bf_hi(x[i]) * rstd * wv[2 * i + 1]);
      if (HALF) xp[i] = kv4_pk_bf16(bf_lo(xp[i]) * rstd * wp[2 * i], bf_hi(xp[i]) * rstd * wp[2 * i + 1]);
    }
  }
  __device__ inline void rotate(u32x4& x, const u32x4& xp) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x0 = bf_lo(x[i]), x1 = bf_hi(x[i]);
      if (!HALF) x[i] = kv4_pk_bf16(x0 * cs[i] - x1 * sn[i], x1 * cs[i] + x0 * sn[i]);
      else x[i] = kv4_pk_bf16(x0 * cs[2 * i] + bf_lo(xp[i]) * sn[2 * i], x1 * cs[2 * i + 1] + bf_hi(xp[i]) * sn[2 * i + 1]);
    }
  }
};
// the chunk that holds the partners of chunk `sub`
__device__ inline int kv4_partner(int sub, int rot) { return sub * 8 < rot / 2 ? sub + rot / 16 : sub - rot / 16; }

// 8 dims -> 8 codes; 4 lanes hold a block.  -> its scale byte
__device__ inline uint32_t kv4_quantise(const u32x4& x, int lane, uint32_t& codes) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(x[i] & 0x7fffu, (x[i] >> 16) & 0x7fffu));
  top = max(top, (uint32_t)xor_lane<1>((int)top, lane));
  top = max(top, (uint32_t)xor_lane<2>((int)top, lane));
  const bool finite = top < 0x7f80u;
  // max = 1.f * 2^(exp - 127): the power with max <= 7 * 2^e is exp - 127 - 2, one more above f = 1.75
  const int b = min(max((int)(top >> 7) - 2 + ((top & 0x7fu) > 0x60u ? 1 : 0), KV4_MIN_SCALE), KV4_MAX_SCALE);
  const float sc = kv4_scale((uint32_t)b);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, (uint32_t)x[0]), sc, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, (uint32_t)x[1]), sc, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, (uint32_t)x[2]), sc, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, (uint32_t)x[3]), sc, 3);
  codes = finite ? r : 0u;
  return finite ? (uint32_t)b : (uint32_t)KV4_NAN_SCALE;
}
// ... and into the block of a page
template <int D>
__device__ inline void kv4_store(uint8_t* blk, int tok, int sub, uint32_t codes, uint32_t scale) {
  *reinterpret_cast<uint32_t*>(blk + tok * (D / 2) + sub * 4) = codes;
  if ((sub & 3) == 0) blk[KV_PAGE * (D / 2) + tok * (D / 32) + sub / 4] = (uint8_t)scale;
}

// D / 8 lanes own one (row, head), 8 dims each; a wave takes 64 / (D / 8) consecutive rows of one head, so its code bytes are
// consecutive in the page, and up to HC heads of one kind (q, k or v) one after the other: indices, page and rotation are
// looked up once for them, the next head's values are in flight.  grid (chunks of heads; groups of rows).  Every rounding
// is fixed by the definition (sum of squares in fp64, reciprocal norm and both products rounded to fp32, value to bf16;
// products of the rotation are exact in fp32, one rounding of their sum, then bf16), so the stored codes do not depend on
// how the lanes are arranged or on fused products.
// Bound by memory for prompts: 16 384 tokens of 32 + 8 + 8 heads x 128 dims (12 288 bytes read, 8 192 of q and 1 088 of codes
// written per token) take 67 to 74 us, 4.8 to 5.3 TB/s where a copy reaches 5.2.  One head per wave instead of eight: 104 us.
// Few tokens are bound by the launch (8 tokens: 2.2 to 3.4 us) and better off with every head in a wave of its own.
template <int D, bool HALF, int HC>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4AppendArgs a) {
  constexpr int LPH = D / 8, RPW = 64 / LPH, BLK = kv4_block_bytes(D);
  const int lane = threadIdx.x & 63, sub = lane % LPH;
  const int qc = (a.H + HC - 1) / HC, kc = (a.c.KVH + HC - 1) / HC, chunk = blockIdx.x;
  const int kind = chunk < qc ? 0 : chunk < qc + kc ? 1 : 2;   // q, k, v
  const int h0 = (kind == 0 ? chunk : kind == 1 ? chunk - qc : chunk - qc - kc) * HC;
  const int h1 = min(h0 + HC, kind == 0 ? a.H : a.c.KVH);
  const int64_t row64 = (((int64_t)blockIdx.z * 65535 + blockIdx.y) * 4 + (threadIdx.x >> 6)) * RPW + lane / LPH;
  const bool in_rows = row64 < a.rows;             // rows past the last one read row 0 and are dropped by their position
  const int64_t row = in_rows ? row64 : 0;
  const int64_t stride = kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride;
  const bf16_t* src = (kind == 0 ? a.q : kind == 1 ? a.k : a.v) + row * stride;
  const bf16_t* nw = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
  const bool rotated = kind != 2 && a.rope && sub * 8 < a.rot;
  const int psub = HALF && rotated ? kv4_partner(sub, a.rot) : sub;
  u32x4 nx = *reinterpret_cast<const u32x4*>(src + h0 * D + sub * 8), nxp;
  if (HALF) nxp = *reinterpret_cast<const u32x4*>(src + h0 * D + psub * 8);
  const int seq = in_rows ? a.row_seq[row] : -1;
  const bool seq_ok = seq >= 0 && seq < a.c.n_slots;
  const int pos = seq_ok ? a.row_pos[row] : -1;
  const bool valid = pos >= 0 && pos < (a.rope ? min(a.c.max_pages * KV_PAGE, a.rope_len) : a.c.max_pages * KV_PAGE);
  const bool rot = rotated && valid;
  const int page = kind != 0 && valid ? a.c.block_table[(int64_t)seq * a.c.max_pages + pos / KV_PAGE] : -1;
  Kv4Chunk<D, HALF> ch;
  if (nw) ch.load_norm(nw, sub, psub);
  if (rot) ch.load_rope(a.rope + (int64_t)pos * a.rot, a.rot, sub);
  const bool store = page >= 0 && page < a.c.n_pages;
  const int tok = pos % KV_PAGE;
  // (a lane without a page never uses its addresses)
  uint8_t* blk = a.c.pool + ((store ? (int64_t)page : 0) * a.c.KVH * 2 + (kind - 1)) * BLK;
#pragma unroll 1
  for (int h = h0; h < h1; ++h) {
    u32x4 x = nx, xp = nxp;
    if (HC > 1 && h + 1 < h1) {
      nx = *reinterpret_cast<const u32x4*>(src + (h + 1) * D + sub * 8);
      if (HALF) nxp = *reinterpret_cast<const u32x4*>(src + (h + 1) * D + psub * 8);
    }
    if (nw) ch.norm(x, xp, a.eps, lane);
    if (rot) ch.rotate(x, xp);
    if (kind == 0) {
      if (valid) *reinterpret_cast<u32x4*>(a.q_out + row * a.q_out_stride + h * D + sub * 8) = x;
      continue;
    }
    uint32_t codes;
    const uint32_t scale = kv4_quantise(x, lane, codes);
    if (store) kv4_store<D>(blk + (int64_t)h * 2 * BLK, tok, sub, codes, scale);
  }
}

static int kv4_check_cache(const Kv4Cache& c) {
  FMI_REQUIRE(c.pool && c.block_table, "kv4: null pool or block table");
  FMI_REQUIRE(c.D == 32 || c.D == 64 || c.D == 128, "kv4: head_dim %d unsupported (32/64/128)", c.D);
  FMI_REQUIRE(c.KVH >= 1 && c.n_pages >= 1 && c.n_slots >= 1 && c.max_pages >= 1,
              "kv4: n_kv_head %d, n_pages %d, n_seqs %d and max_pages %d must be positive", c.KVH, c.n_pages, c.n_slots, c.max_pages);
  FMI_REQUIRE(c.max_pages <= (1 << 24) && c.KVH <= (1 << 16), "kv4: max_pages %d, n_kv_head %d: at most 2^24, 2^16", c.max_pages, c.KVH);
  FMI_REQUIRE(((uintptr_t)c.pool & 15) == 0 && ((uintptr_t)c.block_table & 3) == 0, "kv4: misaligned pool or block table");
  return FMI_OK;
}

static int kv4_check_rows(const char* what, const void* p, int64_t stride, int heads, int D) {
  FMI_REQUIRE(p, "kv4: %s is null", what);
  FMI_REQUIRE(((uintptr_t)p & 15) == 0 && stride % 8 == 0 && stride >= (int64_t)heads * D,
              "kv4: %s needs 16-byte aligned rows of %d x %d values (row stride %lld)", what, heads, D, (long long)stride);
  return FMI_OK;
}

// grid of the row kernels: (heads, groups of `per` rows); y holds 65535 groups, z the rest
static dim3 kv4_row_grid(int64_t heads, int rows, int per) {
  const int64_t groups = ((int64_t)rows + per - 1) / per;
  return dim3((unsigned)heads, (unsigned)std::min<int64_t>(groups, 65535), (unsigned)((groups + 65534) / 65535));
}

static int kv4_check_append(const Kv4AppendArgs& a) {   // of an append or a step
  FMI_CHECK(kv4_check_cache(a.c));
  const int D = a.c.D;
  FMI_CHECK(kv4_check_rows("k", a.k, a.k_stride, a.c.KVH, D));
  FMI_CHECK(kv4_check_rows("v", a.v, a.v_stride, a.c.KVH, D));
  FMI_REQUIRE(a.row_seq, "kv4: null row sequences");
  if (a.q) {
    FMI_REQUIRE(a.H >= 1 && a.H <= (1 << 16), "kv4 append: q of %d query heads (1 to 2^16)", a.H);
    FMI_CHECK(kv4_check_rows("q", a.q, a.q_stride, a.H, D));
  } else {
    FMI_REQUIRE(a.H == 0 && !a.q_norm, "kv4 append: query heads or q_norm without q");
  }
  FMI_REQUIRE(((uintptr_t)a.q_norm & 15) == 0 && ((uintptr_t)a.k_norm & 15) == 0, "kv4 append: misaligned norm weight");
  if (a.rope) {
    FMI_REQUIRE(((uintptr_t)a.rope & 15) == 0 && a.rope_len >= 1, "kv4 append: empty or misaligned rotation table");
    FMI_REQUIRE(a.rot >= 16 && a.rot <= D && a.rot % 16 == 0, "kv4 append: %d rotated dims (a multiple of 16 up to head_dim %d)", a.rot, D);
  }
  return FMI_OK;
}

int launch_kv4_append(const Kv4AppendArgs& a, hipStream_t s) {
  FMI_REQUIRE(a.rows >= 0, "kv4 append: negative row count");
  if (a.rows == 0) return FMI_OK;
  FMI_CHECK(kv4_check_append(a));
  FMI_REQUIRE(a.row_pos, "kv4 append: null row positions");
  const int D = a.c.D;
  if (a.q) {
    FMI_CHECK(kv4_check_rows("q_out", a.q_out, a.q_out_stride, a.H, D));
    FMI_REQUIRE(a.q_out != a.q || (a.q_out_stride == a.q_stride && !(a.rope && a.half)),
                "kv4 append: q_out over q needs the same row stride and no half-split rotation");
  }
  // one head per wave / eight, in us by the call's values: 32 + 16 heads x 128 dims 2^21.6 5.5 / 8.6, 2^22.6 9.4 / 10.6, 2^23.6 14.7 /
  // 12.9, 2^26.6 104 / 73; 14 + 4 heads x 64 dims 2^22.2 8.0 / 9.7, 2^23.2 12.1 / 12.6, 2^24.2 19.3 / 18.8
  const bool half = a.rope && a.half, many = (int64_t)a.rows * (a.H + 2 * a.c.KVH) * D > (int64_t)1 << 23;
  const int hc = many ? 8 : 1;
  const dim3 grid = kv4_row_grid((a.H + hc - 1) / hc + 2 * ((a.c.KVH + hc - 1) / hc), a.rows, 4 * (64 / (D / 8)));
#define FMI_KV4_APPEND(D_)                                                                                             \
  do {                                                                                                                 \
    if (many && half) hipLaunchKernelGGL((kv4_append_kernel<D_, true, 8>), grid, dim3(256), 0, s, a);                  \
    else if (many) hipLaunchKernelGGL((kv4_append_kernel<D_, false, 8>), grid, dim3(256), 0, s, a);                    \
    else if (half) hipLaunchKernelGGL((kv4_append_kernel<D_, true, 1>), grid, dim3(256), 0, s, a);                     \
    else hipLaunchKernelGGL((kv4_append_kernel<D_, false, 1>), grid, dim3(256), 0, s, a);                              \
  } while (0)
  if (D == 128) FMI_KV4_APPEND(128);
  else if (D == 64) FMI_KV4_APPEND(64);
  else FMI_KV4_APPEND(32);
#undef FMI_KV4_APPEND
  FMI_CHECK_HIP(hipGetLastError());
  return FMI_OK;
}

// =====================================================================================
// read-back
// =====================================================================================

// the append's arrangement: a wave takes 64 / (D / 8) rows, a lane 8 dims, and HC of the 2 n_kv_head blocks of K and V of a
// page, whose codes are all requested before the first is unpacked: a row's three dependent lookups (indices, page, codes)
// are paid once for HC blocks (32 768 rows of 8 heads, one launch after the other: 38 us = 4.5 TB/s, one block per wave 55;
// 130 rows: 2.7 us, the launch)
template <int D, int HC>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4ReadArgs a) {
  constexpr int LPH = D / 8, RPW = 64 / LPH, BLK = kv4_block_bytes(D);
  const int lane = threadIdx.x & 63, sub = lane % LPH;
  const int hb0 = blockIdx.x * HC, blocks = 2 * a.c.KVH;
  const int64_t row = (((int64_t)blockIdx.z * 65535 + blockIdx.y) * 4 + (threadIdx.x >> 6)) * RPW + lane / LPH;
  if (row >= a.rows) return;
  const int seq = a.row_seq ? a.row_seq[row] : a.seq0, pos = a.row_seq ? a.row_pos[row] : (int)row;
  int page = -1;
  if (seq >= 0 && seq < a.c.n_slots && pos >= 0 && pos < a.c.max_pages * KV_PAGE)
    page = a.c.block_table[(int64_t)seq * a.c.max_pages + pos / KV_PAGE];
  const bool there = page >= 0 && page < a.c.n_pages;
  uint32_t code[HC], scale[HC];
  const uint8_t* base = a.c.pool + ((there ? (int64_t)page : 0) * blocks + hb0) * BLK;
  const int tok = there ? pos % KV_PAGE : 0, c_off = tok * (D / 2) + sub * 4, s_off = KV_PAGE * (D / 2) + tok * (D / 32) + sub / 4;
#pragma unroll
  for (int i = 0; i < HC; ++i) {
    const int64_t o = (int64_t)min(i, blocks - 1 - hb0) * BLK;
    code[i] = *reinterpret_cast<const uint32_t*>(base + o + c_off);
    scale[i] = base[o + s_off];
  }
#pragma unroll
  for (int i = 0; i < HC; ++i) {
    const int hb = hb0 + i;
    if (hb >= blocks) break;
    const u32x4 x = kv4_unpack8(there ? code[i] : 0u, kv4_scale(there ? scale[i] : 127u));
    *reinterpret_cast<u32x4*>((hb & 1 ? a.v : a.k) + (row * a.c.KVH + (hb >> 1)) * D + sub * 8) = x;
  }
}

int launch_kv4_read(const Kv4ReadArgs& a, hipStream_t s) {
  FMI_REQUIRE(a.rows >= 0, "kv4 read: negative row count");
  if (a.rows == 0) return FMI_OK;
  FMI_CHECK(kv4_check_cache(a.c));
  const int D = a.c.D;
  FMI_REQUIRE(!a.row_seq == !a.row_pos, "kv4 read: null row indices");
  FMI_CHECK(kv4_check_rows("k", a.k, (int64_t)a.c.KVH * D, a.c.KVH, D));
  FMI_CHECK(kv4_check_rows("v", a.v, (int64_t)a.c.KVH * D, a.c.KVH, D));
  // one block per wave / eight, in us by the values of K: 8 heads x 128 dims 2^19 3.4 / 3.6, 2^21 4.8 / 4.6, 2^22 7.1 / 6.4, 2^24 19.3 /
  // 16.3; 2 heads x 64 dims 2^17 3.1 / 3.3, 2^20 4.0 / 3.8, 2^21 4.9 / 4.6
  const bool many = (int64_t)a.rows * a.c.KVH * D > (int64_t)1 << 21;
  const dim3 grid = kv4_row_grid((2 * a.c.KVH + (many ? 7 : 0)) / (many ? 8 : 1), a.rows, 4 * (64 / (D / 8)));
#define FMI_KV4_READ(D_)                                                                              \
  do {                                                                                                \
    if (many) hipLaunchKernelGGL((kv4_read_kernel<D_, 8>), grid, dim3(256), 0, s, a);                 \
    else hipLaunchKernelGGL((kv4_read_kernel<D_, 1>), grid, dim3(256), 0, s, a);                      \
  } while (0)
  if (D == 128) FMI_KV4_READ(128);
  else if (D == 64) FMI_KV4_READ(64);
  else FMI_KV4_READ(32);
#undef FMI_KV4_READ
  FMI_CHECK_HIP(hipGetLastError());
  return FMI_OK;
}

// =====================================================================================
// attention
// =====================================================================================
//
// out[row][head] = sum_key softmax_key(scale * q . k) v over the keys [0, pos(row)] of the row's sequence; a row
// without keys gives 0.  Query columns -- column = (query row, head of the kv head's group), so K and V are read once for
// all heads of a group -- are cut into tiles; a work-group owns a tile and one of up to `splits` ranges of its keys.
// Keys that a column may not see enter neither the maximum nor the sum nor, where their V is NaN, the product: such blocks
// are read as 0 and the columns that do see them are set to NaN at the end.
struct Kv4Span {       // one sequence's query rows and keys, clamped to what the buffers hold
  int slot, row0, nq, pos0, cached;   // pos0: position of the first query row (negative: sees nothing)
};
__device__ inline Kv4Span kv4_span(const Kv4AttnArgs& a, int s) {
  Kv4Span r;
  if (a.step_len > 0) {      // one row, at a given position; none if that or its sequence is not there
    const int seq = a.seq_slot[s];
    const bool seq_ok = seq >= 0 && seq < a.c.n_slots;
    r.slot = seq_ok ? seq : 0;
    r.row0 = s;
    r.pos0 = seq_ok ? (a.row_pos ? a.row_pos[s] : a.slot_pos[r.slot]) : -1;
    r.nq = r.pos0 >= 0 && r.pos0 < a.step_len;
    r.cached = r.pos0 + 1;
    return r;
  }
  r.slot = a.seq_slot ? a.seq_slot[s] : s;
  r.row0 = min(max(a.q_start[s], 0), a.total_q);
  const int n = max(min(a.q_start[s + 1], a.total_q) - r.row0, 0), kv = min(max(a.kv_len[s], 0), 1 << 30);
  r.nq = min(n, a.max_q);
  r.pos0 = kv - n;
  r.cached = (int)min((int64_t)kv, (int64_t)a.c.max_pages * KV_PAGE);
  return r;
}

// pages of 64 keys that the tile of `tile_cols` columns from col0 sees
__device__ inline int kv4_tile_pages(const Kv4Span& sp, int G, int col0, int tile_cols) {
  const int nk = min(sp.pos0 + min(col0 + tile_cols - 1, sp.nq * G - 1) / G + 1, sp.cached);
  return nk > 0 ? (nk + KV_PAGE - 1) / KV_PAGE : 0;
}
// the ranges a tile of np pages really uses: a function of the tile alone.  One range: its work-group writes the output itself
// and the merge passes the tile's rows by.  Below KV4_SINGLE_PAGES it is one (8 x 512 keys 7.5 us, in two ranges and a merge
// 9.1; 8 x 1k 10.5 and 9.9; 8 x 2k 16.3 and 12.7), above it a range has KV4_MIN_PAGES at least (a block per wave of a narrow
// tile).
constexpr int KV4_MIN_PAGES = 4;
__device__ inline int kv4_attn_ranges(const Kv4AttnArgs& a, int np) {
  return np < KV4_SINGLE_PAGES ? 1 : max(1, min(a.splits, np / KV4_MIN_PAGES));
}

// partial states of the key ranges: (m, l) pairs [splits][total_q * H][2], then O [splits][total_q * H][D]
__device__ inline float* kv4_part_ml(const Kv4AttnArgs& a, int z, int64_t idx) {
  return a.part + ((int64_t)z * a.total_q * a.H + idx) * 2;
}
template <int D>
__device__ inline float* kv4_part_o(const Kv4AttnArgs& a, int z, int64_t idx) {
  const int64_t n = (int64_t)a.total_q * a.H;
  return a.part + (a.splits * n * 2 + 3) / 4 * 4 + (z * n + idx) * D;
}

// max / sum over lanes l, l ^ 32 and over l, l ^ 16 inside the VALU
__device__ inline float max_swap32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float max_swap16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float sum_swap32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ inline float sum_swap16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 8 values of q.  Negated for a negative scale: the largest product is then the largest score; 0 for a scale of 0, whose
// products are left as they are (a hidden key's minus infinity times 0 would be NaN).  With an infinity among them the
// scores are infinite or NaN and the row's softmax NaN; as NaNs from the start they cannot all be minus infinity, which would
// pass for a row without keys.
__device__ inline void kv4_prepare_q(u32x4& t, float scale) {
  if (scale < 0.f) t ^= 0x80008000u;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(t[i] & 0x7fffu, (t[i] >> 16) & 0x7fffu));
  if (scale == 0.f) t = (u32x4){0, 0, 0, 0};
  if (top >= 0x7f80u) t = (u32x4){0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
}

// scores in units of log2
__device__ inline float kv4_log2_scale(float scale) { return scale == 0.f ? 1.f : fabsf(scale) * 1.4426950408889634f; }

// A running reference r of a softmax whose weights are 2^(s sl - r), set when its largest score reaches mx: `above` it, and by two
// steps of mx more, so that no weight exceeds 2^-above whatever the rounding of large scores.  r itself goes into every weight and
// into every change of reference: both round alike.
__device__ inline float kv4_reference(float mx, float above) { return fmaf(fabsf(mx), 0x1p-22f, mx + above); }

// ---- few query columns: tiles of 16, the kernel of single tokens.  NW waves; wave w takes the 32-key blocks w, w + NW, ...
// of the range.  Per block:
//   scores   S^T = K Q^T, v_mfma_f32_16x16x32_bf16: lane (c, g) holds the D / 4 dims from g D / 4 of key c, which is one
//            consecutive piece of the page and one scale; Q is read in the same order, so no dim is moved;
//   softmax  fp32, online, per column; the probabilities stay in registers as the B operand of the next product, split
//            into bf16 high and low parts (two products: 16 significant bits of weight);
//   output   O^T += V^T P: V is unpacked to bf16 into the wave's LDS rows and read back transposed by
//            ds_read_b64_tr_b16 (4 keys of one dim per lane).
// The next block's codes are in flight during a block's arithmetic.  The waves' (m, l, O) are merged through LDS in wave
// order.  Bound by memory once the card is full: 64 x 8k keys of 8 kv heads x 128 dims 110 us = 5.2 TB/s, 64 x 16k 202 us =
// 5.65; 32 sequences of 4k to 8k keys 50 us = 4.3 TB/s (the longest sequences' work-groups run on alone at the end); 1 x 128k
// 36 us = 3.9 TB/s (the merge is 4 us of it).  One sequence of 300 keys is 5 to 6.5 us of dependent loads (lengths, page,
// codes) and two blocks of arithmetic.  Of 4, 8 and 16 waves, 8 were the fastest.
//
// STEP 1 / 2 (rotation interleaved / half split): a generation step of one new token per sequence in the same launch.  Every
// work-group norms and rotates its own query heads (into LDS rows); the one of a kv head's last range also quantises the new
// token's K and V, stores them, and puts them over what it fetched of that token: nothing is read back from memory, and no
// other work-group reads that token.  The values and their bits are those of an append followed by an attention.  In a
// captured graph 8 x 300 keys take 8.5 us where the two launches take 9.7, 16 x 1k 13.1 and 14.3, 32 x 6k 50 and 52; a
// model's frame of 36 layers went from 4.15 to 4.09 ms at 200 tokens, the host's part of a call pair from 18.8 to 10.8 us.
struct Kv4None {};
template <int D, int NW, int STEP>
__global__ __launch_bounds__(64 * NW) void kv4_attn_kernel(Kv4AttnArgs a, std::conditional_t<STEP != 0, Kv4AppendArgs, Kv4None> p) {
  constexpr int KB = 32, NT = 64 * NW, BLK = kv4_block_bytes(D), NB = D / 32;
  constexpr int KS = D / 32;                     // k-steps of a score product
  constexpr int VROW = D * 2 + 32;               // bytes of a key's row in LDS: 32 more, so that the 4 rows a 16-lane
                                                 // group reads together lie in different banks (the writes' conflicts:
                                                 // 8 cycles of 18 each)
  constexpr int VL = D / 32, VP = 64 / VL;       // lanes per key and keys per pass of the V unpacking
  constexpr int VPASS = VP >= KB ? 1 : KB / VP;
  __shared__ __attribute__((aligned(16))) unsigned char s_v[NW][KB * VROW];
  __shared__ float s_m[NW][16], s_l[NW][16];
  __shared__ int s_nan[NW][NB];
  static_assert(KB * VROW >= 16 * D * 4, "the merge keeps a wave's 16 x D fp32 sums where its V rows were");

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int KVH = a.c.KVH, G = a.H / KVH;
  const int tile = blockIdx.x / KVH, kvh = blockIdx.x % KVH, z = blockIdx.y;
  const Kv4Span sp = kv4_span(a, blockIdx.z);
  const int cols = sp.nq * G, col0 = tile * 16;
  if (col0 >= cols) return;
  const int np = kv4_tile_pages(sp, G, col0, 16), nz = kv4_attn_ranges(a, np);
  if (z >= nz) return;
  const int col = min(col0 + c, cols - 1);
  const int qrow = sp.row0 + col / G, head = kvh * G + col % G;
  const int vis = min(sp.pos0 + col / G + 1, sp.cached);          // keys [0, vis) are this column's
  const int all_see = min(sp.pos0 + col0 / G + 1, sp.cached);     // keys that every column of the tile sees
  const int b_lo = (int)((int64_t)z * np / nz) * 2, b_hi = (int)((int64_t)(z + 1) * np / nz) * 2;
  const int32_t* bt = a.c.block_table + (int64_t)sp.slot * a.c.max_pages;

  // the new token: D / 8 lanes per head, the tile's query heads, then K, then V; requested before the codes, which take longer
  constexpr int LPH = D / 8, QROW = D * 2 + 16;
  static_assert(NT / LPH >= 18, "16 query heads, K and V at a time");
  __shared__ __attribute__((aligned(16))) unsigned char s_q[STEP ? 16 * QROW : 16];
  __shared__ __attribute__((aligned(16))) uint32_t s_code[STEP ? 2 : 1][LPH];
  __shared__ uint32_t s_scale[STEP ? 2 : 1][NB];
  Kv4Chunk<D, STEP == 2> ch;
  u32x4 x, xp;
  const int item = tid / LPH, sub = tid % LPH, heads = min(16, cols - col0), newest = z == nz - 1 ? sp.pos0 / KB : -1;
  bool normed = false, rotated = false;
  if constexpr (STEP != 0) {
    const int64_t row = sp.row0;
    const bf16_t* src = p.q + row * p.q_stride + (kvh * G + col0 + min(item, heads - 1)) * D;
    const bf16_t* nw = p.q_norm;
    if (item == heads) {
      src = p.k + row * p.k_stride + kvh * D;
      nw = p.k_norm;
    } else if (item == heads + 1) {
      src = p.v + row * p.v_stride + kvh * D;
      nw = nullptr;
    }
    normed = nw;
    rotated = p.rope && item != heads + 1 && sub * 8 < p.rot;
    const int psub = STEP == 2 && rotated ? kv4_partner(sub, p.rot) : sub;
    x = *reinterpret_cast<const u32x4*>(src + sub * 8);
    if (STEP == 2) xp = *reinterpret_cast<const u32x4*>(src + psub * 8);
    if (normed) ch.load_norm(nw, sub, psub);
    if (rotated) ch.load_rope(p.rope + (int64_t)sp.pos0 * p.rot, p.rot, sub);
  }

  // K and V codes and scales of one block; a missing page reads page 0 and is skipped later.  A lane's place in the block is
  // fixed: 32-bit offsets from a scalar base.
  u32x4 vcode[VPASS];
  uint32_t kcode[2][KS], kscale[2], vscale[VPASS];
  const uint32_t k_off = c * (D / 2) + g * (D / 8), ks_off = c * NB + g * NB / 4;
  const uint32_t vkey = VP <= KB ? lane / VL : min(lane, KB - 1), v_off = vkey * (D / 2) + lane % VL * 16, vs_off = vkey * NB + lane % VL;
  auto fetch = [&](int kb, int page) {
    const int pg = page >= 0 && page < a.c.n_pages ? page : 0, tok0 = kb & 1 ? KB : 0;
    const uint8_t* kblk = a.c.pool + ((int64_t)pg * KVH + kvh) * 2 * BLK;
    const uint8_t *kc = kblk + tok0 * (D / 2), *ksc = kblk + KV_PAGE * (D / 2) + tok0 * NB;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const uint8_t* kp = kc + (k_off + kt * 16 * (D / 2));
      if constexpr (D == 128) *reinterpret_cast<u32x4*>(kcode[kt]) = *reinterpret_cast<const u32x4*>(kp);
      else if constexpr (D == 64) *reinterpret_cast<uint2*>(kcode[kt]) = *reinterpret_cast<const uint2*>(kp);
      else kcode[kt][0] = *reinterpret_cast<const uint32_t*>(kp);
      kscale[kt] = ksc[ks_off + kt * 16 * NB];
    }
#pragma unroll
    for (int it = 0; it < VPASS; ++it) {
      vcode[it] = *reinterpret_cast<const u32x4*>(kc + BLK + (v_off + it * VP * (D / 2)));
      vscale[it] = (ksc + BLK)[vs_off + it * VP * NB];
    }
  };
  auto page_of = [&](int kb) { return kb < b_hi ? bt[kb >> 1] : -1; };

  int kb = b_lo + wave;
  int page = page_of(kb);
  if (kb < b_hi) fetch(kb, page);
  int next_page = page_of(kb + NW);

  if constexpr (STEP != 0) {
    if (normed) ch.norm(x, xp, p.eps, lane);
    if (rotated) ch.rotate(x, xp);
    if (item < heads) *reinterpret_cast<u32x4*>(s_q + item * QROW + sub * 16) = x;
    uint32_t codes;
    const uint32_t scale = kv4_quantise(x, lane, codes);
    const int kv = item - heads;
    if (newest >= 0 && (kv == 0 || kv == 1)) {
      s_code[kv][sub] = codes;
      if ((sub & 3) == 0) s_scale[kv][sub / 4] = scale;
      const int pg = bt[sp.pos0 / KV_PAGE];
      if (pg >= 0 && pg < a.c.n_pages && !(p.slot_done && p.slot_done[sp.slot]))
        kv4_store<D>(a.c.pool + (((int64_t)pg * KVH + kvh) * 2 + kv) * BLK, sp.pos0 % KV_PAGE, sub, codes, scale);
    }
    __syncthreads();
  }
  bf16x8 qf[KS];                                 // B operand: column c, dims g D / 4 + 8 kk ..
  {
    const bf16_t* qp = STEP ? nullptr : a.q + qrow * a.q_stride + (int64_t)head * D + g * (D / 4);
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      u32x4 t = STEP ? *reinterpret_cast<const u32x4*>(s_q + min(c, heads - 1) * QROW + (g * (D / 4) + kk * 8) * 2)
                     : *reinterpret_cast<const u32x4*>(qp + kk * 8);
      kv4_prepare_q(t, a.scale);
      qf[kk] = *reinterpret_cast<bf16x8*>(&t);
    }
  }
  f32x4 o[D / 16];
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) o[dt] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float m = -FLT_MAX, l = 0.f;                   // l: this lane's keys only, joined after the loop
  int nan_key[NB];                               // first key whose V block is NaN, per 32-dim block
#pragma unroll
  for (int i = 0; i < NB; ++i) nan_key[i] = INT32_MAX;
  const float sl = kv4_log2_scale(a.scale);
  unsigned char* sv = s_v[wave];
  const unsigned char* vr = sv + (g * 4 + (c >> 2)) * VROW + (c & 3) * 8;

  for (; kb < b_hi; kb += NW) {
    const bool there = page >= 0 && page < a.c.n_pages;
    if (there) {
      if (STEP != 0 && kb == newest) {     // the new token's K and V over what the page held there
        const int key_new = sp.pos0 % KB;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
          if (kt * 16 + c == key_new) {
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) kcode[kt][kk] = s_code[0][g * KS + kk];
            kscale[kt] = s_scale[0][g * NB / 4];
          }
#pragma unroll
        for (int it = 0; it < VPASS; ++it)
          if (it * VP + lane / VL == key_new) {
            vcode[it] = *reinterpret_cast<const u32x4*>(&s_code[STEP ? 1 : 0][lane % VL * 4]);
            vscale[it] = s_scale[STEP ? 1 : 0][lane % VL];
          }
      }
      // ---- scores
      f32x4 sacc[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const float ks = kv4_scale(kscale[kt]);
        sacc[kt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
          u32x4 kf = kv4_unpack8(kcode[kt][kk], ks);
          sacc[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<bf16x8*>(&kf), qf[kk], sacc[kt], 0, 0, 0);
        }
      }
      // ---- V -> bf16 rows in LDS; rows past the sequence's keys hold whatever was there before: read as 0
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
      __builtin_amdgcn_wave_barrier();             // the previous block's reads are done (same wave)
      const bool whole = kb * KB + KB <= sp.cached;
#pragma unroll
      for (int it = 0; it < VPASS; ++it) {
        const int key = it * VP + lane / VL, part = lane % VL;
        if (VP <= KB || key < KB) {
          const bool use = whole || kb * KB + key < sp.cached, bad = use && vscale[it] == KV4_NAN_SCALE;
          if (__builtin_amdgcn_ballot_w64(bad)) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
              const uint64_t hit = __builtin_amdgcn_ballot_w64(bad && part == i);
              if (hit) nan_key[i] = min(nan_key[i], kb * KB + it * VP + (int)__builtin_ctzll(hit) / VL);
            }
          }
          if (!use || bad) {
            vcode[it] = (u32x4){0, 0, 0, 0};
            vscale[it] = 127;
          }
          const float vs = kv4_scale(vscale[it]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<u32x4*>(sv + key * VROW + part * 64 + i * 16) = kv4_unpack8(vcode[it][i], vs);
        }
      }
      const int kb_cur = kb;
      if (kb + NW < b_hi) fetch(kb + NW, next_page);
      // ---- softmax: lane (c, g) holds keys kt * 16 + g * 4 + j of column c
      float t[8], mx = -INFINITY;
      const bool part = kb_cur * KB + KB > all_see;
      const int lim = vis - kb_cur * KB - g * 4;
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = sacc[i >> 2][i & 3];
      if (part) {       // an unseen key's score is minus infinity whatever its K holds
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!((i >> 2) * 16 + (i & 3) < lim)) t[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, t[i]);
      mx = max_swap32(max_swap16(mx));
      // the reference m lies 2^8 above the largest score when it moves, and moves when a score exceeds it: O is seldom rescaled, no
      // weight is above 1 and O no larger than with the true maximum (V may be as large as 2^127)
      const float mn = fmaf(mx, sl, -m) > 0.f ? kv4_reference(mx * sl, 8.f) : m, corr = __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = __builtin_amdgcn_exp2f(fmaf(t[i], sl, -mn));
      l = l * corr + (((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7])));
      m = mn;
      u32x4 ph, pl;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ph[i] = kv4_pk_bf16(t[2 * i], t[2 * i + 1]);
        pl[i] = kv4_pk_bf16(t[2 * i] - bf_lo(ph[i]), t[2 * i + 1] - bf_hi(ph[i]));
      }
      if (__builtin_amdgcn_ballot_w64(corr != 1.f)) {
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[dt][j] *= corr;
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
      __builtin_amdgcn_wave_barrier();             // this wave's V rows are complete
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
      // ---- O^T += V^T P: lanes 4 r .. 4 r + 3 of a 16-lane group name row (key) r, lane i gets column (dim) i of the 4
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vr + dt * 32));
        const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vr + 16 * VROW + dt * 32));
        const bf16x8 vf = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
        o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, *reinterpret_cast<bf16x8*>(&ph), o[dt], 0, 0, 0);
        o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, *reinterpret_cast<bf16x8*>(&pl), o[dt], 0, 0, 0);
      }
    } else if (kb + NW < b_hi) {
      fetch(kb + NW, next_page);
    }
    page = next_page;
    next_page = page_of(kb + 2 * NW);
  }

  // ---- merge the waves in wave order
  l = sum_swap32(sum_swap16(l));
  const int ncol = min(16, cols - col0);
  __syncthreads();
  float* s_o = reinterpret_cast<float*>(&s_v[0][0]);       // NW rows of 16 x D sums, KB * VROW bytes apart
  constexpr int SO = KB * VROW / 4;
  if (g == 0) {
    s_m[wave][c] = m;
    s_l[wave][c] = l;
  }
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < NB; ++i) s_nan[wave][i] = nan_key[i];
  if (c < ncol) {
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) *reinterpret_cast<f32x4*>(s_o + wave * SO + c * D + dt * 16 + g * 4) = o[dt];
  }
  __syncthreads();
  for (int i = tid; i < ncol * D; i += NT) {
    const int cc = i / D, d = i % D;
    const int row = (col0 + cc) / G, hd = kvh * G + (col0 + cc) % G;
    float M = -FLT_MAX;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, s_m[w][cc]);
    float L = 0.f, O = 0.f;
    int bad = INT32_MAX;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float wgt = __builtin_amdgcn_exp2f(s_m[w][cc] - M);
      L += s_l[w][cc] * wgt;
      O += s_o[w * SO + cc * D + d] * wgt;
      bad = min(bad, s_nan[w][d / 32]);
    }
    if (bad < min(sp.pos0 + row + 1, sp.cached)) O = __uint_as_float(0x7fc00000u);
    if (nz == 1) {
      a.out[(sp.row0 + row) * a.out_stride + (int64_t)hd * D + d] = L != 0.f ? f2bf(O / L) : (bf16_t)0;
    } else {
      const int64_t idx = (int64_t)(sp.row0 + row) * a.H + hd;
      kv4_part_o<D>(a, z, idx)[d] = O;
      if (d == 0) {
        kv4_part_ml(a, z, idx)[0] = M;
        kv4_part_ml(a, z, idx)[1] = L;
      }
    }
  }
}

// ---- many query columns: tiles of 32 NW = 128, the kernel of prompts.  NW waves of 32 columns each share the pages of 64 keys,
// staged once per work-group: K unpacked to bf16 and V to fp16 rows in LDS, two buffers and one barrier per page, the next
// page's codes in flight during a page's arithmetic.  Per page and wave:
//   scores   S^T = K Q^T, v_mfma_f32_32x32x16_bf16, Q in registers for the whole kernel;
//   softmax  as above; the probabilities are rounded to fp16 (11 bits: with bf16's 8 a second product with the remainder
//            would be needed, half as much matrix work again) and stay in registers.  fp16 has few powers of two, so all of
//            them are used: the largest probability is 2^10 when the reference m is set and m moves when one would pass 2^15.
//            11 bits then hold down to 2^-24 of the largest, and only what is under 2^-35 of it rounds to 0 (around 1: 2^-14
//            and 2^-25, which is where the keys beside an attention sink lie).  2^3 between the two instead of 2^5 costs 2 %
//            more (rescales), 2^8 nothing less;
//   output   O^T += V^T P, v_mfma_f32_32x32x16_f16, V^T by ds_read_b64_tr_b16.
// V is held in fp16 relative to 2^E, E = the largest block power of the range's first key, which every row sees that sees
// any key of it.  fp16 is sound only while powers are alike: while every block's is within 2^-4 .. 2^5 of 2^E, V is exact and
// the weights that round to 0 lose less than 2^-23 of the weights' sum of block powers per key (n keys under 2^-35, 7 * 2^(4 + 5)).
// From the first key on that has another power (`first_out`; an all-zero block has the smallest there is), the rows that see
// it go on in bf16, whose powers are fp32's: V exact, the weights as high and low part (16 bits), a second product.  The page
// of that key is taken twice, for the rows before it in fp16 and for those from it on in bf16; what a row gives depends on no
// key behind it, on no other row and not on the tile that it is in.  fp16 / bf16 from the first page on: 8 prompts of 2k tokens
// over 4k keys 1431 / 1805 us, two ragged ones 246 / 284, 8 ragged prompts of up to 200 tokens 15.6 / 18.6.
// Bound by issue: per page and wave 32 matrix instructions (34 % of the time) and 245 others (42 %), two waves per SIMD to
// overlap them.  8 prompts of 2k tokens over 4k keys run at 960 TFLOP/s, two ragged ones at 850 (224 us where calls come one by
// one, 246 without a pause between them; the last work-groups run alone), 8 ragged prompts of up to 200 tokens in 14.7 us,
// mostly the latency of their 1 to 4 pages.
// The native product of 4-bit K with Q in two 8-bit parts needs no unpacking and the same matrix time, but its sums came out
// 9e-5 of the absolute sum away from the exact ones (bf16 products: 1e-7), too coarse for scores.
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;

__device__ inline u32x4 kv4_unpack8_f16(uint32_t codes, float scale) {
  u32x4 r;
  r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0));
  r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1));
  r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2));
  r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3));
  return r;
}
__device__ inline uint32_t kv4_pk_f16(float lo, float hi) {
  const f32x2_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
}

template <int D, int NW>
__global__ __launch_bounds__(64 * NW, 2) void kv4_attn_wide_kernel(Kv4AttnArgs a) {
  constexpr int NT = 64 * NW, BLK = kv4_block_bytes(D), NB = D / 32, TC = 32 * NW;
  // LDS rows: K reads take 16 keys at 16 bytes each (rows 4 banks apart), V reads 4 keys at 2 x 32 bytes (16 banks apart), both
  // without bank conflicts.  The writes have some: 8 cycles per 16-byte write on top of its 10, for V because the four words of
  // a piece go out in an order that differs by key (24 in the same order).  64 of a page's 3000 cycles per wave.
  constexpr int KROW = D * 2 + 16, VROW = D * 2 + (D > 32 ? 64 : 0);
  constexpr int PIECES = 2 * KV_PAGE * NB;                  // 16-byte pieces (32 codes) of K and V of a page
  constexpr int PPT = (PIECES + NT - 1) / NT;
  constexpr float DEFER = 5.f, TOP = 15.f;                  // powers of two: see "softmax" above
  constexpr uint32_t BELOW = 4, ABOVE = 5;                  // V's powers around E
  __shared__ __attribute__((aligned(16))) unsigned char s_k[2][KV_PAGE * KROW];
  __shared__ __attribute__((aligned(16))) unsigned char s_v[2][KV_PAGE * VROW];
  __shared__ int s_nan[NB];

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int KVH = a.c.KVH, G = a.H / KVH;
  // heads fastest (the work-groups of a kv head's keys share an XCD and its L2 when there are 8), then a sequence's tiles from
  // the one with the most keys down, then sequences (sequences before tiles: 326 us for 240 on two ragged 2k-token prompts
  // over 4k keys, 129 for 96 on four ragged prompts of up to 2k; even at best elsewhere)
  const int kvh = blockIdx.x % KVH, z = blockIdx.y;
  const Kv4Span sp = kv4_span(a, blockIdx.z);
  const int cols = sp.nq * G, tiles = (cols + TC - 1) / TC;
  const int tile = tiles - 1 - (int)(blockIdx.x / KVH);
  if (tile < 0) return;
  const int col0 = tile * TC;
  const int np = kv4_tile_pages(sp, G, col0, TC), nz = kv4_attn_ranges(a, np);
  if (z >= nz) return;
  const int p_lo = (int)((int64_t)z * np / nz), p_hi = (int)((int64_t)(z + 1) * np / nz);
  const int wcol = col0 + 32 * wave;                        // this wave's first column
  const int col = min(wcol + c, cols - 1);
  const int qrow = sp.row0 + col / G, head = kvh * G + col % G;
  int vis = min(sp.pos0 + col / G + 1, sp.cached);             // keys [0, vis) are this column's (of the phase, below)
  const int seen = vis;
  // keys that all / any of the wave's columns see (a wave behind the last column sees none), and of the tile's
  int all_see = min(sp.pos0 + min(wcol, cols - 1) / G + 1, sp.cached);
  int any_see = wcol < cols ? min(sp.pos0 + min(wcol + 31, cols - 1) / G + 1, sp.cached) : 0;
  const int tile_any = min(sp.pos0 + min(col0 + TC - 1, cols - 1) / G + 1, sp.cached);
  const int32_t* bt = a.c.block_table + (int64_t)sp.slot * a.c.max_pages;

  if (tid < NB) s_nan[tid] = INT32_MAX;
  bf16x8 qf[D / 16];
  {
    const bf16_t* qp = a.q + qrow * a.q_stride + (int64_t)head * D + h * 8;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      u32x4 t = *reinterpret_cast<const u32x4*>(qp + kk * 16);
      kv4_prepare_q(t, a.scale);
      qf[kk] = *reinterpret_cast<bf16x8*>(&t);
    }
  }
  f32x16 o[NB];
#pragma unroll
  for (int dt = 0; dt < NB; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  float m = -FLT_MAX, l = 0.f;
  int E = -1, first_out = INT32_MAX;                        // E: none yet
  const float sl = kv4_log2_scale(a.scale);

  u32x4 code[PPT];
  uint32_t scale[PPT], vtok = 0;                            // vtok: the V scales of token `lane`
  uint32_t c_off[PPT], s_off[PPT];                          // this thread's pieces: 32-bit offsets from the page's scalar base
#pragma unroll
  for (int i = 0; i < PPT; ++i) {
    const int pc = min(tid + i * NT, PIECES - 1), isv = pc >= PIECES / 2, j = pc % (PIECES / 2);
    c_off[i] = isv * BLK + j * 16;
    s_off[i] = isv * BLK + KV_PAGE * (D / 2) + j;
  }
  const uint32_t t_off = BLK + KV_PAGE * (D / 2) + lane * NB;
  auto fetch = [&](int page) {
    const int p = page >= 0 && page < a.c.n_pages ? page : 0;
    const uint8_t* blk = a.c.pool + ((int64_t)p * KVH + kvh) * 2 * BLK;
#pragma unroll
    for (int i = 0; i < PPT; ++i) {
      code[i] = *reinterpret_cast<const u32x4*>(blk + c_off[i]);
      scale[i] = blk[s_off[i]];
    }
    if constexpr (NB == 4) vtok = *reinterpret_cast<const uint32_t*>(blk + t_off);
    else if constexpr (NB == 2) vtok = *reinterpret_cast<const uint16_t*>(blk + t_off);
    else vtok = blk[t_off];
  };

  int pg = p_lo, page = pg < p_hi ? bt[pg] : -1, next_page = pg + 1 < p_hi ? bt[pg + 1] : -1;
  if (pg < p_hi) fetch(page);
  __syncthreads();                                          // s_nan
  int it = 0;
  // the pages from pg on, whose codes are in flight: in fp16 up to that of first_out, where the columns that see that key
  // see nothing; in bf16
  int p_end = p_hi;
  auto pages = [&](auto in_bf16) {
    constexpr bool BF = decltype(in_bf16)::value;
    for (; pg < p_end; ++pg, it ^= 1) {
      const bool there = page >= 0 && page < a.c.n_pages;
      const int tok_end = sp.cached - pg * KV_PAGE;           // tokens of the page at or past this are not the sequence's
      uint64_t hit = 0;
      if (there) {
        if constexpr (!BF) {
          if (E < 0) {
            const int first = __builtin_amdgcn_readfirstlane((int)vtok);
            E = 0;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
              const int b = (first >> (8 * i)) & 255;
              E = max(E, b == KV4_NAN_SCALE ? 0 : b);
            }
          }
          const uint32_t low = E - BELOW;
          bool out = false;
#pragma unroll
          for (int i = 0; i < NB; ++i) out |= ((vtok >> (8 * i)) & 255u) - low > BELOW + ABOVE;
          hit = __builtin_amdgcn_ballot_w64(out && lane < tok_end);
        }
        // ---- stage
#pragma unroll
        for (int i = 0; i < PPT; ++i) {
          const int pc = tid + i * NT, isv = pc >= PIECES / 2, j = pc % (PIECES / 2), key = j / NB, part = j % NB;
          if (PIECES % NT == 0 || pc < PIECES) {
            if (!isv) {
              const float ks = kv4_scale(scale[i]);
#pragma unroll
              for (int w = 0; w < 4; ++w)
                *reinterpret_cast<u32x4*>(&s_k[it][key * KROW + part * 64 + w * 16]) = kv4_unpack8(code[i][w], ks);
            } else {
              const bool use = key < tok_end, bad = use && scale[i] == KV4_NAN_SCALE;
              if (bad) atomicMin(&s_nan[part], pg * KV_PAGE + key);
              // (a masked block must not pass its scale on: 255 gives NaN even for 0; V that no column of the phase sees stays finite)
              const float vs = kv4_scale(!use || bad ? 127u : BF ? scale[i] : (uint32_t)min(max((int)scale[i] - E + 127, 96), 140));
              u32x4 cw = use && !bad ? code[i] : (u32x4){0, 0, 0, 0};
              const int turn = NB == 4 ? key & 3 : NB == 2 ? (key & 1) | ((key >> 1) & 2) : (key >> 2) & 3;
              if (turn & 1) cw = (u32x4){cw[1], cw[2], cw[3], cw[0]};
              if (turn & 2) cw = (u32x4){cw[2], cw[3], cw[0], cw[1]};
              unsigned char* vw = &s_v[it][key * VROW + part * 64];
#pragma unroll
              for (int w = 0; w < 4; ++w)
                *reinterpret_cast<u32x4*>(vw + ((w + turn) & 3) * 16) = BF ? kv4_unpack8(cw[w], vs) : kv4_unpack8_f16(cw[w], vs);
            }
          }
        }
      }
      if (__builtin_expect(hit != 0, 0)) {       // (asked here, the staging does not wait for it)
        first_out = pg * KV_PAGE + (int)__builtin_ctzll(hit);
        if (first_out < tile_any) {
          p_end = pg + 1;
          vis = seen > first_out ? 0 : seen;
          any_see = all_see > first_out ? 0 : any_see;
        }
      }
      __syncthreads();      // the page is staged; and every wave is done with the page before the previous one (same buffer)
      if (pg + 1 < p_end) fetch(next_page);
      if (there && pg * KV_PAGE < any_see) {
        // V^T fragments of 16 keys: lanes 4 r .. 4 r + 3 of a 16-lane group name row (key) r; lane i of the group gets dim i of
        // the 4 rows.  The first are requested before the scores, the others a product ahead.
        const unsigned char* vr = &s_v[it][(4 * h + ((lane & 15) >> 2)) * VROW + ((lane >> 4) & 1) * 32 + (lane & 3) * 8];
        auto read_v = [&](int st, bf16x8* f) {
#pragma unroll
          for (int dt = 0; dt < NB; ++dt) {
            const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vr + st * 16 * VROW + dt * 64));
            const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vr + (st * 16 + 8) * VROW + dt * 64));
            f[dt] = (bf16x8){v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
          }
        };
        bf16x8 vf[NB];
        // ---- scores
        f32x16 sacc[2];
        bf16x8 kf[2][D / 16];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            kf[kt][kk] = *reinterpret_cast<const bf16x8*>(&s_k[it][(kt * 32 + c) * KROW + h * 16 + kk * 32]);
#pragma unroll
        for (int i = 0; i < 16; ++i) sacc[0][i] = sacc[1][i] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) sacc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kt][kk], qf[kk], sacc[kt], 0, 0, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * (D / 16), 0);   // the reads first
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * (D / 16), 0);
        // ---- softmax: register i of tile kt is key kt * 32 + 8 (i / 4) + 4 h + i % 4 of column c
        const bool part = pg * KV_PAGE + KV_PAGE > all_see;
        const int lim = vis - pg * KV_PAGE - 4 * h;
        float mx = -INFINITY;
        if (part) {       // an unseen key's score is minus infinity whatever its K holds
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (!(kt * 32 + 8 * (i >> 2) + (i & 3) < lim)) sacc[kt][i] = -INFINITY;
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sacc[kt][i]);
        mx = max_swap32(mx);
        // weights are at most 2^TOP; the reference m moves when one would exceed that, DEFER beyond: O is seldom rescaled
        constexpr float MOST = BF ? 0.f : TOP;
        const float mn = fmaf(mx, sl, -m) > MOST ? kv4_reference(mx * sl, DEFER - MOST) : m, corr = __builtin_amdgcn_exp2f(m - mn);
        float ps = 0.f;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 16; ++i) sacc[kt][i] = __builtin_amdgcn_exp2f(fmaf(sacc[kt][i], sl, -mn));
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 16; ++i) ps += sacc[kt][i];
        l = l * corr + ps;
        m = mn;
        read_v(0, vf);
        if (__builtin_amdgcn_ballot_w64(corr != 1.f)) {
#pragma unroll
          for (int dt = 0; dt < NB; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[dt][i] *= corr;
        }
        // ---- O^T += V^T P, 16 keys per product: slots (h, 0..3) = keys 4 h .., slots (h, 4..7) = keys 8 + 4 h ..
        auto weights = [&](int st, int i) { return sacc[st >> 1][(st & 1) * 8 + i]; };
        u32x4 pf[4], pl[4];
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float t0 = weights(st, 2 * i), t1 = weights(st, 2 * i + 1);
            pf[st][i] = BF ? kv4_pk_bf16(t0, t1) : kv4_pk_f16(t0, t1);
            if constexpr (BF) pl[st][i] = kv4_pk_bf16(t0 - bf_lo(pf[st][i]), t1 - bf_hi(pf[st][i]));
          }
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          bf16x8 vn[NB];
          if (st < 3) read_v(st + 1, vn);
#pragma unroll
          for (int dt = 0; dt < NB; ++dt) {
            if constexpr (BF) {
              o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[dt], __builtin_bit_cast(bf16x8, pf[st]), o[dt], 0, 0, 0);
              o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[dt], __builtin_bit_cast(bf16x8, pl[st]), o[dt], 0, 0, 0);
            } else {
              o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, vf[dt]),
                                                             __builtin_bit_cast(f16x8_t, pf[st]), o[dt], 0, 0, 0);
            }
          }
#pragma unroll
          for (int dt = 0; dt < NB; ++dt) vf[dt] = vn[dt];
        }
      }
      page = next_page;
      next_page = pg + 2 < p_hi ? bt[pg + 2] : -1;
    }
  };
  const int any = any_see;
  pages(std::false_type{});
  // from here on weights of at most 1, and O in units of 1
  const float top = m + TOP, down = __builtin_amdgcn_exp2f(m - top);
  float unit = E >= 0 ? kv4_scale((uint32_t)max(E, KV4_MIN_SCALE)) * down : 1.f;
  m = top;
  l *= down;
  if (__builtin_expect(first_out < tile_any, 0)) {
#pragma unroll
    for (int dt = 0; dt < NB; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] *= unit;
    unit = 1.f;
    vis = seen > first_out ? seen : 0;
    any_see = any > first_out ? any : 0;
    all_see = all_see > first_out ? all_see : 0;
    --pg;
    p_end = p_hi;
    page = bt[pg];
    next_page = pg + 1 < p_hi ? bt[pg + 1] : -1;
    fetch(page);
    pages(std::true_type{});
  }

  l = sum_swap32(l);
  __syncthreads();        // s_nan is complete
  if (wcol + c >= cols) return;
  // lane (c, h): dims dt * 32 + 8 (i / 4) + 4 h + i % 4 of column c
  const int64_t idx = (int64_t)qrow * a.H + head;
  const float inv = nz > 1 ? 1.f : l != 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int dt = 0; dt < NB; ++dt) {
    const bool bad = s_nan[dt] < seen;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      f32x4 r;
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = bad ? __uint_as_float(0x7fc00000u) : o[dt][q * 4 + j] * inv * unit;
      const int d = dt * 32 + q * 8 + h * 4;
      if (nz == 1)
        *reinterpret_cast<uint2*>(a.out + qrow * a.out_stride + (int64_t)head * D + d) = make_uint2(kv4_pk_bf16(r[0], r[1]), kv4_pk_bf16(r[2], r[3]));
      else
        *reinterpret_cast<f32x4*>(kv4_part_o<D>(a, z, idx) + d) = r;
    }
  }
  if (nz > 1 && h == 0) {
    kv4_part_ml(a, z, idx)[0] = m;
    kv4_part_ml(a, z, idx)[1] = l;
  }
}

// joins the key ranges of a query row and head: D / 4 lanes per range, WPR waves (1, or 4 for more than 16 ranges) per row
// and head, the ranges dealt over the groups of D / 4 lanes and their sums joined in group order.  grid (rows and heads of
// the longest sequence, 4 / WPR to a work-group; n_seqs).  A group's first ranges are requested before the weights are
// known: the two loads of a range wait for each other no more than once.  2.4 to 3.4 us for 8 rows x 32 heads x 4 ranges, 3.8
// to 4.6 for 1 x 32 x 32: a launch and its latency.  Attention and merge over 1 x 40k keys, one wave / four: 16 ranges 23.1 / 23.3
// us, 24 20.9 / 19.7, 32 19.8 / 17.7, 64 25.3 / 19.3; 8 x 8k in 16 24.3 / 24.4, in 32 34.4 / 32.3.
template <int D, int WPR>
__global__ __launch_bounds__(256) void kv4_attn_merge_kernel(Kv4AttnArgs a) {
  constexpr int LN = D / 4, NG = 64 * WPR / LN, PRE = WPR == 1 ? 16 / NG : 4;
  static_assert(KV4_MAX_SPLITS == 256, "one thread per range below");
  __shared__ float s_w[4][64], s_red[4], s_sum[4];
  __shared__ f32x4 s_o[WPR == 1 ? 1 : NG][LN];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int tid = WPR == 1 ? lane : (int)threadIdx.x;
  const Kv4Span sp = kv4_span(a, blockIdx.y);
  const int item = WPR == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
  const int row = item / a.H, hd = item % a.H;
  if (row >= sp.nq) return;
  const int G = a.H / a.c.KVH, col0 = (row * G + hd % G) / a.tile_cols * a.tile_cols;
  const int nz = kv4_attn_ranges(a, kv4_tile_pages(sp, G, col0, a.tile_cols));
  if (nz == 1) return;
  const int64_t idx = (int64_t)(sp.row0 + row) * a.H + hd;
  const int gr = tid / LN, ln = tid % LN;
  const float mz = tid < nz ? kv4_part_ml(a, tid, idx)[0] : -FLT_MAX, lz = tid < nz ? kv4_part_ml(a, tid, idx)[1] : 0.f;
  f32x4 pre[PRE];
#pragma unroll
  for (int k = 0; k < PRE; ++k) pre[k] = *reinterpret_cast<const f32x4*>(kv4_part_o<D>(a, min(gr + k * NG, nz - 1), idx) + ln * 4);
  float M = wave_max(mz);
  if constexpr (WPR > 1) {
    if (lane == 0) s_red[wave] = M;
    __syncthreads();
    M = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  }
  const float w = __builtin_amdgcn_exp2f(mz - M);
  s_w[wave][lane] = w;
  float L = wave_sum(lz * w);
  if constexpr (WPR > 1) {
    if (lane == 0) s_sum[wave] = L;
    __syncthreads();
    L = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
  } else {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_wave_barrier();               // this wave's weights
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  }
  f32x4 O = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](int zz, f32x4 v) {
    const float wz = WPR == 1 ? s_w[wave][zz] : s_w[zz >> 6][zz & 63];
#pragma unroll
    for (int j = 0; j < 4; ++j) O[j] += v[j] * wz;
  };
#pragma unroll
  for (int k = 0; k < PRE; ++k)
    if (gr + k * NG < nz) add(gr + k * NG, pre[k]);
  for (int zz = gr + PRE * NG; zz < nz; zz += NG) add(zz, *reinterpret_cast<const f32x4*>(kv4_part_o<D>(a, zz, idx) + ln * 4));
  if constexpr (WPR > 1) {
    s_o[gr][ln] = O;
    __syncthreads();
    if (gr != 0) return;
    for (int k = 1; k < min(NG, nz); ++k) {
      const f32x4 v = s_o[k][ln];
#pragma unroll
      for (int j = 0; j < 4; ++j) O[j] += v[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (LN <= 8) O[j] += xor_lane_f<8>(O[j], lane);
      if constexpr (LN <= 16) O[j] = sum_swap16(O[j]);
      O[j] = sum_swap32(O[j]);
    }
    if (gr != 0) return;
  }
  float r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = L != 0.f ? O[j] / L : 0.f;
  *reinterpret_cast<uint2*>(a.out + (sp.row0 + row) * a.out_stride + (int64_t)hd * D + ln * 4) =
      make_uint2(kv4_pk_bf16(r[0], r[1]), kv4_pk_bf16(r[2], r[3]));
}

// Narrow tiles (16 columns, 8 waves along the keys) or wide ones (128 columns, 4 waves along the columns).  Both take any
// count; measured on 8 kv heads x 128 dims, 4 query heads each, narrow / wide in us, at 32, 64 and 128 columns:
// 1 x 4k keys 14 / 17, 15 / 19, 18 / 23; 8 x 4k 25 / 27, 32 / 34, 51 / 42; 32 x 4k 53 / 78, 94 / 94, 174 / 114.
constexpr int KV4_NARROW_COLS = 64, KV4_NARROW_TILE = 16, KV4_WIDE_TILE = 128;
static bool kv4_wide(int max_q, int H, int KVH) { return (int64_t)max_q * (H / KVH) > KV4_NARROW_COLS; }

// Enough work-groups to fill the 256 CUs, no more: a range costs its work-group's start and a partial state.
// Narrow: one work-group per CU (8 x 2k keys: 256 work-groups 12.0 us, 512 12.9); two where ranges of 32 pages remain, for
// sequences of different lengths (32 ragged x 8k: 54 us for 512, 60 for 256; 32 x 4k: 36 for 512, 32 for 256).  Equal shares of
// all pages instead, cut without regard to sequences, were slower throughout (32 ragged x 8k 60 us, 8 x 2k 19): a share
// that crosses a border pays a second start and merge.
// Wide: two fit a CU (8 x 4k keys at 128 columns: 49 us for 256 work-groups, 42 for 512, 52 for 1024), with ranges of at
// least 8 pages where more than 128 rows would write partial states (32 x 500 keys at 128 columns: 24 us in one range, 50 in
// two of 4 pages; 1 x 4k at 96 columns: 21 us in ranges of 4 pages, 26 in ranges of 8).
int kv4_attn_splits(int n_seqs, int max_q, int max_kv, int H, int KVH) {
  const bool wide = kv4_wide(max_q, H, KVH);
  const int tc = wide ? KV4_WIDE_TILE : KV4_NARROW_TILE, pages = max_kv / KV_PAGE + (max_kv % KV_PAGE != 0);
  if (pages < 20) return 1;      // the merge is a second launch, 3 us of the host's time: not for the last microsecond
  const int64_t tiles = std::max<int64_t>(1, (int64_t)n_seqs * KVH * (((int64_t)max_q * (H / KVH) + tc - 1) / tc));
  int64_t want = (wide ? 512 : 256) / tiles;
  if (!wide && tiles >= 128 && 512 / tiles * 32 <= pages) want = 512 / tiles;
  const int least = wide && (int64_t)n_seqs * max_q > 128 ? 8 : KV4_MIN_PAGES;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, pages / least), KV4_MAX_SPLITS));
}

int64_t kv4_attn_part_floats(int total_q, int H, int D, int splits) {
  const int64_t n = (int64_t)total_q * H * splits;
  return splits > 1 ? (n * 2 + 3) / 4 * 4 + n * D : 0;
}

int launch_kv4_attn(const Kv4AttnArgs& a_, hipStream_t s) {
  Kv4AttnArgs a = a_;
  const int D = a.c.D;
  FMI_REQUIRE(a.n_seqs >= 0 && a.n_seqs <= 65535 && a.total_q >= 0 && a.max_q >= 0 && a.max_kv >= 0,
              "kv4 attention: bad sizes (n_seqs %d, total_q %d, max_q %d, max_kv %d)", a.n_seqs, a.total_q, a.max_q, a.max_kv);
  if (a.n_seqs == 0 || a.total_q == 0 || a.max_q == 0) return FMI_OK;
  FMI_CHECK(kv4_check_cache(a.c));
  FMI_REQUIRE(a.H >= 1 && a.H <= (1 << 16) && a.H % a.c.KVH == 0, "kv4 attention: %d query heads over %d kv heads", a.H, a.c.KVH);
  FMI_REQUIRE(isfinite(a.scale), "kv4 attention: scale %g", (double)a.scale);
  FMI_CHECK(kv4_check_rows("q", a.q, a.q_stride, a.H, D));
  FMI_CHECK(kv4_check_rows("out", a.out, a.out_stride, a.H, D));
  FMI_REQUIRE(a.seq_slot || a.n_seqs <= a.c.n_slots, "kv4 attention: %d sequences, block table of %d", a.n_seqs, a.c.n_slots);
  FMI_REQUIRE(a.splits >= 1 && a.splits <= KV4_MAX_SPLITS && (a.splits == 1 || a.part), "kv4 attention: bad split of the keys");
  const int64_t cols = (int64_t)a.max_q * (a.H / a.c.KVH);
  const bool wide = a.wide || kv4_wide(a.max_q, a.H, a.c.KVH);
  a.tile_cols = wide ? KV4_WIDE_TILE : KV4_NARROW_TILE;
  const int64_t tiles = (cols + a.tile_cols - 1) / a.tile_cols;
  const int64_t merges = a.splits > 16 ? (int64_t)a.max_q * a.H : ((int64_t)a.max_q * a.H + 3) / 4;
  // (a grid dimension counts threads in 32 bits)
  FMI_REQUIRE((int64_t)a.max_q * a.H < (int64_t)1 << 31 && tiles * a.c.KVH < (int64_t)1 << 23 &&
                  (a.splits == 1 || merges < (int64_t)1 << 24), "kv4 attention: too many query rows per sequence (%d)", a.max_q);
  const dim3 grid((unsigned)(tiles * a.c.KVH), a.splits, a.n_seqs), mgrid((unsigned)merges, a.n_seqs);
#define FMI_KV4_ATTN(D_)                                                                                       \
  do {                                                                                                         \
    if (wide) hipLaunchKernelGGL((kv4_attn_wide_kernel<D_, KV4_WIDE_TILE / 32>), grid, dim3(2 * KV4_WIDE_TILE), 0, s, a); \
    else hipLaunchKernelGGL((kv4_attn_kernel<D_, 8, 0>), grid, dim3(512), 0, s, a, Kv4None{});                 \
    if (a.splits > 16) hipLaunchKernelGGL((kv4_attn_merge_kernel<D_, 4>), mgrid, dim3(256), 0, s, a);          \
    else if (a.splits > 1) hipLaunchKernelGGL((kv4_attn_merge_kernel<D_, 1>), mgrid, dim3(256), 0, s, a);      \
  } while (0)
  if (D == 128) FMI_KV4_ATTN(128);
  else if (D == 64) FMI_KV4_ATTN(64);
  else FMI_KV4_ATTN(32);
#undef FMI_KV4_ATTN
  FMI_CHECK_HIP(hipGetLastError());
  return FMI_OK;
}

int launch_kv4_step(const Kv4AppendArgs& p, const Kv4AttnArgs& a_, hipStream_t s) {
  Kv4AttnArgs a = a_;
  FMI_REQUIRE(p.rows >= 0 && p.rows <= 65535, "kv4 step: %d rows (0 to 65535)", p.rows);
  if (p.rows == 0) return FMI_OK;
  FMI_CHECK(kv4_check_append(p));
  FMI_REQUIRE(p.row_pos || p.slot_pos, "kv4 step: null row positions");
  const int D = p.c.D;
  FMI_REQUIRE(p.q && p.H % p.c.KVH == 0, "kv4 step: %d query heads over %d kv heads", p.H, p.c.KVH);
  FMI_CHECK(kv4_check_rows("out", a.out, a.out_stride, p.H, D));
  FMI_REQUIRE(isfinite(a.scale), "kv4 step: scale %g", (double)a.scale);
  FMI_REQUIRE(a.splits >= 1 && a.splits <= KV4_MAX_SPLITS && (a.splits == 1 || a.part), "kv4 step: bad split of the keys");
  a.c = p.c; a.H = p.H; a.seq_slot = p.row_seq; a.row_pos = p.row_pos; a.slot_pos = p.slot_pos;
  a.n_seqs = a.total_q = p.rows; a.max_q = 1; a.tile_cols = KV4_NARROW_TILE;
  a.step_len = p.rope ? std::min(p.c.max_pages * KV_PAGE, p.rope_len) : p.c.max_pages * KV_PAGE;
  const int tiles = (p.H / p.c.KVH + KV4_NARROW_TILE - 1) / KV4_NARROW_TILE, half = p.rope && p.half;
  const dim3 grid((unsigned)(tiles * p.c.KVH), a.splits, p.rows), mgrid((unsigned)(a.splits > 16 ? p.H : (p.H + 3) / 4), p.rows);
#define FMI_KV4_STEP(D_)                                                                                       \
  do {                                                                                                         \
    if (half) hipLaunchKernelGGL((kv4_attn_kernel<D_, 8, 2>), grid, dim3(512), 0, s, a, p);                    \
    else hipLaunchKernelGGL((kv4_attn_kernel<D_, 8, 1>), grid, dim3(512), 0, s, a, p);                         \
    if (a.splits > 16) hipLaunchKernelGGL((kv4_attn_merge_kernel<D_, 4>), mgrid, dim3(256), 0, s, a);          \
    else if (a.splits > 1) hipLaunchKernelGGL((kv4_attn_merge_kernel<D_, 1>), mgrid, dim3(256), 0, s, a);      \
  } while (0)
  if (D == 128) FMI_KV4_STEP(128);
  else if (D == 64) FMI_KV4_STEP(64);
  else FMI_KV4_STEP(32);
#undef FMI_KV4_STEP
  FMI_CHECK_HIP(hipGetLastError());
  return FMI_OK;
}

}  // namespace fmi

// ------------------------------------------------------------------------------------ C ABI

using namespace fmi;

static Kv4Cache kv4_cache_of(const fmi_kv4_cache& c) {
  return Kv4Cache{(uint8_t*)c.pool_dev, c.block_table_dev, c.n_pages, c.n_kv_head, c.head_dim, c.n_seqs, c.max_pages};
}

extern "C" {

int64_t fmi_kv4_page_bytes(int n_kv_head, int head_dim) {
  if (n_kv_head < 1 || (head_dim != 32 && head_dim != 64 && head_dim != 128))
    return set_error(FMI_EINVAL, "kv4: %d kv heads of %d dims (head_dim 32/64/128)", n_kv_head, head_dim);
  return (int64_t)n_kv_head * 2 * kv4_block_bytes(head_dim);
}

static Kv4AppendArgs kv4_append_args(const fmi_kv4_cache* cache, const fmi_kv4_rows* r) {
  Kv4AppendArgs a{};
  a.c = kv4_cache_of(*cache);
  a.q = (const bf16_t*)r->q_dev; a.k = (const bf16_t*)r->k_dev; a.v = (const bf16_t*)r->v_dev;
  a.q_stride = r->q_stride; a.k_stride = r->k_stride; a.v_stride = r->v_stride;
  a.q_out = (bf16_t*)r->q_out_dev; a.q_out_stride = r->q_out_stride; a.H = r->q_dev ? r->n_head : 0;
  a.q_norm = (const bf16_t*)r->q_norm_dev; a.k_norm = (const bf16_t*)r->k_norm_dev; a.eps = r->norm_eps;
  a.rope = (const bf16_t*)r->rope_dev; a.rope_len = r->rope_len; a.rot = r->rope_dim; a.half = r->rope_half != 0;
  a.row_seq = r->row_seq_dev; a.row_pos = r->row_pos_dev; a.rows = r->rows;
  return a;
}

int fmi_op_kv4_append(const fmi_kv4_cache* cache, const fmi_kv4_rows* r, void* stream) {
  FMI_REQUIRE(cache && r, "null argument");
  return launch_kv4_append(kv4_append_args(cache, r), (hipStream_t)stream);
}

int fmi_op_kv4_read(const fmi_kv4_cache* cache, const int32_t* row_seq_dev, const int32_t* row_pos_dev, int rows,
                    void* k_out_dev, void* v_out_dev, void* stream) {
  FMI_REQUIRE(cache, "null argument");
  FMI_REQUIRE(rows == 0 || (row_seq_dev && row_pos_dev), "kv4 read: null row indices");
  Kv4ReadArgs a{};
  a.c = kv4_cache_of(*cache);
  a.row_seq = row_seq_dev; a.row_pos = row_pos_dev; a.rows = rows; a.k = (bf16_t*)k_out_dev; a.v = (bf16_t*)v_out_dev;
  return launch_kv4_read(a, (hipStream_t)stream);
}

static int kv4_splits_of(const fmi_kv4_cache* cache, const fmi_kv4_query* q) {
  return q->splits > 0 ? q->splits : kv4_attn_splits(q->n_seqs, q->max_q, q->max_kv, q->n_head, cache->n_kv_head);
}

int64_t fmi_kv4_attention_ws_bytes(const fmi_kv4_cache* cache, const fmi_kv4_query* q) {
  if (!cache || !q || cache->n_kv_head < 1 || q->n_head < 1 || q->n_head > (1 << 16) || q->splits < 0 ||
      q->splits > KV4_MAX_SPLITS || q->total_q < 0 || q->max_q < 0 || q->n_seqs < 0 || q->max_kv < 0 ||
      (int64_t)q->total_q * q->n_head >= (int64_t)1 << 40)
    return set_error(FMI_EINVAL, "kv4 attention: bad sizes");
  return 4 * kv4_attn_part_floats(q->total_q, q->n_head, cache->head_dim, kv4_splits_of(cache, q));
}

int fmi_op_kv4_attention(const fmi_kv4_cache* cache, const fmi_kv4_query* q, void* out_dev, int64_t out_stride, void* ws_dev,
                         int64_t ws_bytes, void* stream) {
  FMI_REQUIRE(cache && q, "null argument");
  const int64_t need = fmi_kv4_attention_ws_bytes(cache, q);
  if (need < 0) return (int)need;
  Kv4AttnArgs a{};
  a.c = kv4_cache_of(*cache);
  a.q = (const bf16_t*)q->q_dev; a.out = (bf16_t*)out_dev; a.q_stride = q->q_stride; a.out_stride = out_stride;
  a.q_start = q->q_start_dev; a.kv_len = q->kv_len_dev; a.n_seqs = q->n_seqs; a.total_q = q->total_q; a.max_q = q->max_q;
  a.max_kv = q->max_kv; a.H = q->n_head; a.scale = q->scale; a.splits = kv4_splits_of(cache, q); a.part = (float*)ws_dev;
  FMI_REQUIRE(a.n_seqs == 0 || (a.q_start && a.kv_len), "kv4 attention: null q_start or kv_len");
  FMI_REQUIRE(ws_bytes >= need, "kv4 attention: workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
  FMI_REQUIRE(need == 0 || (ws_dev && ((uintptr_t)ws_dev & 15) == 0), "kv4 attention: null or misaligned workspace");
  return launch_kv4_attn(a, (hipStream_t)stream);
}

int fmi_op_kv4_step(const fmi_kv4_cache* cache, const fmi_kv4_rows* r, float scale, int max_kv, int splits, void* out_dev,
                    int64_t out_stride, void* ws_dev, int64_t ws_bytes, void* stream) {
  FMI_REQUIRE(cache && r, "null argument");
  const Kv4AppendArgs p = kv4_append_args(cache, r);
  FMI_REQUIRE(!p.q_out, "kv4 step: the rotated q is not written (q_out_dev must be null)");
  fmi_kv4_query q{};
  q.n_head = std::max(p.H, 1); q.n_seqs = q.total_q = p.rows; q.max_q = 1; q.max_kv = max_kv; q.splits = splits;
  const int64_t need = fmi_kv4_attention_ws_bytes(cache, &q);
  if (need < 0) return (int)need;
  FMI_REQUIRE(ws_bytes >= need, "kv4 step: workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
  FMI_REQUIRE(need == 0 || (ws_dev && ((uintptr_t)ws_dev & 15) == 0), "kv4 step: null or misaligned workspace");
  Kv4AttnArgs a{};
  a.out = (bf16_t*)out_dev; a.out_stride = out_stride; a.scale = scale; a.splits = kv4_splits_of(cache, &q); a.part = (float*)ws_dev;
  return launch_kv4_step(p, a, (hipStream_t)stream);
}

}  // extern "C"
