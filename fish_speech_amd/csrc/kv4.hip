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

// D / 8 lanes own one (row, head), 8 dims each; a wave takes 64 / (D / 8) consecutive rows of ONE head, so its code
// bytes are consecutive in the page.  Every rounding is fixed by the definition (sum of squares in fp64, reciprocal
// norm and both products rounded to fp32, value to bf16; rotation in fp32 without fused products, then bf16), so the
// stored codes do not depend on how the lanes are arranged.
template <int D>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4AppendArgs a) {
  constexpr int LPH = D / 8, RPW = 64 / LPH;
  const int lane = threadIdx.x & 63, sub = lane % LPH;
  const int heads = a.H + 2 * a.c.KVH;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int head = (int)(w % heads);
  const int64_t row64 = (w / heads) * RPW + lane / LPH;
  const bool in_rows = row64 < a.rows;
  const int row = in_rows ? (int)row64 : 0;
  const int seq = in_rows ? a.row_seq[row] : -1;
  const bool seq_ok = seq >= 0 && seq < a.c.n_slots;
  const int pos = seq_ok ? (a.row_pos ? a.row_pos[row] : a.slot_pos[seq]) : -1;
  const int64_t limit = (int64_t)a.c.max_pages * KV_PAGE;
  const bool valid = pos >= 0 && pos < limit && (!a.rope || pos < a.rope_len);

  const int kind = head < a.H ? 0 : head < a.H + a.c.KVH ? 1 : 2;   // q, k, v
  const int hh = kind == 0 ? head : kind == 1 ? head - a.H : head - a.H - a.c.KVH;
  const bf16_t* src = kind == 0 ? a.q + row * a.q_stride : kind == 1 ? a.k + row * a.k_stride : a.v + row * a.v_stride;
  src += (int64_t)hh * D;
  u32x4 x = *reinterpret_cast<const u32x4*>(src + sub * 8);

  if (kind != 2) {
    const bf16_t* nw = kind == 0 ? a.q_norm : a.k_norm;
    const bool rot = a.rope && sub * 8 < a.rot && valid;
    // half layout: the other element of each pair lies rot / 2 dims away, in another lane's chunk
    const int hr = a.rot / 2;
    const bool first = sub * 8 < hr;
    const int psub = rot && a.half ? (first ? sub + hr / 8 : sub - hr / 8) : sub;
    u32x4 xp = x;
    if (rot && a.half) xp = *reinterpret_cast<const u32x4*>(src + psub * 8);
    if (nw) {
      const u32x4 wv = *reinterpret_cast<const u32x4*>(nw + sub * 8), wp = *reinterpret_cast<const u32x4*>(nw + psub * 8);
      double ss = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double e0 = (double)bf_lo(x[i]), e1 = (double)bf_hi(x[i]);
        ss = fma(e0, e0, ss);
        ss = fma(e1, e1, ss);
      }
      ss += xor_lane_d<1>(ss, lane);
      ss += xor_lane_d<2>(ss, lane);
      if (LPH > 4) ss += xor_lane_d<4>(ss, lane);
      if (LPH > 8) ss += xor_lane_d<8>(ss, lane);
      const float rstd = kv4_rstd(ss / (double)D + a.eps);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = kv4_pk_bf16(__fmul_rn(__fmul_rn(bf_lo(x[i]), rstd), bf_lo(wv[i])),
                           __fmul_rn(__fmul_rn(bf_hi(x[i]), rstd), bf_hi(wv[i])));
        xp[i] = kv4_pk_bf16(__fmul_rn(__fmul_rn(bf_lo(xp[i]), rstd), bf_lo(wp[i])),
                            __fmul_rn(__fmul_rn(bf_hi(xp[i]), rstd), bf_hi(wp[i])));
      }
    }
    if (rot) {
      const bf16_t* tab = a.rope + (int64_t)pos * a.rot;
      if (!a.half) {
        const u32x4 cs = *reinterpret_cast<const u32x4*>(tab + sub * 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x0 = bf_lo(x[i]), x1 = bf_hi(x[i]), c = bf_lo(cs[i]), s = bf_hi(cs[i]);
          x[i] = kv4_pk_bf16(__fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s)), __fadd_rn(__fmul_rn(x1, c), __fmul_rn(x0, s)));
        }
      } else {
        const bf16_t* tp = tab + (first ? sub * 8 : sub * 8 - hr) * 2;
        const u32x4 c0 = *reinterpret_cast<const u32x4*>(tp), c1 = *reinterpret_cast<const u32x4*>(tp + 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t csa = i < 2 ? c0[2 * i] : c1[2 * i - 4], csb = i < 2 ? c0[2 * i + 1] : c1[2 * i - 3];
          float r[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float me = j ? bf_hi(x[i]) : bf_lo(x[i]), other = j ? bf_hi(xp[i]) : bf_lo(xp[i]);
            const float c = bf_lo(j ? csb : csa), s = bf_hi(j ? csb : csa);
            r[j] = first ? __fsub_rn(__fmul_rn(me, c), __fmul_rn(other, s)) : __fadd_rn(__fmul_rn(me, c), __fmul_rn(other, s));
          }
          x[i] = kv4_pk_bf16(r[0], r[1]);
        }
      }
    }
  }
  if (kind == 0) {
    if (valid) *reinterpret_cast<u32x4*>(a.q_out + row * a.q_out_stride + (int64_t)hh * D + sub * 8) = x;
    return;
  }
  // ---- quantise: 4 lanes hold a 32-dim block
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(x[i] & 0x7fffu, (x[i] >> 16) & 0x7fffu));
  top = max(top, (uint32_t)xor_lane<1>((int)top, lane));
  top = max(top, (uint32_t)xor_lane<2>((int)top, lane));
  const bool finite = top < 0x7f80u;
  // max = 1.f * 2^(exp - 127): the power with max <= 7 * 2^e is exp - 127 - 2, one more above f = 1.75
  const int b = min(max((int)(top >> 7) - 2 + ((top & 0x7fu) > 0x60u ? 1 : 0), KV4_MIN_SCALE), KV4_MAX_SCALE);
  const float sc = kv4_scale((uint32_t)b);
  uint32_t codes = 0;
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf16x2_t, (uint32_t)x[0]), sc, 0);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf16x2_t, (uint32_t)x[1]), sc, 1);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf16x2_t, (uint32_t)x[2]), sc, 2);
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf16x2_t, (uint32_t)x[3]), sc, 3);
  if (!valid || (a.slot_done && a.slot_done[seq])) return;
  const int page = a.c.block_table[(int64_t)seq * a.c.max_pages + pos / KV_PAGE];
  if (page < 0 || page >= a.c.n_pages) return;
  constexpr int BLK = kv4_block_bytes(D);
  const int tok = pos % KV_PAGE;
  uint8_t* blk = a.c.pool + (((int64_t)page * a.c.KVH + hh) * 2 + (kind - 1)) * BLK;
  *reinterpret_cast<uint32_t*>(blk + tok * (D / 2) + sub * 4) = finite ? codes : 0u;
  if ((sub & 3) == 0) blk[KV_PAGE * (D / 2) + tok * (D / 32) + sub / 4] = (uint8_t)(finite ? b : KV4_NAN_SCALE);
}

static int kv4_check_cache(const Kv4Cache& c) {
  FMI_REQUIRE(c.pool && c.block_table, "kv4: null pool or block table");
  FMI_REQUIRE(c.D == 32 || c.D == 64 || c.D == 128, "kv4: head_dim %d unsupported (32/64/128)", c.D);
  FMI_REQUIRE(c.KVH >= 1 && c.n_pages >= 1 && c.n_slots >= 1 && c.max_pages >= 1,
              "kv4: n_kv_head %d, n_pages %d, n_seqs %d and max_pages %d must be positive", c.KVH, c.n_pages, c.n_slots, c.max_pages);
  FMI_REQUIRE(c.max_pages <= (1 << 24), "kv4: max_pages %d exceeds 2^24", c.max_pages);
  FMI_REQUIRE(((uintptr_t)c.pool & 15) == 0 && ((uintptr_t)c.block_table & 3) == 0, "kv4: misaligned pool or block table");
  return FMI_OK;
}

static int kv4_check_rows(const char* what, const void* p, int64_t stride, int heads, int D) {
  FMI_REQUIRE(p, "kv4: %s is null", what);
  FMI_REQUIRE(((uintptr_t)p & 15) == 0 && stride % 8 == 0 && stride >= (int64_t)heads * D,
              "kv4: %s needs 16-byte aligned rows of %d x %d values (row stride %lld)", what, heads, D, (long long)stride);
  return FMI_OK;
}

int launch_kv4_append(const Kv4AppendArgs& a, hipStream_t s) {
  FMI_CHECK(kv4_check_cache(a.c));
  const int D = a.c.D;
  FMI_REQUIRE(a.rows >= 0, "kv4 append: negative row count");
  if (a.rows == 0) return FMI_OK;
  FMI_CHECK(kv4_check_rows("k", a.k, a.k_stride, a.c.KVH, D));
  FMI_CHECK(kv4_check_rows("v", a.v, a.v_stride, a.c.KVH, D));
  FMI_REQUIRE(a.row_seq && (a.row_pos || a.slot_pos), "kv4 append: null row indices");
  if (a.q) {
    FMI_REQUIRE(a.H >= 1, "kv4 append: q without query heads");
    FMI_CHECK(kv4_check_rows("q", a.q, a.q_stride, a.H, D));
    FMI_CHECK(kv4_check_rows("q_out", a.q_out, a.q_out_stride, a.H, D));
  } else {
    FMI_REQUIRE(a.H == 0 && !a.q_norm, "kv4 append: query heads or q_norm without q");
  }
  FMI_REQUIRE(((uintptr_t)a.q_norm & 15) == 0 && ((uintptr_t)a.k_norm & 15) == 0, "kv4 append: misaligned norm weight");
  if (a.rope) {
    FMI_REQUIRE(((uintptr_t)a.rope & 15) == 0 && a.rope_len >= 1, "kv4 append: empty or misaligned rotation table");
    FMI_REQUIRE(a.rot >= 16 && a.rot <= D && a.rot % 16 == 0, "kv4 append: %d rotated dims (a multiple of 16 up to head_dim %d)", a.rot, D);
  }
  const int rpw = 64 / (D / 8);
  const int64_t waves = ((int64_t)a.rows + rpw - 1) / rpw * (a.H + 2 * a.c.KVH);
  const int64_t blocks = (waves + 3) / 4;
  FMI_REQUIRE(blocks < (int64_t)1 << 31, "kv4 append: too many rows");
  if (D == 128) hipLaunchKernelGGL((kv4_append_kernel<128>), dim3((unsigned)blocks), dim3(256), 0, s, a);
  else if (D == 64) hipLaunchKernelGGL((kv4_append_kernel<64>), dim3((unsigned)blocks), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((kv4_append_kernel<32>), dim3((unsigned)blocks), dim3(256), 0, s, a);
  FMI_CHECK_HIP(hipGetLastError());
  return FMI_OK;
}

// =====================================================================================
// read-back
// =====================================================================================

// the append's arrangement: a wave takes 64 / (D / 8) rows of one head of K or V, a lane 8 dims
template <int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4ReadArgs a) {
  constexpr int LPH = D / 8, RPW = 64 / LPH, BLK = kv4_block_bytes(D);
  const int lane = threadIdx.x & 63, sub = lane % LPH;
  const int heads = 2 * a.c.KVH;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int head = (int)(w % heads), isv = head & 1, kh = head >> 1;
  const int64_t row = (w / heads) * RPW + lane / LPH;
  if (row >= a.rows) return;
  const int seq = a.row_seq ? a.row_seq[row] : a.seq0, pos = a.row_seq ? a.row_pos[row] : (int)row;
  u32x4 x = {0, 0, 0, 0};
  if (seq >= 0 && seq < a.c.n_slots && pos >= 0 && pos < (int64_t)a.c.max_pages * KV_PAGE) {
    const int page = a.c.block_table[(int64_t)seq * a.c.max_pages + pos / KV_PAGE];
    if (page >= 0 && page < a.c.n_pages) {
      const int tok = pos % KV_PAGE;
      const uint8_t* blk = a.c.pool + (((int64_t)page * a.c.KVH + kh) * 2 + isv) * BLK;
      const uint32_t codes = *reinterpret_cast<const uint32_t*>(blk + tok * (D / 2) + sub * 4);
      x = kv4_unpack8(codes, kv4_scale(blk[KV_PAGE * (D / 2) + tok * (D / 32) + sub / 4]));
    }
  }
  *reinterpret_cast<u32x4*>((isv ? a.v : a.k) + (row * a.c.KVH + kh) * D + sub * 8) = x;
}

int launch_kv4_read(const Kv4ReadArgs& a, hipStream_t s) {
  FMI_CHECK(kv4_check_cache(a.c));
  FMI_REQUIRE(a.rows >= 0, "kv4 read: negative row count");
  if (a.rows == 0) return FMI_OK;
  const int D = a.c.D;
  FMI_REQUIRE(!a.row_seq == !a.row_pos, "kv4 read: null row indices");
  FMI_CHECK(kv4_check_rows("k", a.k, (int64_t)a.c.KVH * D, a.c.KVH, D));
  FMI_CHECK(kv4_check_rows("v", a.v, (int64_t)a.c.KVH * D, a.c.KVH, D));
  const int rpw = 64 / (D / 8);
  const int64_t blocks = (((int64_t)a.rows + rpw - 1) / rpw * (2 * a.c.KVH) + 3) / 4;
  FMI_REQUIRE(blocks < (int64_t)1 << 31, "kv4 read: too many rows");
  if (D == 128) hipLaunchKernelGGL((kv4_read_kernel<128>), dim3((unsigned)blocks), dim3(256), 0, s, a);
  else if (D == 64) hipLaunchKernelGGL((kv4_read_kernel<64>), dim3((unsigned)blocks), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((kv4_read_kernel<32>), dim3((unsigned)blocks), dim3(256), 0, s, a);
  FMI_CHECK_HIP(hipGetLastError());
  return FMI_OK;
}

// =====================================================================================
// attention
// =====================================================================================
//
// out[row][head] = sum_key softmax_key(scale * q . k) v over the keys [0, pos(row)] of the row's sequence; a row
// without keys gives 0.  A work-group of 4 waves owns a tile of 16 query columns of one sequence and kv head -- column =
// (query row, head of the kv head's group), so K and V are read once for all of them -- and one of up to `splits` ranges
// of 32-key blocks; wave w takes blocks w, w + 4, ... of the range.  Per block:
//   scores   S^T = K Q^T, v_mfma_f32_16x16x32_bf16: lane (c, g) holds the D / 4 dims from g D / 4 of key c, which is one
//            consecutive piece of the page and one scale; Q is read in the same order, so no dim is moved;
//   softmax  fp32, online, per column; the probabilities stay in registers as the B operand of the next product, split
//            into bf16 high and low parts (two products: 16 significant bits of weight);
//   output   O^T += V^T P: V is unpacked to bf16 into the wave's LDS rows and read back transposed by
//            ds_read_b64_tr_b16 (4 keys of one dim per lane).
// The waves' (m, l, O) are merged through LDS in wave order; with splits > 1 the merged state goes to `part` and
// kv4_attn_merge_kernel joins the ranges in order.  Keys that a column may not see enter neither the maximum nor the
// sum nor, where their V is NaN, the product: such blocks are read as 0 and the columns that do see them are set to NaN
// at the end.
struct Kv4Span {       // one sequence's query rows and keys, clamped to what the buffers hold
  int slot, row0, nq, kv, cached;
};
__device__ inline Kv4Span kv4_span(const Kv4AttnArgs& a, int s) {
  Kv4Span r;
  r.slot = a.seq_slot ? a.seq_slot[s] : s;
  const int lo = a.q_start ? a.q_start[s] : s, hi = a.q_start ? a.q_start[s + 1] : s + 1;
  r.row0 = min(max(lo, 0), a.total_q);
  r.nq = min(max(min(hi, a.total_q) - r.row0, 0), a.max_q);
  r.kv = min(max(a.kv_len ? a.kv_len[s] : a.slot_pos[r.slot] + 1, 0), 1 << 30);
  r.cached = (int)min((int64_t)r.kv, (int64_t)a.c.max_pages * KV_PAGE);
  return r;
}

// the ranges a tile of nb key blocks really uses, at least 8 blocks (256 keys) each: a function of the tile alone.  One
// range: its work-group writes the output itself and the merge passes the tile's rows by.
__device__ inline int kv4_attn_ranges(int nb, int splits) { return max(1, min(splits, nb / 8)); }
// key blocks of 32 that the tile of 16 columns from col0 sees
__device__ inline int kv4_tile_blocks(const Kv4Span& sp, int G, int col0) {
  const int nk = min(sp.kv - sp.nq + min(col0 + 15, sp.nq * G - 1) / G + 1, sp.cached);
  return nk > 0 ? (nk + 31) / 32 : 0;
}

template <int D>
__global__ __launch_bounds__(256) void kv4_attn_kernel(Kv4AttnArgs a) {
  constexpr int KB = 32, NW = 4, BLK = kv4_block_bytes(D), NB = D / 32;
  constexpr int KS = D / 32;                     // k-steps of a score product
  constexpr int VROW = D * 2 + 32;               // bytes of a key's row in LDS: 32 more, so that the 4 rows a 16-lane
                                                 // group reads together lie in different banks
  constexpr int VL = D / 32, VP = 64 / VL;       // lanes per key and keys per pass of the V unpacking
  constexpr int VPASS = VP >= KB ? 1 : KB / VP;
  __shared__ __attribute__((aligned(16))) unsigned char s_v[NW][KB * VROW];
  __shared__ float s_m[NW][16], s_l[NW][16];
  __shared__ int s_nan[NW][NB];
  static_assert(KB * VROW >= 16 * D * 4, "the merge keeps a wave's 16 x D fp32 sums where its V rows were");

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int KVH = a.c.KVH, G = a.H / KVH;
  const int tile = blockIdx.x / KVH, kvh = blockIdx.x % KVH, z = blockIdx.y;
  const Kv4Span sp = kv4_span(a, blockIdx.z);
  const int cols = sp.nq * G, col0 = tile * 16;
  if (col0 >= cols) return;
  const int pos0 = sp.kv - sp.nq;                // position of the sequence's first query row (negative: sees nothing)
  const int col = min(col0 + c, cols - 1);
  const int qrow = sp.row0 + col / G, head = kvh * G + col % G, qpos = pos0 + col / G;
  const int vis = min(qpos + 1, sp.cached);      // keys [0, vis) are this column's
  const int nb = kv4_tile_blocks(sp, G, col0), nz = kv4_attn_ranges(nb, a.splits);
  if (z >= nz) return;
  const int b_lo = (int)((int64_t)z * nb / nz), b_hi = (int)((int64_t)(z + 1) * nb / nz);
  const int32_t* bt = a.c.block_table + (int64_t)sp.slot * a.c.max_pages;

  bf16x8 qf[KS];                                 // B operand: column c, dims g D / 4 + 8 kk ..
  {
    const bf16_t* qp = a.q + qrow * a.q_stride + (int64_t)head * D + g * (D / 4);
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) qf[kk] = *reinterpret_cast<const bf16x8*>(qp + kk * 8);
  }
  f32x4 o[D / 16];
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) o[dt] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float m = -FLT_MAX, l = 0.f;
  int nan_key[NB];                               // first key whose V block is NaN, per 32-dim block
#pragma unroll
  for (int i = 0; i < NB; ++i) nan_key[i] = INT32_MAX;
  const float sl = a.scale * 1.4426950408889634f;   // scores in units of log2
  unsigned char* sv = s_v[wave];

  for (int kb = b_lo + wave; kb < b_hi; kb += NW) {
    const int page = bt[(kb * KB) / KV_PAGE];
    if (page < 0 || page >= a.c.n_pages) continue;         // no page: its keys are masked
    const int tok0 = (kb * KB) % KV_PAGE;
    const uint8_t* kblk = a.c.pool + ((int64_t)page * KVH + kvh) * 2 * BLK;
    const uint8_t* vblk = kblk + BLK;
    // ---- scores
    f32x4 sacc[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int tok = tok0 + kt * 16 + c;
      const float ks = kv4_scale(kblk[KV_PAGE * (D / 2) + tok * NB + g * NB / 4]);
      uint32_t kw[KS];
      const uint8_t* kp = kblk + tok * (D / 2) + g * (D / 8);
      if (D == 128) *reinterpret_cast<u32x4*>(kw) = *reinterpret_cast<const u32x4*>(kp);
      else if (D == 64) *reinterpret_cast<uint2*>(kw) = *reinterpret_cast<const uint2*>(kp);
      else kw[0] = *reinterpret_cast<const uint32_t*>(kp);
      sacc[kt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        u32x4 kf = kv4_unpack8(kw[kk], ks);
        sacc[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<bf16x8*>(&kf), qf[kk], sacc[kt], 0, 0, 0);
      }
    }
    // ---- V -> bf16 rows in LDS; rows past the sequence's keys hold whatever was there before: read as 0
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_wave_barrier();             // the previous block's reads are done (same wave)
#pragma unroll
    for (int it = 0; it < VPASS; ++it) {
      const int key = it * VP + lane / VL, part = lane % VL;
      if (VP <= KB || key < KB) {
        const int tok = tok0 + key, kabs = kb * KB + key;
        u32x4 vw = *reinterpret_cast<const u32x4*>(vblk + tok * (D / 2) + part * 16);
        uint32_t b = vblk[KV_PAGE * (D / 2) + tok * NB + part];
        const bool use = kabs < sp.cached, bad = use && b == KV4_NAN_SCALE;
        if (__builtin_amdgcn_ballot_w64(bad)) {
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            const uint64_t hit = __builtin_amdgcn_ballot_w64(bad && part == i);
            if (hit) nan_key[i] = min(nan_key[i], kb * KB + it * VP + (int)__builtin_ctzll(hit) / VL);
          }
        }
        if (!use || bad) {
          vw = (u32x4){0, 0, 0, 0};
          b = 127;
        }
        const float vs = kv4_scale(b);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<u32x4*>(sv + key * VROW + part * 64 + i * 16) = kv4_unpack8(vw[i], vs);
      }
    }
    // ---- softmax: lane (c, g) holds keys kt * 16 + g * 4 + j of column c
    float t[8], mx = -FLT_MAX;
    bool see[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      see[i] = kb * KB + (i >> 2) * 16 + g * 4 + (i & 3) < vis;
      t[i] = sacc[i >> 2][i & 3] * sl;
      if (see[i]) mx = fmaxf(mx, t[i]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mn = fmaxf(m, mx), corr = __builtin_amdgcn_exp2f(m - mn);
    float ps = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[i] = see[i] ? __builtin_amdgcn_exp2f(t[i] - mn) : 0.f;
      ps += t[i];
    }
    ps += __shfl_xor(ps, 16, 64);
    ps += __shfl_xor(ps, 32, 64);
    l = l * corr + ps;
    m = mn;
    u32x4 ph, pl;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ph[i] = kv4_pk_bf16(t[2 * i], t[2 * i + 1]);
      pl[i] = kv4_pk_bf16(t[2 * i] - bf_lo(ph[i]), t[2 * i + 1] - bf_hi(ph[i]));
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_wave_barrier();             // this wave's V rows are complete
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    // ---- O^T += V^T P: lanes 4 r .. 4 r + 3 of a 16-lane group name row (key) r, lane i gets column (dim) i of the 4
    const unsigned char* vr = sv + (g * 4 + (c >> 2)) * VROW + (c & 3) * 8;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
      const s16x4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vr + dt * 32));
      const s16x4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vr + 16 * VROW + dt * 32));
      const bf16x8 vf = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
#pragma unroll
      for (int j = 0; j < 4; ++j) o[dt][j] *= corr;
      o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, *reinterpret_cast<bf16x8*>(&ph), o[dt], 0, 0, 0);
      o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, *reinterpret_cast<bf16x8*>(&pl), o[dt], 0, 0, 0);
    }
  }

  // ---- merge the four waves in wave order
  __syncthreads();
  float* s_o = reinterpret_cast<float*>(&s_v[0][0]);       // [NW][16][D]
  if (g == 0) {
    s_m[wave][c] = m;
    s_l[wave][c] = l;
  }
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < NB; ++i) s_nan[wave][i] = nan_key[i];
  float* so = s_o + wave * 16 * D;
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j) so[c * D + dt * 16 + g * 4 + j] = o[dt][j];
  __syncthreads();
  for (int i = tid; i < 16 * D; i += 256) {
    const int cc = i / D, d = i % D;
    if (col0 + cc >= cols) continue;
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
      O += s_o[(w * 16 + cc) * D + d] * wgt;
      bad = min(bad, s_nan[w][d / 32]);
    }
    const int v = min(pos0 + row + 1, sp.cached);
    if (bad < v) O = __uint_as_float(0x7fc00000u);
    const int64_t idx = (int64_t)(sp.row0 + row) * a.H + hd;
    if (nz == 1) {
      a.out[(sp.row0 + row) * a.out_stride + (int64_t)hd * D + d] = L != 0.f ? f2bf(O / L) : (bf16_t)0;
    } else {
      float* part = a.part + ((int64_t)z * a.total_q * a.H + idx) * (D + 2);
      part[2 + d] = O;
      if (d == 0) {
        part[0] = M;
        part[1] = L;
      }
    }
  }
}

// joins the key ranges of one query row and head, in range order.  grid (max_q * H / 2, n_seqs), a wave per (row, head)
template <int D>
__global__ __launch_bounds__(128) void kv4_attn_merge_kernel(Kv4AttnArgs a) {
  const int lane = threadIdx.x & 63;
  const Kv4Span sp = kv4_span(a, blockIdx.y);
  const int i = blockIdx.x * 2 + (threadIdx.x >> 6);
  const int row = i / a.H, hd = i % a.H;
  if (row >= sp.nq) return;
  const int G = a.H / a.c.KVH;
  const int nz = kv4_attn_ranges(kv4_tile_blocks(sp, G, (row * G + hd % G) & ~15), a.splits);
  if (nz == 1) return;
  const int64_t step = (int64_t)a.total_q * a.H * (D + 2);
  const float* part = a.part + ((int64_t)(sp.row0 + row) * a.H + hd) * (D + 2);
  float M = -FLT_MAX;
  for (int z = 0; z < nz; ++z) M = fmaxf(M, part[z * step]);
  float L = 0.f, O[D > 64 ? 2 : 1] = {};
  for (int z = 0; z < nz; ++z) {
    const float wgt = __builtin_amdgcn_exp2f(part[z * step] - M);
    L += part[z * step + 1] * wgt;
#pragma unroll
    for (int k = 0; k < (D > 64 ? 2 : 1); ++k)
      if (k * 64 + lane < D) O[k] += part[z * step + 2 + k * 64 + lane] * wgt;
  }
  bf16_t* out = a.out + (sp.row0 + row) * a.out_stride + (int64_t)hd * D;
#pragma unroll
  for (int k = 0; k < (D > 64 ? 2 : 1); ++k)
    if (k * 64 + lane < D) out[k * 64 + lane] = L != 0.f ? f2bf(O[k] / L) : (bf16_t)0;
}

int kv4_attn_splits(int n_seqs, int max_q, int max_kv, int H, int KVH) {
  const int64_t tiles = (int64_t)n_seqs * KVH * (((int64_t)max_q * (H / KVH) + 15) / 16);
  const int64_t want = (1024 + tiles - 1) / std::max<int64_t>(tiles, 1), most = std::max(1, max_kv / 256);
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 256));
}

int64_t kv4_attn_part_floats(int total_q, int H, int D, int splits) {
  return splits > 1 ? (int64_t)splits * total_q * H * (D + 2) : 0;
}

int launch_kv4_attn(const Kv4AttnArgs& a, hipStream_t s) {
  FMI_CHECK(kv4_check_cache(a.c));
  const int D = a.c.D;
  FMI_REQUIRE(a.H >= 1 && a.H % a.c.KVH == 0, "kv4 attention: %d query heads over %d kv heads", a.H, a.c.KVH);
  FMI_REQUIRE(a.n_seqs >= 0 && a.n_seqs <= 65535 && a.total_q >= 0 && a.max_q >= 0 && a.max_kv >= 0,
              "kv4 attention: bad sizes (n_seqs %d, total_q %d, max_q %d, max_kv %d)", a.n_seqs, a.total_q, a.max_q, a.max_kv);
  if (a.n_seqs == 0 || a.total_q == 0 || a.max_q == 0) return FMI_OK;
  FMI_CHECK(kv4_check_rows("q", a.q, a.q_stride, a.H, D));
  FMI_CHECK(kv4_check_rows("out", a.out, a.out_stride, a.H, D));
  FMI_REQUIRE(a.seq_slot || a.n_seqs <= a.c.n_slots, "kv4 attention: %d sequences, block table of %d", a.n_seqs, a.c.n_slots);
  FMI_REQUIRE(a.splits >= 1 && a.splits <= 256 && (a.splits == 1 || a.part), "kv4 attention: bad split of the keys");
  const int64_t tiles = ((int64_t)a.max_q * (a.H / a.c.KVH) + 15) / 16;
  FMI_REQUIRE(tiles * a.c.KVH < (int64_t)1 << 31 && (int64_t)a.max_q * a.H < (int64_t)1 << 31, "kv4 attention: too many query rows");
  const dim3 grid((unsigned)(tiles * a.c.KVH), a.splits, a.n_seqs), mgrid((unsigned)(((int64_t)a.max_q * a.H + 1) / 2), a.n_seqs);
#define FMI_KV4_ATTN(D_)                                                                        \
  do {                                                                                          \
    hipLaunchKernelGGL((kv4_attn_kernel<D_>), grid, dim3(256), 0, s, a);                        \
    if (a.splits > 1) hipLaunchKernelGGL((kv4_attn_merge_kernel<D_>), mgrid, dim3(128), 0, s, a); \
  } while (0)
  if (D == 128) FMI_KV4_ATTN(128);
  else if (D == 64) FMI_KV4_ATTN(64);
  else FMI_KV4_ATTN(32);
#undef FMI_KV4_ATTN
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

int fmi_op_kv4_append(const fmi_kv4_cache* cache, const fmi_kv4_rows* r, void* stream) {
  FMI_REQUIRE(cache && r, "null argument");
  Kv4AppendArgs a{};
  a.c = kv4_cache_of(*cache);
  a.q = (const bf16_t*)r->q_dev; a.k = (const bf16_t*)r->k_dev; a.v = (const bf16_t*)r->v_dev;
  a.q_stride = r->q_stride; a.k_stride = r->k_stride; a.v_stride = r->v_stride;
  a.q_out = (bf16_t*)r->q_out_dev; a.q_out_stride = r->q_out_stride; a.H = r->q_dev ? r->n_head : 0;
  a.q_norm = (const bf16_t*)r->q_norm_dev; a.k_norm = (const bf16_t*)r->k_norm_dev; a.eps = r->norm_eps;
  a.rope = (const bf16_t*)r->rope_dev; a.rope_len = r->rope_len; a.rot = r->rope_dim; a.half = r->rope_half != 0;
  a.row_seq = r->row_seq_dev; a.row_pos = r->row_pos_dev; a.rows = r->rows;
  FMI_REQUIRE(a.rows <= 0 || a.row_pos, "kv4 append: null row positions");
  return launch_kv4_append(a, (hipStream_t)stream);
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
  if (!cache || !q || cache->n_kv_head < 1 || q->n_head < 1 || q->splits < 0 || q->splits > 256 || q->total_q < 0 ||
      q->max_q < 0 || q->n_seqs < 0 || q->max_kv < 0)
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

}  // extern "C"
