// Backward pass of softmax attention for gfx950: dQ, dK and dV from Q, K, V,
// the output, its log-sum-exp and the output's gradient, with the
// probabilities recomputed from Q, K and the LSE.
//
//   S = c Q K^T,  P = exp(S - L),  delta_i = sum_d dO_id O_id - dL_i
//   dP = dO V^T,  dS = P o (dP - delta)
//   dV = P^T dO,  dK = c dS^T Q,  dQ = c dS K        (c = sm_scale)
//
// Two kinds of items, in one launch: a KV item owns 128 keys of a kv head and
// streams the query rows of all query heads of its group (S, dP, dV, dK: four
// products); a Q item owns 128 query rows and streams the keys (S, dP, dQ:
// three).  S and dP are computed twice so that every gradient is summed in the
// registers of the one block that owns it: no atomics, the same bits on every
// run, and the sum over a group's query heads costs nothing.  The Q items fill
// the tail that the KV items leave.
//
// Both kinds share one shape.  A wave holds 32 rows X of its own tensors
// (KV: K and V; Q: Q and dO) as MFMA B operands in registers; rows Y of the
// streamed tensors come 32 at a time through an LDS ring:
//   S[y][x]  = Y1 X1^T   (A operand: rows of Y1)
//   dP[y][x] = Y2 X2^T   (A operand: rows of Y2)
//   out1^T[d][x] += Y1^T dS,  out2^T[d][x] += Y2^T P  (A operand: columns of Y)
// The accumulator layout of S (lane = x, registers = y) is the B operand layout
// of the last two products when their inner index y is permuted alike on both
// sides, so P and dS never leave registers; the columns of Y are read with
// ds_read_b64_tr_b16 in just that order.
//
// Roundings: scores, probabilities, dP, delta and all sums are fp32; P and dS
// are rounded once to the input type as operands of the last two products.
// fp16 has too few exponents for that: P is scaled by 2^14 (as small as 1/n for
// n keys), and dS by a power of two from a bound on |dP - delta| of the kv head:
// the largest row norms of dO and of the V at hand, and the largest |delta|,
// which an output merged from other key ranges can make far larger than those.
// So neither overflows and only values 2^-28 below the largest lose bits; both
// come off the fp32 sums.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn_device.h"

namespace sage {
namespace {

constexpr int kBwdWaves = 4;
constexpr int kBwdThreads = kBwdWaves * 64;
constexpr int kOwnRows = kBwdWaves * 32;  // rows X of an item
constexpr int kStageRows = 32;            // streamed rows of a stage
constexpr int kKbPitch = 1088;            // LDS bytes per 1 KB load: 64 of padding shift the banks
constexpr int kStatBytes = 1024;          // row statistics of a stage (256 bytes, loaded four times over)
constexpr int kStatRows = 64;             // row statistics are padded to a multiple of these
constexpr float kF16PScale = 14.0f;       // log2 of the factor on P (fp16)
// A row all of whose keys are masked by a finite value has a finite LSE too.  P = exp(S - L) is off by some 2^-22 |L|
// of itself; below this LSE (whose last bit is a quarter) it would be 0 or infinite by chance, and the row counts as
// one without a live key.
constexpr float kDeadLse = -2097152.0f;

struct Rows {  // a [B,H,N,D] tensor: strides in elements
  const void* p;
  int64_t sb, sh, sn;
};

struct ItemOrder {
  int32_t items, head_items, xcds, group;  // group 0: heads one after the other
  FastDiv d_group;
};

struct BwdParams {
  Rows q, k, v, dout, dq, dk, dv;  // dq null: no Q items; dk and dv null: no KV items
  const float* stat;  // [B*Hq][stat_tiles][2][32]: -L log2 e (-inf: P = 0; fp16: + kF16PScale), -delta
  const float* omax;  // fp16: [B*Hq][omax_n][2]: largest row norm of dO, largest |delta|, of rows with a live key
  const float* vmax;  // fp16: [B*Hkv][vmax_n]: largest row norm of V
  float* part;        // fp32 partial sums of split items
  int64_t q_part;     // where the Q pieces start, in tiles of kOwnRows x D
  float sc, sm_scale; // sm_scale * log2 e
  int32_t hq, hkv, group, sq, sk, causal;
  int32_t stat_tiles, omax_n, vmax_n;
  // items of a head: its `long` longest tiles in `splits` pieces each, then the others whole
  int32_t kv_tiles, kv_long, kv_splits, q_tiles, q_long, q_splits;
  ItemOrder kv_order, q_order;
  FastDiv d_kvi, d_kvs, d_kvl, d_hkv, d_qi, d_qs, d_ql, d_hq, d_group;
};

template <int D>
struct BwdCfg {
  static constexpr int kRow = 2 * D;
  static constexpr int kKbRows = 1024 / kRow;        // rows of a 1 KB load
  static constexpr int kKb = kStageRows / kKbRows;   // loads of a tensor per stage
  static constexpr int kTensorBytes = kKb * kKbPitch;
  static constexpr int kStageBytes = 2 * kTensorBytes + kStatBytes;
  static constexpr int kSlots = D == 128 ? 2 : 3;
  static constexpr int kX2Bytes = kBwdWaves * 32 * kRow;  // KV: the own V operands
  static constexpr int kLdsBytes = kSlots * kStageBytes + kX2Bytes;
  static constexpr int kSteps = D / 16;
  static constexpr int kDB = D / 32;
  static constexpr int kWaves = D == 128 ? 2 : 3;    // per SIMD
};

template <int N>
__device__ __forceinline__ void bwd_wait_vm() {
  // lgkmcnt: this wave's reads of the slot that the barrier after this frees have returned
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

template <bool BF16>
__device__ __forceinline__ float16_t_ mfma16(int4_t a, int4_t b, float16_t_ c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

// v_mul_legacy_f32: a product that is 0 where either factor is, infinite and NaN ones included
__device__ float mul_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  return BF16 ? pack_bf16x2(a, b) : pack_f16x2(a, b);
}

// Consecutive items to blocks of one XCD, so that the tiles of a head stream
// their rows from one L2.  Causal items differ in length: the longest of all
// heads come first, where whole heads share out (`group` of them to an XCD)
// still with a head on one XCD.  Head after head / longest first, all launches
// of a causal pass, D128: B1 H24 S2048 115 / 100 us, S8192 1228 / 1207, H9
// S8192 (heads on all XCDs) 589 / 514, B1 H28 of 4 S4096 441 / 394.
__device__ __forceinline__ int item_of(int block, const ItemOrder& o) {
  if (o.group > 0) {
    const int xcd = o.xcds > 1 ? block % kXcds : 0, slot = o.xcds > 1 ? block / kXcds : block;
    const int i = div_by(slot, o.d_group);
    return (xcd * o.group + slot - i * o.group) * o.head_items + i;
  }
  const int per = o.items / kXcds, rem = o.items % kXcds;
  const int xcd = block % kXcds, slot = block / kXcds;
  return xcd * per + min(xcd, rem) + slot;
}

// fp16: log2 of the factor on dS for kv head `bhk`, from bounds over its query heads
__device__ __forceinline__ int ds_exponent(const BwdParams& p, int bhk, char* smem) {
  float om = 0.0f, lm = 0.0f, vm = 0.0f;
  const float* o = p.omax + static_cast<int64_t>(bhk) * p.group * p.omax_n * 2;
#pragma unroll 1
  for (int i = threadIdx.x; i < p.group * p.omax_n; i += kBwdThreads) {
    om = __builtin_fmaxf(om, o[2 * i]);
    lm = __builtin_fmaxf(lm, o[2 * i + 1]);
  }
  const float* v = p.vmax + static_cast<int64_t>(bhk) * p.vmax_n;
#pragma unroll 1
  for (int i = threadIdx.x; i < p.vmax_n; i += kBwdThreads) vm = __builtin_fmaxf(vm, v[i]);
  om = wave_max64(om), lm = wave_max64(lm), vm = wave_max64(vm);
  float* s = reinterpret_cast<float*>(smem);
  if ((threadIdx.x & 63) == 0) {
    s[3 * (threadIdx.x >> 6)] = om;
    s[3 * (threadIdx.x >> 6) + 1] = lm;
    s[3 * (threadIdx.x >> 6) + 2] = vm;
  }
  __syncthreads();
  for (int w = 0; w < kBwdWaves; ++w) {
    om = __builtin_fmaxf(om, s[3 * w]);
    lm = __builtin_fmaxf(lm, s[3 * w + 1]);
    vm = __builtin_fmaxf(vm, s[3 * w + 2]);
  }
  __syncthreads();
  const float bound = om * vm + lm;  // of |dP - delta|
  int e = 0;
  if (bound > 0.0f && bound < INFINITY) e = 1 - static_cast<int>((__float_as_uint(bound) >> 23) & 255) + 126;
  return __builtin_amdgcn_readfirstlane(min(max(e, -100), 100));
}

template <int D, bool BF16, bool CAP, bool KV>
__device__ __forceinline__ void bwd_item(const BwdParams& p, int item, char* smem) {
  using C = BwdCfg<D>;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int m = lane & 31, half = lane >> 5;

  // ---- the item: head, own rows, range of streamed stages
  const int tiles = KV ? p.kv_tiles : p.q_tiles, longs = KV ? p.kv_long : p.q_long;
  int splits = KV ? p.kv_splits : p.q_splits;
  const int bh = div_by(item, KV ? p.d_kvi : p.d_qi);  // (b, kv head) or (b, query head)
  int tile = item - bh * (tiles + longs * (splits - 1)), split = 0;  // tiles from the longest (causal) on
  if (tile < longs * splits) {
    const int r = tile;
    tile = div_by(r, KV ? p.d_kvs : p.d_qs);
    split = r - tile * splits;
  } else {
    tile -= longs * (splits - 1);
    splits = 1;
  }
  const int part_id = (bh * longs + tile) * splits + split;
  if (!KV) tile = p.q_tiles - 1 - tile;  // KV: the first tile is the longest, Q: the last
  const int b = div_by(bh, KV ? p.d_hkv : p.d_hq);
  const int h = bh - b * (KV ? p.hkv : p.hq);
  const int hk = KV ? h : div_by(h, p.d_group);
  const int own0 = tile * kOwnRows;
  const int own_n = KV ? p.sk : p.sq, str_n = KV ? p.sq : p.sk;
  const int stages = (str_n + kStageRows - 1) / kStageRows;
  int first = 0, last = stages;  // of one head
  if (p.causal) {
    if (KV) first = min(own0 / kStageRows, stages);
    else last = min(stages, (own0 + kOwnRows + kStageRows - 1) / kStageRows);
  }
  const int per_head = last - first;
  const int total = KV ? per_head * p.group : per_head;
  const int i0 = static_cast<int>(static_cast<int64_t>(total) * split / splits);
  const int i1 = static_cast<int>(static_cast<int64_t>(total) * (split + 1) / splits);
  const int n = i1 - i0;

  // ---- own rows as B operands: lane (m, half) holds elements 16 t + 8 half .. of row wrow0 + m
  constexpr bool kX2Lds = KV;  // V operands: registers for the accumulators
  const int wrow0 = own0 + 32 * wave, row = wrow0 + m;
  int4_t x1[C::kSteps], x2[kX2Lds ? 1 : C::kSteps];
  char* const x2_lds = smem + C::kSlots * C::kStageBytes + wave * 32 * C::kRow;
  {
    const Rows& r1 = KV ? p.k : p.q;
    const Rows& r2 = KV ? p.v : p.dout;
    const uint16_t* a = static_cast<const uint16_t*>(r1.p) + b * r1.sb + h * r1.sh + static_cast<int64_t>(row) * r1.sn + 8 * half;
    const uint16_t* c = static_cast<const uint16_t*>(r2.p) + b * r2.sb + h * r2.sh;
#pragma unroll
    for (int t = 0; t < C::kSteps; ++t) {
      x1[t] = int4_t{0, 0, 0, 0};
      if (row < own_n) x1[t] = *reinterpret_cast<const int4_t*>(a + 16 * t);
    }
    if constexpr (kX2Lds) {
      const uint32_t pitch = static_cast<uint32_t>(r2.sn * 2);
      const auto rx = make_rsrc(c, own_n > 0 ? static_cast<uint32_t>(own_n - 1) * pitch + C::kRow : 0);
#pragma unroll
      for (int t = 0; t < C::kSteps; ++t)
        lds_direct_load16(rx, x2_lds + t * 1024, static_cast<uint32_t>(row) * pitch + 16 * half + 32 * t, 0);
    } else {
#pragma unroll
      for (int t = 0; t < C::kSteps; ++t) {
        x2[t] = int4_t{0, 0, 0, 0};
        if (row < own_n) x2[t] = *reinterpret_cast<const int4_t*>(c + static_cast<int64_t>(row) * r2.sn + 8 * half + 16 * t);
      }
    }
  }
  float own_nl = 0.0f;  // Q: the own rows' statistics, -delta as the start of dP
  float16_t_ own_nd = {};
  if constexpr (!KV) {
    const bool in = wrow0 / 32 < p.stat_tiles;
    const float* st = p.stat + (static_cast<int64_t>(bh) * p.stat_tiles + wrow0 / 32) * 64;
    own_nl = in ? st[m] : -INFINITY;
    const float nd = in ? st[32 + m] : 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) own_nd[r] = nd;
  }
  float ds_scale = 1.0f;
  [[maybe_unused]] float max_x = BF16 ? 0.0f : kF16PScale;  // CAP: exponent of P = 1
  int ds_exp = 0;
  if constexpr (!BF16) {
    ds_exp = ds_exponent(p, b * p.hkv + hk, smem);
    ds_scale = __builtin_ldexpf(1.0f, ds_exp);
    if constexpr (!KV) {  // here P feeds dS alone, and takes its factor along
      own_nl += static_cast<float>(ds_exp);
      max_x += static_cast<float>(ds_exp);
    }
  }

  // ---- the stream.  Chunk c (16 bytes) of row r of a group of four rows lies at position 4 c + r of the group: a
  // transposing read (4 rows, 4 chunks) covers 256 contiguous bytes.  A row read takes one chunk of 16 rows a cycle, the
  // groups {0, 3, 5, 6} or {1, 2, 4, 7} of the 32 rows; with 64 bytes of padding per 1 KB load (one group at D = 128,
  // two at D = 64) those meet every bank once.  Steps along a row, along rows and between tensors are constants of
  // the instruction.
  const Rows& y1r = KV ? p.q : p.k;
  const Rows& y2r = KV ? p.dout : p.v;
  const uint32_t pitch1 = static_cast<uint32_t>(y1r.sn * 2), pitch2 = static_cast<uint32_t>(y2r.sn * 2);
  uint32_t voff1, voff2;
  {
    int r, c;
    if constexpr (D == 128) {
      r = lane & 3, c = lane >> 2;
    } else {
      r = 4 * half + (lane & 3), c = (lane & 31) >> 2;
    }
    voff1 = static_cast<uint32_t>(r) * pitch1 + 16 * c;
    voff2 = static_cast<uint32_t>(r) * pitch2 + 16 * c;
  }
  constexpr int kLoadsWave = C::kKb / kBwdWaves;  // of either tensor per stage; the first wave also the statistics
  // cursor of the loads: head of the group and stage
  const int g0 = KV && per_head > 0 ? i0 / per_head : 0;
  int lg = g0, ls = first + i0 - g0 * per_head;
  const int64_t y_head = KV ? hk * p.group : hk;
  const char* const y1_base = static_cast<const char*>(y1r.p) + 2 * (b * y1r.sb + y_head * y1r.sh);
  const char* const y2_base = static_cast<const char*>(y2r.p) + 2 * (b * y2r.sb + y_head * y2r.sh);
  const char* const st_base = reinterpret_cast<const char*>(p.stat) + (b * p.hq + y_head) * p.stat_tiles * 256;
  const uint32_t bytes1 = str_n > 0 ? static_cast<uint32_t>(str_n - 1) * pitch1 + C::kRow : 0;
  const uint32_t bytes2 = str_n > 0 ? static_cast<uint32_t>(str_n - 1) * pitch2 + C::kRow : 0;
  const uint32_t stat_bytes = static_cast<uint32_t>(p.stat_tiles) * 256;
  auto ry1 = make_rsrc(y1_base + 2 * lg * y1r.sh, bytes1);
  auto ry2 = make_rsrc(y2_base + 2 * lg * y2r.sh, bytes2);
  auto rst = make_rsrc(st_base + static_cast<int64_t>(lg) * stat_bytes, stat_bytes);
  auto issue = [&](int slot) __attribute__((always_inline)) {
    char* dst = smem + slot * C::kStageBytes;
#pragma unroll
    for (int x = 0; x < kLoadsWave; ++x) {
      const int kb = wave * kLoadsWave + x;
      const uint32_t r = static_cast<uint32_t>(ls * kStageRows + kb * C::kKbRows);
      lds_direct_load16(ry1, dst + kb * kKbPitch, voff1, r * pitch1);
      lds_direct_load16(ry2, dst + C::kTensorBytes + kb * kKbPitch, voff2, r * pitch2);
    }
    if (KV && wave == 0) lds_direct_load16(rst, dst + 2 * C::kTensorBytes, (lane % 16) * 16, ls * 256);
    ++ls;
    if (KV && ls == last) {
      ls = first;
      ++lg;
      if (lg < p.group) {
        ry1 = make_rsrc(y1_base + 2 * lg * y1r.sh, bytes1);
        ry2 = make_rsrc(y2_base + 2 * lg * y2r.sh, bytes2);
        rst = make_rsrc(st_base + static_cast<int64_t>(lg) * stat_bytes, stat_bytes);
      }
    }
  };

  // operand addresses
  const int row_base = (m >> 2) * (D == 128 ? kKbPitch : 512) + (D == 128 ? 0 : (m >> 3) * (kKbPitch - 1024)) + (m & 3) * 16 + half * 64;
  [[maybe_unused]] int tr_base;
  {
    const int g = lane >> 4, j = lane & 15, u = j >> 2, qd = j & 3;
    const int c = 2 * (g & 1) + (qd >> 1);
    tr_base = half * (D == 128 ? kKbPitch : 512) + (4 * c + u) * 16 + 8 * (qd & 1);
  }
  [[maybe_unused]] constexpr int kTr8 = D == 128 ? 2 * kKbPitch : kKbPitch;  // 8 rows further

  float16_t_ out1[C::kDB], out2[C::kDB];
#pragma unroll
  for (int db = 0; db < C::kDB; ++db) {
    out1[db] = float16_t_{};
    out2[db] = float16_t_{};
  }

  // One stage: the MFMAs in the order S, dP, [KV: dV,] dK or dQ, each step's A operand read kAhead steps before its use
  // and the softmax's pieces between them: exp2 of S under dP, dS under dV.  The order is kept as written.
  constexpr int kS = C::kSteps, kG = 2 * C::kDB;      // steps of a score product and of a gradient
  constexpr int kDv = 2 * kS, kDk = kDv + (KV ? kG : 0), kAll = kDk + kG;
  constexpr int kAhead = D == 128 ? (KV ? 4 : 6) : 4;
  // a softmax piece follows the step that it is spread to: from a step after the last MFMA of its input, to the step
  // before the first use of its half (registers 0-7, 8-15)
  constexpr int kExp = kS + 1, kDs = KV ? kDv + 1 : kDv;
  auto exp_step = [](int r) constexpr { return KV ? kExp + r * (kDv + C::kDB - kExp) / 16 : kExp + r * (kDv - kExp) / 16; };
  auto ds_step = [](int r) constexpr { return KV ? kDs + r * (kDk + C::kDB - kDs) / 16 : r < 8 ? -1 : kDv + (r - 8) * C::kDB / 8; };
  const float dead_s = __builtin_copysignf(INFINITY, -p.sc);
  auto run = [&](const char* st, int y0, bool masked) __attribute__((always_inline)) {
    const char* y1 = st;
    const char* y2 = st + C::kTensorBytes;
    const char* stats = st + 2 * C::kTensorBytes + 16 * half;
    auto operand = [&](int k) __attribute__((always_inline)) {
      if (k < kDv) return lds_read16((k < kS ? y1 : y2) + row_base + 128 * (k % kS));
#if defined(__HIP_DEVICE_COMPILE__)
      const int g = (k - kDv) % kG;
      const char* a = (k < kDk ? y2 : y1) + tr_base + 2 * kTr8 * (g / C::kDB) + 256 * (g % C::kDB);
      const uint2 lo = lds_read_tr(a), hi = lds_read_tr(a + kTr8);
      return int4_t{static_cast<int>(lo.x), static_cast<int>(lo.y), static_cast<int>(hi.x), static_cast<int>(hi.y)};
#else
      return int4_t{};
#endif
    };
    int4_t f[kAhead], v[2];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) f[k] = operand(k);
    float16_t_ s = {}, dp = own_nd;
    if constexpr (KV) {  // dP starts at -delta
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 d = __builtin_bit_cast(float4, lds_read16(stats + 128 + 32 * i));
        dp[4 * i] = d.x, dp[4 * i + 1] = d.y, dp[4 * i + 2] = d.z, dp[4 * i + 3] = d.w;
      }
    }
    // register r of a lane is streamed row y0 + 8 (r / 4) + 4 half + r % 4
    auto dead = [&](int r) __attribute__((always_inline)) {
      const int y = y0 + 8 * (r >> 2) + 4 * half + (r & 3);
      return KV ? y < row : y > min(p.causal ? row : INT32_MAX, p.sk - 1);
    };
    int4_t pw[2], dw[2];
    float nl[4];
    auto probability = [&](int r) __attribute__((always_inline)) {
      if constexpr (KV) {
        if (r % 4 == 0) {
          const float4 l4 = __builtin_bit_cast(float4, lds_read16(stats + 8 * r));
          nl[0] = l4.x, nl[1] = l4.y, nl[2] = l4.z, nl[3] = l4.w;
        }
      }
      float x = __builtin_fmaf(s[r], p.sc, KV ? nl[r % 4] : own_nl);
      if constexpr (CAP) x = __builtin_elementwise_minimum(x, max_x);  // (keeps NaN)
      s[r] = fast_exp2(x);
      if (KV && (r & 1)) pw[r / 8][r % 8 / 2] = static_cast<int>(pack16<BF16>(s[r - 1], s[r]));
    };
    auto gradient = [&](int r) __attribute__((always_inline)) {
      // 0 times infinity or NaN is 0 here: masked keys may hold anything
      dp[r] = mul_legacy(s[r], dp[r]);
      if constexpr (KV && !BF16) dp[r] *= ds_scale;
      if (r & 1) dw[r / 8][r % 8 / 2] = static_cast<int>(pack16<BF16>(dp[r - 1], dp[r]));
    };
    if constexpr (kX2Lds) v[0] = lds_read16(x2_lds + lane * 16);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < kAll; ++k) {
      // dead pairs: the S that gives P = 0 (and, by the multiplication, dS = 0 whatever dP is)
      if (k == kExp && masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = dead(r) ? dead_s : s[r];
      }
      if (!KV && k == kDv) {
#pragma unroll
        for (int r = 0; r < 8; ++r) gradient(r);
      }
      const int4_t a = f[k % kAhead];
      if (k < kS) {
        s = mfma16<BF16>(a, x1[k % kS], s);
      } else if (k < kDv) {
        if constexpr (kX2Lds) {
          if (k + 1 < kDv) v[(k + 1) % 2] = lds_read16(x2_lds + (k + 1 - kS) * 1024 + lane * 16);
          dp = mfma16<BF16>(a, v[k % 2], dp);
        } else {
          dp = mfma16<BF16>(a, x2[k % kS], dp);
        }
      } else if (k < kDk) {
        const int g = k - kDv;
        out2[g % C::kDB] = mfma16<BF16>(a, pw[g / C::kDB], out2[g % C::kDB]);
      } else {
        const int g = k - kDk;
        out1[g % C::kDB] = mfma16<BF16>(a, dw[g / C::kDB], out1[g % C::kDB]);
      }
      if (k + kAhead < kAll) f[k % kAhead] = operand(k + kAhead);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if (k == exp_step(r)) probability(r);
        if (k == ds_step(r)) gradient(r);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // streamed rows that this wave uses, and those where all of its pairs are live
  const int use0 = KV && p.causal ? wrow0 - 31 : INT32_MIN, use1 = !KV && p.causal ? wrow0 + 32 : INT32_MAX;
  const int live0 = KV && p.causal ? wrow0 + 31 : INT32_MIN;
  const int live1 = KV ? INT32_MAX : min(p.causal ? wrow0 : INT32_MAX, p.sk - 1) - 31;

  // ---- ring: wait for the stage's own loads, then the barrier says that all of it has landed and that the slot of
  // the stage before is free
  int cs = first + i0 - g0 * per_head;  // stage of the compute
  constexpr int kFly = C::kSlots - 1;  // stages loaded ahead of the wait: the last one is issued after the barrier
#pragma unroll
  for (int i = 0; i < kFly; ++i)
    if (i < n) issue(i);
  int slot = 0;
  for (int i = 0; i < n; ++i) {
    // loads of the stage after this one may stay in flight
    static_assert(kFly <= 2, "one later stage at most");
    constexpr int kV = 2 * kLoadsWave;
    if (kFly == 1 || i == n - 1) bwd_wait_vm<0>();
    else KV && wave == 0 ? bwd_wait_vm<kV + 1>() : bwd_wait_vm<kV>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");  // no LDS read of the stage moves above the barrier
    if (i + kFly < n) issue(slot == 0 ? C::kSlots - 1 : slot - 1);
    const int y0 = cs * kStageRows;
    if (y0 >= use0 && y0 < use1) {
      const char* st = smem + slot * C::kStageBytes;
      run(st, y0, y0 < live0 || y0 > live1);
    }
    if (++cs == last) cs = first;
    slot = slot == C::kSlots - 1 ? 0 : slot + 1;
  }

  // ---- results: lane (m, half) has elements 32 db + 8 (i / 4) + 4 half + i % 4 of its row
  float f1 = p.sm_scale, f2 = 1.0f;
  if constexpr (!BF16) {
    f1 = __builtin_ldexpf(f1, -ds_exp - static_cast<int>(kF16PScale));
    f2 = __builtin_ldexpf(1.0f, -static_cast<int>(kF16PScale));
  }
  if (splits > 1) {
    // [piece][own row][D] (KV: dK rows, then dV rows); Q pieces after the KV pieces
    float* part = p.part + (KV ? static_cast<int64_t>(part_id) * 2 : p.q_part + part_id) * kOwnRows * D +
                  (32 * wave + m) * D + 4 * half;
    if (row < own_n) {
#pragma unroll
      for (int db = 0; db < C::kDB; ++db) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          *reinterpret_cast<float4*>(part + 32 * db + 8 * i) =
              make_float4(out1[db][4 * i] * f1, out1[db][4 * i + 1] * f1, out1[db][4 * i + 2] * f1, out1[db][4 * i + 3] * f1);
          if constexpr (KV)
            *reinterpret_cast<float4*>(part + kOwnRows * D + 32 * db + 8 * i) =
                make_float4(out2[db][4 * i] * f2, out2[db][4 * i + 1] * f2, out2[db][4 * i + 2] * f2, out2[db][4 * i + 3] * f2);
        }
      }
    }
    return;
  }
  auto store = [&](const Rows& r, const float16_t_(&acc)[C::kDB], float f) __attribute__((always_inline)) {
    if (r.p == nullptr) return;
    uint16_t* o = static_cast<uint16_t*>(const_cast<void*>(r.p)) + b * r.sb + h * r.sh + static_cast<int64_t>(row) * r.sn;
#pragma unroll
    for (int db = 0; db < C::kDB; ++db) {
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        uint32_t w[2][2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          w[x][0] = pack16<BF16>(acc[db][4 * (i + x)] * f, acc[db][4 * (i + x) + 1] * f);
          w[x][1] = pack16<BF16>(acc[db][4 * (i + x) + 2] * f, acc[db][4 * (i + x) + 3] * f);
        }
        // halves exchange 8 bytes, so that each lane has 16 contiguous ones
        const auto a = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
        const auto c = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
        if (row < own_n) *reinterpret_cast<uint4*>(o + 32 * db + 8 * (i + half)) = make_uint4(a[0], c[0], a[1], c[1]);
      }
    }
  };
  if constexpr (KV) {
    store(p.dk, out1, f1);
    store(p.dv, out2, f2);
  } else {
    store(p.dq, out1, f1);
  }
}

// CAP: the LSE is not the one of these scores (the INT8 path's, whose scores are
// quantised), and P = exp(S - L) can come out above 1 without a bound; it counts
// as 1.  (The direct kernel's own LSE needs no such limit: an instruction a
// score, 1-2% of a launch at D = 128, 3-4% at 64.)
template <int D, bool BF16, bool CAP>
__global__ __launch_bounds__(kBwdThreads, BwdCfg<D>::kWaves) void attn_bwd_kernel(BwdParams p) {
  __shared__ __align__(16) char smem[BwdCfg<D>::kLdsBytes];
  const int block = static_cast<int>(blockIdx.x);
  if (block < p.kv_order.items) bwd_item<D, BF16, CAP, true>(p, item_of(block, p.kv_order), smem);
  else bwd_item<D, BF16, CAP, false>(p, item_of(block - p.kv_order.items, p.q_order), smem);
}

// Row statistics: -L log2 e and -delta of kStatRows query rows a block (rows
// past the last: P = 0), and for fp16 the largest row norms of dO and V and the
// largest |delta|, which bound dS (rows that are not finite left out: their own
// results are not either; and rows without a live key: they have no dS).  HBM-bound: reads O and dO (fp16: and V) once.
//
// O's rounding makes an error in delta that weighs like 1 / n in the dS of a row
// of n keys (n = 1: dS is 0, and that error all that is left).  Rows of up to
// kExactKeys keys take delta as the sum of P o dP instead, from two products of
// one wave, where their P sum to 1 and, with a given LSE, both deltas agree
// within half of the forward call's roundings (P to fp16, O to its type; a sum
// over D elements stays well below them): an output merged from several key
// ranges keeps dO O, since what its other keys add is not in the sum, however
// small their P, and so does a quantised forward call.  2-norm error of dQ over
// that of one rounding, without / with: causal B1 H8 S64 1.59 / 1.43, S2048 1.50
// / 1.44, two keys 2.3 / 1.4; 2 to 4 us of a launch that has such rows.
constexpr int kPreRows = kStatRows;
constexpr int kExactKeys = 32;  // of an MFMA

struct PreParams {
  Rows out, dout, v, q, k;
  float sc;
  int32_t causal, own_lse;  // own_lse: these are all of the rows' keys
  FastDiv d_group;
  const float* lse;
  const float* dlse;  // or null
  float* stat;
  float* omax;
  float* vmax;
  int32_t hq, hkv, sq, sk, stat_tiles, q_blocks, q_total, v_blocks, heads, v_heads;
  FastDiv d_hq, d_hkv, d_heads, d_vheads;
};

// Sums of P, P o dP and (unless own_lse) P o |dO| |V|^T of 32 rows over the first 32 keys, one wave: out[row] for the
// rows row0 + 0 .. 31.
template <int D, bool BF16>
__device__ __forceinline__ void exact_sums(const PreParams& p, int b, int h, int64_t bh, int row0, float (*out)[3]) {
  const int lane = threadIdx.x & 63, m = lane & 31, half = lane >> 5;
  const int row = row0 + m, hk = div_by(h, p.d_group);
  const bool in = row < p.sq, key_in = m < p.sk;
  auto at = [&](const Rows& r, int head, int i) {
    return reinterpret_cast<const int4_t*>(static_cast<const uint16_t*>(r.p) + b * r.sb + head * r.sh + i * r.sn + 8 * half);
  };
  const float l = in ? p.lse[bh * p.sq + row] : -INFINITY;
  const float nl = l < kDeadLse ? -INFINITY : l * -1.4426950408889634f;
  float16_t_ s = {}, dp = {}, size = {};
#pragma unroll
  for (int t = 0; t < D / 16; ++t) {
    int4_t x1 = {0, 0, 0, 0}, x2 = x1, y1 = x1, y2 = x1;
    if (in) x1 = at(p.q, h, row)[2 * t], x2 = at(p.dout, h, row)[2 * t];
    if (key_in) y1 = at(p.k, hk, m)[2 * t], y2 = at(p.v, hk, m)[2 * t];
    s = mfma16<BF16>(y1, x1, s);
    dp = mfma16<BF16>(y2, x2, dp);
    if (!p.own_lse) size = mfma16<BF16>(y2 & 0x7fff7fff, x2 & 0x7fff7fff, size);
  }
  float sum_p = 0.0f, sum = 0.0f, sum_size = 0.0f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {  // lane (m, half): row m, keys 8 (r / 4) + 4 half + r % 4
    const int key = 8 * (r >> 2) + 4 * half + (r & 3);
    const bool dead = key >= p.sk || (p.causal && key > row);
    const float pr = dead ? 0.0f : fast_exp2(__builtin_fmaf(s[r], p.sc, nl));
    sum_p += pr;
    sum += mul_legacy(pr, dp[r]);
    sum_size += mul_legacy(pr, size[r]);
  }
  sum_p = xhalf_sum(sum_p);
  sum = xhalf_sum(sum);
  sum_size = xhalf_sum(sum_size);
  if (half == 0) out[m][0] = sum_p, out[m][1] = sum, out[m][2] = sum_size;
}

template <int D, bool BF16, bool FEW>
__global__ __launch_bounds__(256) void attn_bwd_rows_kernel(PreParams p) {
  constexpr int kLanes = D / 8, kRowsPass = 256 / kLanes, kPasses = kPreRows / kRowsPass;
  __shared__ float red[2][4];
  [[maybe_unused]] __shared__ float exact[FEW ? kPreRows : 1][3];
  const int c = threadIdx.x % kLanes, r0 = threadIdx.x / kLanes;
  const bool is_v = static_cast<int>(blockIdx.x) >= p.q_total;
  // query blocks: the first of every head, then the second, ...: those with few keys take longest
  int id = is_v ? blockIdx.x - p.q_total : blockIdx.x;
  const int blk = div_by(id, is_v ? p.d_vheads : p.d_heads);
  const int bh = id - blk * (is_v ? p.v_heads : p.heads);
  id = bh * (is_v ? p.v_blocks : p.q_blocks) + blk;
  const int b = div_by(bh, is_v ? p.d_hkv : p.d_hq);
  const int h = bh - b * (is_v ? p.hkv : p.hq);
  const int n = is_v ? p.sk : p.sq;
  const Rows& ra = is_v ? p.v : p.dout;
  const uint16_t* pa = static_cast<const uint16_t*>(ra.p) + b * ra.sb + h * ra.sh + 8 * c;
  const uint16_t* po = static_cast<const uint16_t*>(p.out.p) + b * p.out.sb + h * p.out.sh + 8 * c;
  uint4 wa[kPasses], wo[kPasses];
  float wl[kPasses], wd[kPasses];  // LSE and its gradient
#pragma unroll
  for (int x = 0; x < kPasses; ++x) {
    const int row = blk * kPreRows + x * kRowsPass + r0;
    wa[x] = wo[x] = make_uint4(0, 0, 0, 0);
    wl[x] = wd[x] = 0.0f;
    if (row < n) {
      wa[x] = *reinterpret_cast<const uint4*>(pa + row * ra.sn);
      if (!is_v) {
        wo[x] = *reinterpret_cast<const uint4*>(po + row * p.out.sn);
        wl[x] = p.lse[static_cast<int64_t>(bh) * n + row];
        if (p.dlse != nullptr) wd[x] = p.dlse[static_cast<int64_t>(bh) * n + row];
      }
    }
  }
  const bool all = p.sk <= kExactKeys, few = FEW && !is_v && (all || blk == 0);  // causal: the first 32 rows
  if (few) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (w < (all ? kPreRows / 32 : 1)) exact_sums<D, BF16>(p, b, h, bh, blk * kPreRows + 32 * w, exact + 32 * w);
    __syncthreads();
  }
  float norm = 0.0f, lmax = 0.0f;
#pragma unroll
  for (int x = 0; x < kPasses; ++x) {
    const int row = blk * kPreRows + x * kRowsPass + r0;
    const uint32_t a4[4] = {wa[x].x, wa[x].y, wa[x].z, wa[x].w}, o4[4] = {wo[x].x, wo[x].y, wo[x].z, wo[x].w};
    float dot = 0.0f, sq = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2_t a = unpack2<BF16>(a4[i]), o = unpack2<BF16>(o4[i]);
      dot = __builtin_fmaf(a.x, o.x, __builtin_fmaf(a.y, o.y, dot));
      sq = __builtin_fmaf(a.x, a.x, __builtin_fmaf(a.y, a.y, sq));
    }
#pragma unroll
    for (int s = 1; s < kLanes; s *= 2) {
      dot += __shfl_xor(dot, s);
      if constexpr (!BF16) sq += __shfl_xor(sq, s);
    }
    if (few && (all || x * kRowsPass + r0 < 32)) {
      const float(&e)[3] = exact[x * kRowsPass + r0];
      constexpr float kRounding = 0x1p-11f + (BF16 ? 0x1p-9f : 0x1p-11f);  // of the forward call, times e[2]
      const bool whole = p.own_lse || __builtin_fabsf(e[1] - dot) <= 0.5f * kRounding * e[2];
      if (whole && __builtin_fabsf(e[0] - 1.0f) <= 0x1p-14f) dot = e[1];
    }
    // a row without a live key: P = 0 everywhere, and its (arbitrary) delta must not meet it as NaN
    const bool live = is_v || (row < n && !(wl[x] < kDeadLse));
    if (!is_v && c == 0) {
      const int tile = row / 32;
      float nl = -INFINITY, nd = 0.0f;
      if (live) {
        nl = wl[x] * -1.4426950408889634f + (BF16 ? 0.0f : kF16PScale);
        nd = wd[x] - dot;
        if (__builtin_fabsf(nd) < INFINITY) lmax = __builtin_fmaxf(lmax, __builtin_fabsf(nd));
      }
      float* st = p.stat + (static_cast<int64_t>(bh) * p.stat_tiles + tile) * 64 + row % 32;
      st[0] = nl;
      st[32] = nd;
    }
    if (live && sq < INFINITY) norm = __builtin_fmaxf(norm, sq);
  }
  if constexpr (!BF16) {
    norm = wave_max64(norm);
    lmax = wave_max64(lmax);
    if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = norm, red[1][threadIdx.x >> 6] = lmax;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 4; ++w) norm = __builtin_fmaxf(norm, red[0][w]), lmax = __builtin_fmaxf(lmax, red[1][w]);
      norm = __builtin_sqrtf(norm) * 1.001f;  // not below the true one
      if (is_v) {
        p.vmax[id] = norm;
      } else {
        p.omax[2 * id] = norm;
        p.omax[2 * id + 1] = lmax;
      }
    }
  }
}

// Sum of split items' partial results, in split order.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void attn_bwd_sum_kernel(BwdParams p, int kv_rows, int rows) {
  const int c = threadIdx.x % (D / 8);
  const int id = blockIdx.x * (256 / (D / 8)) + threadIdx.x / (D / 8);  // padded own row: dK, dV, then dQ
  if (id >= rows) return;
  const bool kv = id < kv_rows;
  int rest = kv ? id : id - kv_rows, which = 0;
  const int half_rows = kv_rows / 2;
  if (kv && rest >= half_rows) rest -= half_rows, which = 1;
  const int tile_id = rest / kOwnRows, r = rest % kOwnRows;  // (head, one of its split tiles)
  const int splits = kv ? p.kv_splits : p.q_splits;
  const int bh = div_by(tile_id, kv ? p.d_kvl : p.d_ql);
  int tile = tile_id - bh * (kv ? p.kv_long : p.q_long);
  if (!kv) tile = p.q_tiles - 1 - tile;
  const int row = tile * kOwnRows + r;
  if (row >= (kv ? p.sk : p.sq)) return;
  const Rows& out = kv ? (which ? p.dv : p.dk) : p.dq;
  if (out.p == nullptr) return;
  const int b = div_by(bh, kv ? p.d_hkv : p.d_hq);
  const int h = bh - b * (kv ? p.hkv : p.hq);
  const int64_t step = static_cast<int64_t>(kv ? 2 : 1) * kOwnRows * D;  // between splits
  const float* src = p.part + (kv ? 0 : p.q_part) * kOwnRows * D + tile_id * splits * step + which * kOwnRows * D + r * D + 8 * c;
  float a[8] = {};
  for (int s = 0; s < splits; s += 4, src += 4 * step) {
    float4 u[4], w[4];  // four splits' loads in flight; those past the last add 0
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      u[k] = w[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (s + k < splits) {
        u[k] = *reinterpret_cast<const float4*>(src + k * step);
        w[k] = *reinterpret_cast<const float4*>(src + k * step + 4);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      a[0] += u[k].x, a[1] += u[k].y, a[2] += u[k].z, a[3] += u[k].w;
      a[4] += w[k].x, a[5] += w[k].y, a[6] += w[k].z, a[7] += w[k].w;
    }
  }
  uint16_t* o = static_cast<uint16_t*>(const_cast<void*>(out.p)) + b * out.sb + h * out.sh + row * out.sn + 8 * c;
  *reinterpret_cast<uint4*>(o) = make_uint4(pack16<BF16>(a[0], a[1]), pack16<BF16>(a[2], a[3]),
                                            pack16<BF16>(a[4], a[5]), pack16<BF16>(a[6], a[7]));
}

struct BwdPlan {
  int64_t kv_tiles, kv_long, kv_splits, kv_items, q_tiles, q_long, q_splits, q_items, stat_tiles, v_blocks;
  int64_t kv_pieces, q_pieces;  // with partial sums
  int64_t stat_off, omax_off, vmax_off, part_off, bytes;  // of the workspace
};

// Tiles, splits of the streamed range, and the workspace's layout.
//
// An item alone on its CU takes kItemKv / kItemQ us a stage (32 rows), a full
// CU one stage of an item each kCuKv / kCuQ us, and kFixed us go to an item's
// start and end; while every CU has other items too, an item takes kShared
// times as long.  The launch ends when the longest item does or when the work
// is done; partial sums cost kSum us and their bytes at kSumRate once (written
// and read).  Splits are the cheapest of a few counts by that model.  Measured
// on MI355X, all launches of a pass, unsplit / as split: B1 H16 Sq4096 Sk512
// D128 130 / 81 us, B2 H10 Sq4096 Sk77 D64 95 / 36, B2 Hq32 Hkv8 S2048 D128
// causal 304 / 254; and left unsplit / in two: B1 H8 S1024 D128 38 / 42, B1 H12
// S2393 D128 127 / 151.
BwdPlan bwd_plan(bool bf16, int64_t batch, int64_t hq, int64_t hkv, int64_t sq, int64_t sk, int64_t d, bool causal,
                 bool need_q, bool need_kv) {
  BwdPlan f;
  f.kv_tiles = cdiv(sk, kOwnRows);
  f.q_tiles = cdiv(sq, kOwnRows);
  const int64_t kv = need_kv ? batch * hkv * f.kv_tiles : 0, q = need_q ? batch * hq * f.q_tiles : 0;
  const int64_t kv_len = hq / hkv * cdiv(sq, kStageRows), q_len = cdiv(sk, kStageRows);
  const double item_kv = d == 128 ? 0.83 : 0.62, item_q = d == 128 ? 0.62 : 0.45;
  const double cu_kv = d == 128 ? 0.94 : 0.51, cu_q = d == 128 ? 0.68 : 0.39;
  constexpr double kFixed = 3.0, kShared = 1.8, kSum = 4.0, kSumRate = 1.8e6;  // us, bytes a us
  const double cus = device_cus(), part = causal ? 0.5 : 1.0;  // the work of a causal launch, roughly
  const int64_t kv_heads = need_kv ? batch * hkv : 0, q_heads = need_q ? batch * hq : 0;
  // tiles of a head that are longer than a piece of the longest: all, or causal those that start soon enough (KV) or
  // end late enough (Q)
  auto longs = [&](int64_t tiles, int64_t len, int64_t cut, int64_t n) -> int64_t {
    if (n == 1) return 0;
    return causal ? std::clamp<int64_t>(cdiv(cut - len / n, kOwnRows / kStageRows), 0, tiles) : tiles;
  };
  double best = 0.0;
  for (int64_t ks : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
    if (ks > 1 && (kv == 0 || kv_len < 8 * ks)) break;
    const int64_t kl = longs(f.kv_tiles, cdiv(sq, kStageRows), cdiv(sq, kStageRows), ks);
    for (int64_t qs : {1, 2, 4, 8, 16}) {
      if (qs > 1 && (q == 0 || q_len < 8 * qs)) break;
      const int64_t ql = longs(f.q_tiles, q_len, f.q_tiles * (kOwnRows / kStageRows), qs);
      const int64_t kv_pieces = kv_heads * kl * ks, q_pieces = q_heads * ql * qs;
      const double items = static_cast<double>(kv + kv_pieces - kv_heads * kl + q + q_pieces - q_heads * ql);
      const double longest = std::max(kv > 0 ? static_cast<double>(kv_len) / static_cast<double>(ks) * item_kv : 0.0,
                                      q > 0 ? static_cast<double>(q_len) / static_cast<double>(qs) * item_q : 0.0) + kFixed;
      const double work = part * (static_cast<double>(kv * kv_len) * cu_kv + static_cast<double>(q * q_len) * cu_q) +
                          items * kFixed * 0.5;
      const double bytes = static_cast<double>(2 * kv_pieces + q_pieces) * kOwnRows * static_cast<double>(d) * 4;
      const double t = std::max(longest * (items > cus ? kShared : 1.0), work / cus) + (bytes > 0 ? kSum + bytes / kSumRate : 0.0);
      if ((ks == 1 && qs == 1) || t < best) {
        best = t;
        f.kv_splits = ks, f.kv_long = kl, f.kv_pieces = kv_pieces;
        f.q_splits = qs, f.q_long = ql, f.q_pieces = q_pieces;
      }
    }
  }
  f.kv_items = kv + f.kv_pieces - kv_heads * f.kv_long;
  f.q_items = q + f.q_pieces - q_heads * f.q_long;
  f.stat_tiles = cdiv(sq, kStatRows) * (kStatRows / 32);
  f.v_blocks = bf16 ? 0 : cdiv(sk, kPreRows);
  f.stat_off = 0;
  f.omax_off = f.stat_off + batch * hq * f.stat_tiles * 64 * 4;
  f.vmax_off = f.omax_off + (bf16 ? 0 : cdiv(batch * hq * cdiv(sq, kPreRows) * 8, 16) * 16);
  f.part_off = f.vmax_off + (bf16 ? 0 : cdiv(batch * hkv * f.v_blocks * 4, 16) * 16);
  f.bytes = f.part_off + (2 * f.kv_pieces + f.q_pieces) * kOwnRows * d * 4;
  return f;
}

int bwd_sizes(const char* fn, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t q_len, int64_t kv_len,
              int64_t head_dim) {
  if (head_dim != 64 && head_dim != 128)
    return set_error(SAGE_ERR_UNSUPPORTED, "head_dim must be 64 or 128, got %lld", static_cast<long long>(head_dim));
  if (batch < 0 || q_heads <= 0 || kv_heads <= 0 || q_len < 0 || kv_len < 0)
    return set_error(SAGE_ERR_INVALID_ARG, "%s: negative or zero size", fn);
  if (q_heads % kv_heads != 0)
    return set_error(SAGE_ERR_INVALID_ARG, "q_heads (%lld) must be a multiple of kv_heads (%lld)",
                     static_cast<long long>(q_heads), static_cast<long long>(kv_heads));
  // a launch has at most 2^24 - 1 blocks of 256 threads (the row pass: one per 64 rows of a head); a KV item's stages
  // are counted in 32 bits
  constexpr int64_t kMost = INT32_MAX, kBlocks = (1 << 24) - 1;
  if (batch > kMost || q_heads > kMost || q_len > kMost - 256 || kv_len > kMost - 256 || batch * q_heads > kBlocks ||
      q_heads / kv_heads > kMost / (q_len / kStageRows + 1) ||
      batch * q_heads * (cdiv(q_len, kPreRows) + cdiv(kv_len, kPreRows)) > kBlocks)
    return set_error(SAGE_ERR_UNSUPPORTED, "%s: sizes beyond 32-bit grid limits", fn);
  return SAGE_OK;
}

int attn_bwd(const char* fn, bool own_lse, const void* dout, const void* query, const void* key, const void* value,
             const void* out, const float* lse, const float* dlse, void* dq, void* dk, void* dv, int dtype, int64_t batch,
             int64_t q_heads, int64_t kv_heads, int64_t q_len, int64_t kv_len, int64_t head_dim, const int64_t* strides,
             int is_causal, double sm_scale, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (dtype != SAGE_DTYPE_F16 && dtype != SAGE_DTYPE_BF16)
    return set_error(SAGE_ERR_INVALID_ARG, "%s: dtype must be SAGE_DTYPE_F16 or SAGE_DTYPE_BF16, got %d", fn, dtype);
  if (int rc = bwd_sizes(fn, batch, q_heads, kv_heads, q_len, kv_len, head_dim)) return rc;
  if (workspace_bytes < 0) return set_error(SAGE_ERR_INVALID_ARG, "%s: negative workspace size", fn);
  if (strides == nullptr) return set_error(SAGE_ERR_INVALID_ARG, "%s: null strides", fn);
  if ((dk == nullptr) != (dv == nullptr)) return set_error(SAGE_ERR_INVALID_ARG, "%s: dk and dv go together", fn);
  const bool need_q = dq != nullptr && q_len > 0, need_kv = dk != nullptr && kv_len > 0;
  if (batch == 0 || (!need_q && !need_kv)) return SAGE_OK;
  if ((q_len > 0 && (!dout || !query || !out || !lse)) || (kv_len > 0 && (!key || !value)))
    return set_error(SAGE_ERR_INVALID_ARG, "%s: null pointer argument", fn);
  for (const void* ptr : {dout, query, key, value, out, static_cast<const void*>(dq), static_cast<const void*>(dk),
                          static_cast<const void*>(dv)})
    if (!aligned(ptr, 16)) return set_error(SAGE_ERR_ALIGNMENT, "%s: tensors must be 16-byte aligned", fn);
  if (!aligned(lse, 4) || !aligned(dlse, 4)) return set_error(SAGE_ERR_ALIGNMENT, "%s: lse and dlse must be 4-byte aligned", fn);
  Rows rows[8];  // dout, query, key, value, out, dq, dk, dv
  const void* ptrs[8] = {dout, query, key, value, out, dq, dk, dv};
  for (int i = 0; i < 8; ++i) {
    rows[i] = {ptrs[i], strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]};
    if (ptrs[i] == nullptr) continue;
    for (int64_t s : {rows[i].sb, rows[i].sh, rows[i].sn}) {
      if (s < 0) return set_error(SAGE_ERR_INVALID_ARG, "%s: strides must be non-negative", fn);
      if (s % 8) return set_error(SAGE_ERR_ALIGNMENT, "%s: strides must be multiples of 16 bytes", fn);
    }
    const bool is_q = i <= 1 || i == 4 || i == 5;
    const int64_t n = is_q ? q_len : kv_len;
    if (n > 1 && rows[i].sn < head_dim)
      return set_error(SAGE_ERR_INVALID_ARG, "%s: rows must not overlap", fn);
    // byte offsets within a head are 32-bit; the last item runs up to 127 rows past the end
    if (rows[i].sn > UINT32_MAX / 2 || (n + kOwnRows) * rows[i].sn * 2 > static_cast<int64_t>(UINT32_MAX))
      return set_error(SAGE_ERR_UNSUPPORTED, "%s: a head spans more than 32-bit byte offsets", fn);
  }
  const bool bf16 = dtype == SAGE_DTYPE_BF16;
  const BwdPlan f = bwd_plan(bf16, batch, q_heads, kv_heads, q_len, kv_len, head_dim, is_causal != 0, dq != nullptr,
                             dk != nullptr);
  if (f.bytes > 0 && (workspace == nullptr || workspace_bytes < f.bytes || !aligned(workspace, 16)))
    return set_error(SAGE_ERR_INVALID_ARG, "%s: needs a 16-byte aligned workspace of %lld bytes (got %lld)", fn,
                     static_cast<long long>(f.bytes), static_cast<long long>(workspace != nullptr ? workspace_bytes : 0));
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* const ws = static_cast<char*>(workspace);

  BwdParams p;
  p.dout = rows[0];
  p.q = rows[1];
  p.k = rows[2];
  p.v = rows[3];
  p.dq = rows[5];
  p.dk = rows[6];
  p.dv = rows[7];
  p.stat = reinterpret_cast<float*>(ws + f.stat_off);
  p.omax = reinterpret_cast<float*>(ws + f.omax_off);
  p.vmax = reinterpret_cast<float*>(ws + f.vmax_off);
  p.part = reinterpret_cast<float*>(ws + f.part_off);
  p.sm_scale = static_cast<float>(sm_scale);
  p.sc = p.sm_scale * 1.4426950408889634f;
  if (p.sc == 0.0f) p.sc = 0x1p-126f;  // a dead pair's infinite S stays infinite
  p.hq = static_cast<int32_t>(q_heads);
  p.hkv = static_cast<int32_t>(kv_heads);
  p.group = static_cast<int32_t>(q_heads / kv_heads);
  p.sq = static_cast<int32_t>(q_len);
  p.sk = static_cast<int32_t>(kv_len);
  p.causal = is_causal != 0;
  p.stat_tiles = static_cast<int32_t>(f.stat_tiles);
  p.omax_n = static_cast<int32_t>(cdiv(q_len, kPreRows));
  p.vmax_n = static_cast<int32_t>(f.v_blocks);
  p.q_part = 2 * f.kv_pieces;
  p.kv_tiles = static_cast<int32_t>(f.kv_tiles);
  p.kv_long = static_cast<int32_t>(f.kv_long);
  p.kv_splits = static_cast<int32_t>(f.kv_splits);
  p.q_tiles = static_cast<int32_t>(f.q_tiles);
  p.q_long = static_cast<int32_t>(f.q_long);
  p.q_splits = static_cast<int32_t>(f.q_splits);
  auto order = [&](int64_t items, int64_t heads) {
    const bool whole = heads % kXcds == 0;
    const int64_t group = !p.causal || items == 0 ? 0 : whole ? heads / kXcds : heads;
    return ItemOrder{static_cast<int32_t>(items), static_cast<int32_t>(items / heads), whole ? kXcds : 1,
                     static_cast<int32_t>(group), fast_div(std::max<int64_t>(group, 1))};
  };
  p.kv_order = order(f.kv_items, batch * kv_heads);
  p.q_order = order(f.q_items, batch * q_heads);
  p.d_kvi = fast_div(std::max(p.kv_order.head_items, 1));
  p.d_kvs = fast_div(f.kv_splits);
  p.d_kvl = fast_div(std::max<int64_t>(f.kv_long, 1));
  p.d_hkv = fast_div(kv_heads);
  p.d_qi = fast_div(std::max(p.q_order.head_items, 1));
  p.d_qs = fast_div(f.q_splits);
  p.d_ql = fast_div(std::max<int64_t>(f.q_long, 1));
  p.d_hq = fast_div(q_heads);
  p.d_group = fast_div(p.group);

  PreParams r;
  r.out = rows[4];
  r.dout = rows[0];
  r.v = rows[3];
  r.q = rows[1];
  r.k = rows[2];
  r.sc = p.sc;
  r.causal = p.causal;
  r.own_lse = own_lse;
  r.d_group = p.d_group;
  r.lse = lse;
  r.dlse = dlse;
  r.stat = const_cast<float*>(p.stat);
  r.omax = const_cast<float*>(p.omax);
  r.vmax = const_cast<float*>(p.vmax);
  r.hq = p.hq;
  r.hkv = p.hkv;
  r.sq = p.sq;
  r.sk = p.sk;
  r.stat_tiles = p.stat_tiles;
  r.q_blocks = p.omax_n;
  r.q_total = static_cast<int32_t>(batch * q_heads * r.q_blocks);
  r.v_blocks = p.vmax_n;
  r.d_hq = p.d_hq;
  r.d_hkv = p.d_hkv;
  r.heads = static_cast<int32_t>(batch * q_heads);
  r.v_heads = static_cast<int32_t>(batch * kv_heads);
  r.d_heads = fast_div(r.heads);
  r.d_vheads = fast_div(r.v_heads);
  const int64_t pre = r.q_total + batch * kv_heads * r.v_blocks;
  const int64_t kv_rows = 2 * f.kv_pieces / f.kv_splits * kOwnRows;
  const int64_t sum_rows = kv_rows + f.q_pieces / f.q_splits * kOwnRows;

  auto launch = [&](auto d, auto bf) {
    constexpr int D = decltype(d)::value;
    constexpr bool BF = decltype(bf)::value;
    const dim3 rows_grid(static_cast<uint32_t>(pre));
    if (pre > 0 && (p.causal || p.sk <= kExactKeys)) attn_bwd_rows_kernel<D, BF, true><<<rows_grid, dim3(256), 0, st>>>(r);
    else if (pre > 0) attn_bwd_rows_kernel<D, BF, false><<<rows_grid, dim3(256), 0, st>>>(r);
    const dim3 items(static_cast<uint32_t>(f.kv_items + f.q_items));
    if (own_lse) attn_bwd_kernel<D, BF, false><<<items, dim3(kBwdThreads), 0, st>>>(p);
    else attn_bwd_kernel<D, BF, true><<<items, dim3(kBwdThreads), 0, st>>>(p);
    if (sum_rows > 0)
      attn_bwd_sum_kernel<D, BF><<<dim3(static_cast<uint32_t>(cdiv(sum_rows, 256 / (D / 8)))), dim3(256), 0, st>>>(
          p, static_cast<int>(kv_rows), static_cast<int>(sum_rows));
  };
  auto by_type = [&](auto d) {
    if (bf16) launch(d, std::true_type{});
    else launch(d, std::false_type{});
  };
  if (head_dim == 128) by_type(std::integral_constant<int, 128>{});
  else by_type(std::integral_constant<int, 64>{});
  return check_launch(fn);
}
}  // namespace
}  // namespace sage

using namespace sage;

extern "C" int64_t sage_attn_bwd_workspace_bytes(int dtype, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                 int64_t q_len, int64_t kv_len, int64_t head_dim, int is_causal,
                                                 int need_dq, int need_dkv) {
  static const char* const fn = "sage_attn_bwd_workspace_bytes";
  clear_error();
  if (dtype != SAGE_DTYPE_F16 && dtype != SAGE_DTYPE_BF16)
    return set_error(SAGE_ERR_INVALID_ARG, "%s: dtype must be SAGE_DTYPE_F16 or SAGE_DTYPE_BF16, got %d", fn, dtype);
  if (int rc = bwd_sizes(fn, batch, q_heads, kv_heads, q_len, kv_len, head_dim)) return rc;
  if (batch == 0) return 0;
  return bwd_plan(dtype == SAGE_DTYPE_BF16, batch, q_heads, kv_heads, q_len, kv_len, head_dim, is_causal != 0, need_dq != 0,
                  need_dkv != 0).bytes;
}

extern "C" int sage_attn_bwd(const void* dout, const void* query, const void* key, const void* value, const void* out,
                             const float* lse, const float* dlse, void* dq, void* dk, void* dv, int dtype,
                             int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t q_len, int64_t kv_len,
                             int64_t head_dim, const int64_t* strides, int is_causal, double sm_scale,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  return attn_bwd("sage_attn_bwd", false, dout, query, key, value, out, lse, dlse, dq, dk, dv, dtype, batch, q_heads,
                  kv_heads, q_len, kv_len, head_dim, strides, is_causal, sm_scale, workspace, workspace_bytes, stream);
}

extern "C" int sage_attn_direct_bwd(const void* dout, const void* query, const void* key, const void* value,
                                    const void* out, const float* lse, const float* dlse, void* dq, void* dk, void* dv, int dtype,
                                    int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t q_len, int64_t kv_len,
                                    int64_t head_dim, const int64_t* strides, int is_causal, double sm_scale,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
  return attn_bwd("sage_attn_direct_bwd", true, dout, query, key, value, out, lse, dlse, dq, dk, dv, dtype, batch, q_heads,
                  kv_heads, q_len, kv_len, head_dim, strides, is_causal, sm_scale, workspace, workspace_bytes, stream);
}
