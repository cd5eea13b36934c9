// gg_kv8.h -- what the kernels that read the paged 8-bit KV cache share: the arguments of a call, the
// widening of codes and the exponent arithmetic of the softmax.
#pragma once
#include <cuda_fp8.h>

#include "gg_launch.h"
#include "gg_ops.h"

namespace gg {

constexpr float KV8_SLACK = 8.f;    // w_j <= 2^8
constexpr float KV8_WMUL = 128.f;    // weights enter the MMA as w_j 2^7 <= 2^15
// The tensor cores cut the f32 sums they hold (they do not round them). f16 and bf16 outputs leave O there,
// so no sum of theirs takes more than 2^18 keys, in steps of 16 (losses: gg_kv8.cu, gg_kv8_prompt.cu).
constexpr int KV8_LONGEST = 1 << 14;
constexpr float KV8_NEG = -1e30f;   // stands for -inf in running maxima (no inf - inf)

struct Kv8Args {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const void* q;
  void* out;
  float* lse;
  const int32_t *cu, *lens, *table;
  // partial results (r, l: running maximum and sum): many rows [row][head][range], few rows
  // [CTA][row of the tile]
  float* part_o;
  float2* part_ml;
  int* pre;  // few rows: parts before each request, then the steps of a part; or NULL
  long long q_row, q_head, o_row, o_head, table_stride;
  float scale_log2;
  int seqs, rows, max_rows, max_len, num_blocks, block_shift, kv_heads, group, hd, window, q_type;
  int row_tiles, splits, split_steps;  // split_steps: 16-key steps of a key range
  int few_ctas, tile_rows, resident;  // few rows: CTAs of the launch, rows of a tile
  int merge_tokens;                    // tokens of a request that the merge looks at
  int items_lo, items_hi;  // this launch takes requests with items_lo < rows * group <= items_hi
  int q_vec, o_vec;  // every head of q / out starts on a 16-byte boundary
  uint32_t* err;     // takes GG_ERR_WAIT_MBAR when a wait of the many-rows kernel runs out; or NULL
  unsigned long long timeout_ns;
};

GG_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
GG_DEV void mma_f16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
GG_DEV void mma_f16_from_zero(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.f));
}
GG_DEV void add_f32x2(float& a, float& b, float c, float d) {  // a += c, b += d, each rounded to nearest
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}
GG_DEV void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {  // bytes 0: fills zeros, reads nothing
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
GG_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
GG_DEV void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

GG_DEV uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// f32 pair -> f16 hi pair and the f16 pair of what hi leaves.
GG_DEV void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = half2_bits(a - f.x, b - f.y);
}

GG_DEV uint32_t hsub2_bits(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
GG_DEV uint32_t e4m3x2_f16x2(uint32_t two) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"((unsigned short)two));
  return d;
}
// Four codes next to each other -> (0, 1) and (2, 3) as f16 pairs. int8: byte + 128 in the mantissa
// of 1024 (f16 0x6400, steps of 1), minus 1152.
template <int CODE>
GG_DEV void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (CODE == GG_KV8_INT8) {
    w ^= 0x80808080u;
    lo = hsub2_bits(__byte_perm(w, 0x64646464u, 0x4140), 0x64806480u);
    hi = hsub2_bits(__byte_perm(w, 0x64646464u, 0x4342), 0x64806480u);
  } else {
    lo = e4m3x2_f16x2(w);
    hi = e4m3x2_f16x2(w >> 16);
  }
}
// Words a and b of two keys (four dims each) -> for each dim the f16 pair (a, b).
template <int CODE>
GG_DEV void widen4_pairs(uint32_t a, uint32_t b, uint32_t (&d)[4]) {
  if constexpr (CODE == GG_KV8_INT8) {
    const uint32_t x = __byte_perm(a, b, 0x5140) ^ 0x80808080u, y = __byte_perm(a, b, 0x7362) ^ 0x80808080u;
    d[0] = hsub2_bits(__byte_perm(x, 0x64646464u, 0x4140), 0x64806480u);
    d[1] = hsub2_bits(__byte_perm(x, 0x64646464u, 0x4342), 0x64806480u);
    d[2] = hsub2_bits(__byte_perm(y, 0x64646464u, 0x4140), 0x64806480u);
    d[3] = hsub2_bits(__byte_perm(y, 0x64646464u, 0x4342), 0x64806480u);
  } else {
    const uint32_t a0 = e4m3x2_f16x2(a), a1 = e4m3x2_f16x2(a >> 16), b0 = e4m3x2_f16x2(b), b1 = e4m3x2_f16x2(b >> 16);
    d[0] = __byte_perm(a0, b0, 0x5410);
    d[1] = __byte_perm(a0, b0, 0x7632);
    d[2] = __byte_perm(a1, b1, 0x5410);
    d[3] = __byte_perm(a1, b1, 0x7632);
  }
}

GG_DEV float load_elem(const void* p, int type, long long i) {
  if (type == GG_T_F32) return static_cast<const float*>(p)[i];
  if (type == GG_T_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
GG_DEV void store_elem(void* p, int type, long long i, float v) {
  if (type == GG_T_F32) static_cast<float*>(p)[i] = v;
  else if (type == GG_T_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}
// Four elements of each of N x P places (index -1: zeros) as they are in memory, all loads in flight
// together -- the branch on the type stands outside of them, and nothing is widened before the last
// is issued -- and widened afterwards (a CTA's 256 query rows of 128: 16k cycles, 20k with a branch at
// every load).
template <int N, int P, class Index>
GG_DEV void load_raw4(uint4 (&raw)[N][P], const void* p, int type, int vec, Index index) {
  if (!vec) {
#pragma unroll
    for (int j = 0; j < N; j++)
#pragma unroll
      for (int k = 0; k < P; k++) {
        const long long i = index(j, k);
        float f[4] = {0.f, 0.f, 0.f, 0.f};
        if (i >= 0)
#pragma unroll
          for (int e = 0; e < 4; e++) f[e] = load_elem(p, type, i + e);
        raw[j][k] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
      }
  } else if (type == GG_T_F32) {
#pragma unroll
    for (int j = 0; j < N; j++)
#pragma unroll
      for (int k = 0; k < P; k++) {
        const long long i = index(j, k);
        raw[j][k] = make_uint4(0, 0, 0, 0);
        if (i >= 0) raw[j][k] = *reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i);
      }
  } else {
#pragma unroll
    for (int j = 0; j < N; j++)
#pragma unroll
      for (int k = 0; k < P; k++) {
        const long long i = index(j, k);
        uint2 w = make_uint2(0, 0);
        if (i >= 0) w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
        raw[j][k] = make_uint4(w.x, w.y, 0, 0);
      }
  }
}
GG_DEV float4 widen_raw4(const uint4& w, int type, int vec) {
  if (!vec || type == GG_T_F32) return make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
  if (type == GG_T_BF16)
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
GG_DEV void store_elem4(void* p, int type, long long i, const float4& v, int vec) {
  if (!vec) {
    store_elem(p, type, i, v.x);
    store_elem(p, type, i + 1, v.y);
    store_elem(p, type, i + 2, v.z);
    store_elem(p, type, i + 3, v.w);
  } else if (type == GG_T_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = v;
  } else {
    const __nv_bfloat162 b0 = __floats2bfloat162_rn(v.x, v.y), b1 = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) =
        type == GG_T_BF16 ? make_uint2(*reinterpret_cast<const uint32_t*>(&b0), *reinterpret_cast<const uint32_t*>(&b1))
                          : make_uint2(half2_bits(v.x, v.y), half2_bits(v.z, v.w));
  }
}

// The rows of request s: first row, number of rows (within the batch and max_rows), and the keys they
// may see: up to the last row's own, whatever of the request lies behind it. The launch is sized from max_rows,
// max_len and the window (kv8_plan), so no request may have more keys than they allow.
struct Kv8Seq {
  int row0, n, len;
  long long first_pos;  // position of row row0
};
GG_DEV Kv8Seq kv8_seq(const Kv8Args& a, int s) {
  Kv8Seq q;
  const int c0 = max(a.cu[s], 0), c1 = max(a.cu[s + 1], c0), len = max(a.lens[s], 0);  // (in bounds whatever they hold)
  q.row0 = c0;
  q.n = max(min(c1, a.rows) - c0, 0);
  q.first_pos = (long long)len - (c1 - c0);
  q.n = min(q.n, a.max_rows);
  const long long items = (long long)q.n * a.group;
  if (items <= a.items_lo || items > a.items_hi) q.n = 0;  // another launch's request
  q.len = (int)max(min((long long)min(len, a.max_len), q.first_pos + q.n), 0ll);
  return q;
}


// Many rows (gg_kv8_prompt.cu): query rows of a tile, and the launch.
int kv8_prompt_tile(int head_dim);
cudaError_t kv8_launch_prompt(const Kv8Args& a, int code, cudaStream_t s);
// Its wait for a barrier that nobody arrives at, for the self-test.
cudaError_t kv8_wait_probe(uint32_t* err, unsigned long long timeout_ns, cudaStream_t s);

}  // namespace gg
