// gg_kv8.cu -- attention over the paged 8-bit KV cache (the writing side is in gg_ops.cu).
//
// o = sum_j softmax_j(scale q k_j) v_j with k_j = code * ks, v_j = code * vs, one ks and vs for
// each (block, head). In base-2 logarithms, s_j = q k_j scale log2(e); the value scale joins the
// exponent, t_j = s_j + log2(vs_j), and r is a running maximum of t_j:
//   w_j = 2^(t_j - r),   O = sum w_j code_j,   l = sum w_j / vs_j,   o = O / l
// so blocks of any scales share one accumulator. r is only raised when t_j passes it by more than
// KV8_SLACK, so O is rarely rescaled.
//
// Both products run as f16 tensor-core MMAs with f32 sums. The codes are exact in f16 (int8 by a
// byte in the mantissa of 1024, e4m3 by the hardware's widening). A query row is multiplied by a
// power of two that puts its largest value in [2^14, 2^15). f32 queries are split into f16 hi + lo
// (22 bits) and so are their weights: the lo rows fill the half of the 16-row MMA tile that few
// query rows leave empty, and the two halves are added in registers. f16 and bf16 queries are exact
// in one f16; their weights are rounded to f16 (2^-12 relative, below the output's own 2^-9 / 2^-12).
#include <cuda_fp8.h>

#include "gg_launch.h"
#include "gg_ops.h"

namespace gg {

constexpr float KV8_SLACK = 8.f;    // w_j <= 2^8
constexpr float KV8_WMUL = 128.f;    // weights enter the MMA as w_j 2^7 <= 2^15
constexpr float KV8_NEG = -1e30f;   // stands for -inf in running maxima (no inf - inf)

struct Kv8Args {
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const void* q;
  void* out;
  float* lse;
  const int32_t *cu, *lens, *table;
  float* part_o;    // [row][head][split][hd]
  float2* part_ml;  // [row][head][split]: r, l
  long long q_row, q_head, o_row, o_head, table_stride;
  float scale_log2;
  int seqs, rows, max_rows, max_len, num_blocks, block_shift, kv_heads, group, hd, window, q_type;
  int row_tiles, splits, split_steps;
  int q_vec;  // every head of q starts on a 16-byte boundary
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
// Four elements from i on (a multiple of four).
GG_DEV float4 load_elem4(const void* p, int type, long long i, int vec) {
  if (!vec) return make_float4(load_elem(p, type, i), load_elem(p, type, i + 1), load_elem(p, type, i + 2), load_elem(p, type, i + 3));
  if (type == GG_T_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
  const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
  if (type == GG_T_BF16)
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

// The rows of request s: first row, number of rows (within the batch and max_rows), length.
struct Kv8Seq {
  int row0, n, len;
  long long first_pos;  // position of row row0
};
GG_DEV Kv8Seq kv8_seq(const Kv8Args& a, int s) {
  Kv8Seq q;
  const int c0 = a.cu[s], c1 = a.cu[s + 1], len = max(a.lens[s], 0);
  q.row0 = max(c0, 0);
  q.n = max(min(c1, a.rows) - q.row0, 0);
  q.first_pos = (long long)len - (c1 - c0);
  q.n = min(q.n, a.max_rows);
  q.len = min(len, a.max_len);
  return q;
}

// ------------------------------------------------------------------------------ few rows
//
// One CTA: one request, one key head, one tile of query rows (the `group` heads of a few tokens)
// and one range of keys. Bound by the cache's bytes. Each of the four warps streams its own steps of 16 keys
// through a private cp.async ring (no barriers between warps): 16 keys are one MMA's depth for
// the second product and never cross a block. The warps' results meet in shared memory at the
// end; ranges meet in gg_kv8_merge_kernel.
//
// Fragments (lane = 4 g + t): key g of an 8-key tile reads dims 64 j + 16 t .. + 15 as one 16-byte
// word, whose four 4-byte parts are the lane's operand values of four MMA depth steps; q is
// laid out to match. For V the lane reads 16 dims of the four keys 2t, 2t+1, 2t+8, 2t+9: column g of
// output tile (4 w + i) is dim 16 g + 4 w + i. The 16-byte words of a row sit at swizzled places
// so that neither read has bank conflicts.
constexpr int KV8_WARPS = 4;
constexpr int KV8_STEP = 16;

template <int HD>
struct RowsShape {
  static constexpr int STAGES = HD == 256 ? 3 : HD == 128 ? 6 : 8;
  static constexpr int STAGE_BYTES = 2 * KV8_STEP * HD;
  static constexpr int QF_BYTES = HD / 16 * 512;
  static constexpr int RING_BYTES = KV8_WARPS * STAGES * STAGE_BYTES;
  static constexpr int META_BYTES = KV8_WARPS * STAGES * 16;
  static constexpr int SMEM = QF_BYTES + RING_BYTES + META_BYTES;
};

template <int HD>
GG_DEV uint32_t kswz(int key, int c) {  // byte offset of 16-byte word c of key `key`
  if constexpr (HD >= 128) return key * HD + ((c ^ ((key & 1) << 2)) << 4);
  else return key * HD + (c << 4);
}
template <int HD>
GG_DEV uint32_t vswz(int key, int c) {
  if constexpr (HD >= 128) return key * HD + ((c ^ (((key >> 1) & 3) << 1)) << 4);
  else return (key >> 1) * 128 + (((key ^ (key >> 1)) & 1) << 6) + ((c ^ (((key >> 2) & 1) << 1)) << 4);
}

template <int HD, int CODE, bool HILO>
__global__ void __launch_bounds__(KV8_WARPS * 32, 2) gg_kv8_rows_kernel(const Kv8Args a) {
  typedef RowsShape<HD> S;
  constexpr int RT = HILO ? 8 : 16;  // query rows of a tile
  constexpr int NR = HILO ? 1 : 2;   // rows of a lane
  extern __shared__ __align__(128) unsigned char kv8_smem[];
  __shared__ float s_mul[16];
  __shared__ float2 s_ml[KV8_WARPS][16];
  __shared__ int s_pos[16];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  int x = blockIdx.x;
  const int split = x % a.splits;
  x /= a.splits;
  const int rt = x % a.row_tiles;
  x /= a.row_tiles;
  const int h = x % a.kv_heads, s = x / a.kv_heads;
  const Kv8Seq sq = kv8_seq(a, s);
  const int items = sq.n * a.group, base = rt * RT;
  if (base >= items) return;
  const int nitems = min(RT, items - base);
  const int heads = a.kv_heads * a.group;
  // keys that any row of the tile sees
  const long long pos_lo = sq.first_pos + base / a.group, pos_hi = sq.first_pos + (base + nitems - 1) / a.group;
  const int kmax = (int)min((long long)sq.len, pos_hi + 1);
  const int kmin = a.window ? (int)max(0ll, pos_lo - a.window + 1) & ~(KV8_STEP - 1) : 0;
  const int steps = kmax > kmin ? (kmax - kmin + KV8_STEP - 1) / KV8_STEP : 0;
  const int st0 = min(split * a.split_steps, steps), st1 = min(st0 + a.split_steps, steps);

  // ---- query rows -> f16 operand fragments
  unsigned char* qf = kv8_smem;
  for (int row = warp; row < RT; row += KV8_WARPS) {
    const bool live = row < nitems;
    const int it = base + row;
    const long long qi = live ? (long long)(sq.row0 + it / a.group) * a.q_row + (long long)(h * a.group + it % a.group) * a.q_head : 0;
    constexpr int PER = (HD / 4 + 31) / 32;
    float4 v[PER];
    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < PER; p++) {
      const int d = 4 * (lane + 32 * p);
      v[p] = live && d < a.hd ? load_elem4(a.q, a.q_type, qi + d, a.q_vec) : make_float4(0.f, 0.f, 0.f, 0.f);
      top = max(max(top, __float_as_uint(v[p].x) & 0x7fffffffu), __float_as_uint(v[p].y) & 0x7fffffffu);
      top = max(max(top, __float_as_uint(v[p].z) & 0x7fffffffu), __float_as_uint(v[p].w) & 0x7fffffffu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    const int ex = min(max((int)(top >> 23) - 127, -100), 127);
    const float up = __uint_as_float((uint32_t)(14 - ex + 127) << 23);
    if (lane == 0) {
      s_mul[row] = __uint_as_float((uint32_t)(ex - 14 + 127) << 23) * a.scale_log2;
      s_pos[row] = live ? (int)min(sq.first_pos + it / a.group, (long long)sq.len - 1) : -1;
    }
#pragma unroll
    for (int p = 0; p < PER; p++) {
      const int d = 4 * (lane + 32 * p);
      if (d >= HD) break;
      const int ks = 4 * (d >> 6) + ((d >> 2) & 3), tt = (d >> 4) & 3;
      uint32_t* f = reinterpret_cast<uint32_t*>(qf + ((ks * 32) + (row & 7) * 4 + tt) * 16);
      if constexpr (HILO) {
        split_f16(v[p].x * up, v[p].y * up, f[0], f[1]);
        split_f16(v[p].z * up, v[p].w * up, f[2], f[3]);
      } else {
        f[row >> 3] = half2_bits(v[p].x * up, v[p].y * up);
        f[2 + (row >> 3)] = half2_bits(v[p].z * up, v[p].w * up);
      }
    }
  }
  __syncthreads();

  unsigned char* ring = kv8_smem + S::QF_BYTES + warp * S::STAGES * S::STAGE_BYTES;
  const uint32_t ring_u = smem_u32(ring);
  float4* meta = reinterpret_cast<float4*>(kv8_smem + S::QF_BYTES + S::RING_BYTES) + warp * S::STAGES;
  const int first = st0 + warp;
  const int n = st1 > first ? (st1 - first + KV8_WARPS - 1) / KV8_WARPS : 0;
  const int32_t* table = a.table + (long long)s * a.table_stride;

  float mul[NR], rmax[NR], lsum[NR];
  int hi_key[NR], lo_key[NR];
#pragma unroll
  for (int i = 0; i < NR; i++) {
    mul[i] = s_mul[g + 8 * i];
    hi_key[i] = s_pos[g + 8 * i];
    // s_pos is cut at the last key: the window is measured from the row's own position
    const int it = base + g + 8 * i;
    lo_key[i] = a.window ? (int)max(0ll, sq.first_pos + it / a.group - a.window + 1) : 0;
    rmax[i] = KV8_NEG;
    lsum[i] = 0.f;
  }
  float o[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) o[i][j] = 0.f;

  // block ids and scales of 32 steps at a time, one step per lane
  int b_id = -1;
  float4 b_meta = make_float4(0.f, 0.f, 0.f, 0.f);
  const auto issue = [&](int i) {
    if (i < n) {
      if ((i & 31) == 0) {
        const int ii = i + lane;
        b_id = -1;
        b_meta = make_float4(0.f, 0.f, 0.f, 0.f);
        if (ii < n) {
          const int key0 = kmin + (first + ii * KV8_WARPS) * KV8_STEP;
          const int id = table[key0 >> a.block_shift];
          if (id >= 0 && id < a.num_blocks) {
            b_id = id;
            const float vs = a.vs[(long long)id * a.kv_heads + h];
            b_meta = make_float4(a.ks[(long long)id * a.kv_heads + h], log2f(vs), 1.f / vs, 1.f);
          }
        }
      }
      const int stage = i % S::STAGES;
      if (lane == (i & 31)) meta[stage] = b_meta;
      const int id = __shfl_sync(0xffffffffu, b_id, i & 31);
      const int key0 = kmin + (first + i * KV8_WARPS) * KV8_STEP;
      const long long at = (((long long)max(id, 0) * a.kv_heads + h) << a.block_shift) + (key0 & ((1 << a.block_shift) - 1));
      const uint8_t* ksrc = a.kc + at * a.hd;
      const uint8_t* vsrc = a.vc + at * a.hd;
      const uint32_t dst = ring_u + stage * S::STAGE_BYTES;
      constexpr int W = HD / 16;  // 16-byte words of a key
#pragma unroll
      for (int c = 0; c < KV8_STEP * W / 32; c++) {
        const int k = (lane + 32 * c) / W, w = (lane + 32 * c) % W;
        const bool in = id >= 0 && key0 + k < sq.len && w * 16 < a.hd;
        const int off = in ? k * a.hd + w * 16 : 0;
        cp_async16(dst + kswz<HD>(k, w), ksrc + off, in ? 16 : 0);
        cp_async16(dst + KV8_STEP * HD + vswz<HD>(k, w), vsrc + off, in ? 16 : 0);
      }
    }
    cp_async_commit();
  };
  for (int i = 0; i < S::STAGES - 1; i++) issue(i);
  const uint32_t qf_u = smem_u32(qf) + lane * 16;
  for (int i = 0; i < n; i++) {
    cp_async_wait<S::STAGES - 2>();
    __syncwarp();
    issue(i + S::STAGES - 1);
    const uint32_t kst = ring_u + (i % S::STAGES) * S::STAGE_BYTES, vst = kst + KV8_STEP * HD;
    const float4 mt = meta[i % S::STAGES];
    const int key0 = kmin + (first + i * KV8_WARPS) * KV8_STEP;
    // scores: two 8-key tiles, two accumulators each to shorten the chains
    float c[2][2][4] = {};
#pragma unroll
    for (int j = 0; j < HD / 64; j++) {
      const uint4 k0 = lds128(kst + kswz<HD>(g, 4 * j + t)), k1 = lds128(kst + kswz<HD>(g + 8, 4 * j + t));
      const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
      for (int p = 0; p < 4; p++) {
        const uint4 qa = lds128(qf_u + (4 * j + p) * 512);
        uint32_t b0, b1;
        widen4<CODE>(w0[p], b0, b1);
        mma_f16(c[0][p & 1], qa, b0, b1);
        widen4<CODE>(w1[p], b0, b1);
        mma_f16(c[1][p & 1], qa, b0, b1);
      }
    }
    // softmax weights of the lane's rows at keys key0 + 8 tile + 2t, + 1
    float wt[NR][4];
#pragma unroll
    for (int r = 0; r < NR; r++) {
      float sc[4], top = KV8_NEG;
      bool seen[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int ti = e >> 1, el = e & 1, key = key0 + 8 * ti + 2 * t + el;
        float v = c[ti][0][2 * r + el] + c[ti][1][2 * r + el];
        if constexpr (HILO) v += c[ti][0][2 + el] + c[ti][1][2 + el];
        seen[e] = key <= hi_key[r] && key >= lo_key[r] && mt.w != 0.f;
        sc[e] = seen[e] ? fmaf(v * mt.x, mul[r], mt.y) : KV8_NEG;
        top = fmaxf(top, sc[e]);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (__any_sync(0xffffffffu, top > rmax[r] + KV8_SLACK)) {
        const float nr = top > rmax[r] + KV8_SLACK ? top : rmax[r];
        const float f = ex2(rmax[r] - nr);  // rmax = KV8_NEG: 2^-huge = 0
        rmax[r] = nr;
        lsum[r] *= f;
#pragma unroll
        for (int d = 0; d < HD / 8; d++) {
          o[d][2 * r] *= f;
          o[d][2 * r + 1] *= f;
          if constexpr (HILO) {
            o[d][2] *= f;
            o[d][3] *= f;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 4; e++) {
        wt[r][e] = seen[e] ? ex2(sc[e] - rmax[r]) : 0.f;
        lsum[r] += seen[e] ? wt[r][e] * mt.z : 0.f;
        wt[r][e] *= KV8_WMUL;
      }
    }
    uint4 pa;
    if constexpr (HILO) {
      split_f16(wt[0][0], wt[0][1], pa.x, pa.y);
      split_f16(wt[0][2], wt[0][3], pa.z, pa.w);
    } else {
      pa.x = half2_bits(wt[0][0], wt[0][1]);
      pa.y = half2_bits(wt[NR - 1][0], wt[NR - 1][1]);
      pa.z = half2_bits(wt[0][2], wt[0][3]);
      pa.w = half2_bits(wt[NR - 1][2], wt[NR - 1][3]);
    }
    if constexpr (HD >= 128) {
#pragma unroll
      for (int jj = 0; jj < HD / 128; jj++) {
        const uint4 v0 = lds128(vst + vswz<HD>(2 * t, 8 * jj + g)), v1 = lds128(vst + vswz<HD>(2 * t + 1, 8 * jj + g));
        const uint4 v2 = lds128(vst + vswz<HD>(2 * t + 8, 8 * jj + g)), v3 = lds128(vst + vswz<HD>(2 * t + 9, 8 * jj + g));
        const uint32_t x0[4] = {v0.x, v0.y, v0.z, v0.w}, x1[4] = {v1.x, v1.y, v1.z, v1.w};
        const uint32_t x2[4] = {v2.x, v2.y, v2.z, v2.w}, x3[4] = {v3.x, v3.y, v3.z, v3.w};
#pragma unroll
        for (int w = 0; w < 4; w++) {
          uint32_t b0[4], b1[4];
          widen4_pairs<CODE>(x0[w], x1[w], b0);
          widen4_pairs<CODE>(x2[w], x3[w], b1);
#pragma unroll
          for (int e = 0; e < 4; e++) mma_f16(o[16 * jj + 4 * w + e], pa, b0[e], b1[e]);
        }
      }
    } else {  // HD = 64: 8 dims of the four keys per lane
      const uint32_t in = (g & 1) << 3;
      const uint2 v0 = lds64(vst + vswz<HD>(2 * t, g >> 1) + in), v1 = lds64(vst + vswz<HD>(2 * t + 1, g >> 1) + in);
      const uint2 v2 = lds64(vst + vswz<HD>(2 * t + 8, g >> 1) + in), v3 = lds64(vst + vswz<HD>(2 * t + 9, g >> 1) + in);
      const uint32_t x0[2] = {v0.x, v0.y}, x1[2] = {v1.x, v1.y}, x2[2] = {v2.x, v2.y}, x3[2] = {v3.x, v3.y};
#pragma unroll
      for (int w = 0; w < 2; w++) {
        uint32_t b0[4], b1[4];
        widen4_pairs<CODE>(x0[w], x1[w], b0);
        widen4_pairs<CODE>(x2[w], x3[w], b1);
#pragma unroll
        for (int e = 0; e < 4; e++) mma_f16(o[4 * w + e], pa, b0[e], b1[e]);
      }
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int r = 0; r < NR; r++) {
    lsum[r] += __shfl_xor_sync(0xffffffffu, lsum[r], 1);
    lsum[r] += __shfl_xor_sync(0xffffffffu, lsum[r], 2);
    if (t == 0) s_ml[warp][g + 8 * r] = make_float2(rmax[r], lsum[r]);
  }
  __syncthreads();  // every warp has left its ring: it becomes [warp][row][HD + 4] f32
  constexpr int OST = HD + 4;
  static_assert(KV8_WARPS * RT * OST * 4 <= S::QF_BYTES + S::RING_BYTES, "partial outputs fit the ring");
  float* so = reinterpret_cast<float*>(kv8_smem);
#pragma unroll
  for (int r = 0; r < NR; r++) {
    float* dst = so + (warp * RT + g + 8 * r) * OST;
#pragma unroll
    for (int i = 0; i < HD / 8; i++)
#pragma unroll
      for (int el = 0; el < 2; el++) {
        float v = o[i][2 * r + el];
        if constexpr (HILO) v += o[i][2 + el];
        const int col = 2 * t + el;
        const int d = HD >= 128 ? 128 * (i >> 4) + 16 * col + (i & 15) : 8 * col + i;
        dst[d] = v;
      }
  }
  __syncthreads();
  for (int row = warp; row < nitems; row += KV8_WARPS) {
    const int it = base + row, tok = it / a.group, hq = h * a.group + it % a.group;
    float r = KV8_NEG, l = 0.f, f[KV8_WARPS];
#pragma unroll
    for (int w = 0; w < KV8_WARPS; w++) r = fmaxf(r, s_ml[w][row].x);
#pragma unroll
    for (int w = 0; w < KV8_WARPS; w++) {
      f[w] = ex2(s_ml[w][row].x - r);
      l += f[w] * s_ml[w][row].y;
    }
    const long long ri = (long long)(sq.row0 + tok);
    const long long pi = (ri * heads + hq) * a.splits + split;
    const float inv = a.splits == 1 ? (l == 0.f ? 0.f : (1.f / KV8_WMUL) / l) : 1.f / KV8_WMUL;
    for (int d = lane; d < a.hd; d += 32) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < KV8_WARPS; w++) v += f[w] * so[(w * RT + row) * OST + d];
      v *= inv;
      if (a.splits == 1) store_elem(a.out, a.q_type, ri * a.o_row + (long long)hq * a.o_head + d, v);
      else a.part_o[pi * a.hd + d] = v;
    }
    if (lane == 0) {
      if (a.splits > 1) a.part_ml[pi] = make_float2(r, l);
      else if (a.lse) a.lse[ri * heads + hq] = l == 0.f ? -INFINITY : (r + log2f(l)) * 0.6931471805599453f;
    }
  }
}

// One warp per (request, token, query head): the results of the key ranges joined.
__global__ void __launch_bounds__(128) gg_kv8_merge_kernel(const Kv8Args a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int heads = a.kv_heads * a.group;
  long long x = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int hq = (int)(x % heads);
  x /= heads;
  const int tok = (int)(x % a.max_rows);
  x /= a.max_rows;
  if (x >= a.seqs) return;
  const Kv8Seq sq = kv8_seq(a, (int)x);
  if (tok >= sq.n) return;
  const long long ri = sq.row0 + tok, pi = (ri * heads + hq) * a.splits;
  float r = KV8_NEG, l = 0.f;
  for (int z = lane; z < a.splits; z += 32) r = fmaxf(r, a.part_ml[pi + z].x);
  r = warp_max(r);
  for (int z = lane; z < a.splits; z += 32) l += ex2(a.part_ml[pi + z].x - r) * a.part_ml[pi + z].y;
  l = warp_sum(l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int d = lane; d < a.hd; d += 32) {
    float v = 0.f;
    for (int z = 0; z < a.splits; z++) v += ex2(a.part_ml[pi + z].x - r) * a.part_o[(pi + z) * a.hd + d];
    store_elem(a.out, a.q_type, ri * a.o_row + (long long)hq * a.o_head + d, v * inv);
  }
  if (lane == 0 && a.lse) a.lse[ri * heads + hq] = l == 0.f ? -INFINITY : (r + log2f(l)) * 0.6931471805599453f;
}

template <int HD, int CODE, bool HILO>
cudaError_t launch_rows(const Kv8Args& a, cudaStream_t s) {
  auto* k = gg_kv8_rows_kernel<HD, CODE, HILO>;
  cudaError_t r = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, RowsShape<HD>::SMEM);
  if (r != cudaSuccess) return r;
  const long long grid = (long long)a.seqs * a.kv_heads * a.row_tiles * a.splits;
  return launch_pdl(k, dim3((unsigned)grid), dim3(KV8_WARPS * 32), RowsShape<HD>::SMEM, s, a);
}
template <int HD>
cudaError_t launch_rows_hd(const Kv8Args& a, int code, cudaStream_t s) {
  const bool hilo = a.q_type == GG_T_F32;
  if (code == GG_KV8_INT8) return hilo ? launch_rows<HD, GG_KV8_INT8, true>(a, s) : launch_rows<HD, GG_KV8_INT8, false>(a, s);
  return hilo ? launch_rows<HD, GG_KV8_E4M3, true>(a, s) : launch_rows<HD, GG_KV8_E4M3, false>(a, s);
}

// How a call is cut: row tiles of a request and head, key ranges, steps of a range.
struct Kv8Plan {
  int row_tiles, splits, split_steps;
};
static Kv8Plan kv8_plan(const gg_kv8_cache& c, const gg_rows& q, const gg_kv8_batch& b, int window) {
  Kv8Plan p;
  const int rt = q.type == GG_T_F32 ? 8 : 16;
  const long long items = (long long)b.max_rows * (q.heads / c.kv_heads);
  p.row_tiles = (int)((items + rt - 1) / rt);
  // keys that a tile may read: all, or its window with the rows between its first and last
  long long keys = b.max_len;
  if (window) keys = keys < (long long)window + rt + 2 * KV8_STEP ? keys : (long long)window + rt + 2 * KV8_STEP;
  const long long steps = (keys + KV8_STEP - 1) / KV8_STEP;
  const long long units = (long long)b.seqs * c.kv_heads * p.row_tiles;
  // two CTAs fit an SM; four waves of them even out requests of different lengths
  long long splits = (148 * 2 * 4 + units - 1) / units;
  const long long most = (steps + 2 * KV8_WARPS - 1) / (2 * KV8_WARPS);  // at least two steps for each warp
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  p.split_steps = (int)((steps + splits - 1) / splits);
  if (p.split_steps < 1) p.split_steps = 1;
  p.splits = (int)((steps + p.split_steps - 1) / p.split_steps);
  if (p.splits < 1) p.splits = 1;
  return p;
}
static size_t kv8_bytes(const Kv8Plan& p, const gg_kv8_cache& c, const gg_rows& q, const gg_kv8_batch& b) {
  if (p.splits == 1) return 0;
  const size_t parts = (size_t)b.rows * q.heads * p.splits;
  return parts * c.head_dim * 4 + parts * 8;
}

static int kv8_check(const char* fn, const gg_kv8_cache* c, const gg_rows* q, const gg_kv8_batch* b, int window) {
  if (int rc = ops_check_cache(fn, c)) return rc;
  if (int rc = ops_check_rows(fn, "q", q, b->rows, c->head_dim)) return rc;
  if (q->heads % c->kv_heads) return ops_fail(GG_E_ARG, "%s: %d query heads over %d key heads", fn, q->heads, c->kv_heads);
  if (!b->cu_rows || !b->lens || !b->table) return ops_fail(GG_E_ARG, "%s: null array in the batch", fn);
  if (b->seqs < 0 || b->rows < 0 || b->max_rows < 0 || b->max_len < 0)
    return ops_fail(GG_E_ARG, "%s: seqs %d, rows %d, max_rows %d, max_len %d out of range", fn, b->seqs, b->rows, b->max_rows, b->max_len);
  if (b->table_stride < ((long long)b->max_len + c->block_tokens - 1) / c->block_tokens)
    return ops_fail(GG_E_ARG, "%s: table_stride %lld holds fewer than max_len %d tokens", fn, (long long)b->table_stride, b->max_len);
  if (window < 0) return ops_fail(GG_E_ARG, "%s: window %d", fn, window);
  const Kv8Plan p = kv8_plan(*c, *q, *b, window);
  if ((long long)b->seqs * c->kv_heads * p.row_tiles * p.splits >= (1ll << 31))
    return ops_fail(GG_E_ARG, "%s: the batch needs more than 2^31 tiles", fn);
  return GG_OK;
}

}  // namespace gg

extern "C" int gg_kv8_attention_workspace(const gg_kv8_cache* c, const gg_rows* q, const gg_kv8_batch* b, int window, size_t* bytes) {
  using namespace gg;
  const char* fn = "gg_kv8_attention_workspace";
  if (!c || !q || !b || !bytes) return ops_fail(GG_E_ARG, "%s: null argument", fn);
  if (int rc = kv8_check(fn, c, q, b, window)) return rc;
  *bytes = b->seqs ? kv8_bytes(kv8_plan(*c, *q, *b, window), *c, *q, *b) : 0;
  return GG_OK;
}

extern "C" int gg_kv8_attention(const gg_kv8_cache* c, const gg_rows* q, const gg_rows* out, float* lse, const gg_kv8_batch* b,
                                double scale, int window, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace gg;
  const char* fn = "gg_kv8_attention";
  if (!c || !q || !out || !b) return ops_fail(GG_E_ARG, "%s: null argument", fn);
  if (int rc = kv8_check(fn, c, q, b, window)) return rc;
  if (int rc = ops_check_rows(fn, "out", out, b->rows, c->head_dim)) return rc;
  if (out->type != q->type || out->heads != q->heads) return ops_fail(GG_E_ARG, "%s: out has another type or number of heads than q", fn);
  if (!(scale == scale) || scale > 1e30 || scale < -1e30) return ops_fail(GG_E_ARG, "%s: scale is not a number", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int rc = ops_check_stream(fn, s)) return rc;
  if (b->seqs == 0 || b->rows == 0 || b->max_rows == 0) return GG_OK;
  const Kv8Plan p = kv8_plan(*c, *q, *b, window);
  const size_t need = kv8_bytes(p, *c, *q, *b);
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace & 15))
    return ops_fail(GG_E_ARG, "%s: needs %zu bytes of 16-byte aligned workspace, got %zu", fn, need, workspace ? workspace_bytes : (size_t)0);
  Kv8Args a = {};
  a.kc = static_cast<const uint8_t*>(c->k_codes);
  a.vc = static_cast<const uint8_t*>(c->v_codes);
  a.ks = c->k_scale;
  a.vs = c->v_scale;
  a.q = q->data;
  a.out = out->data;
  a.lse = lse;
  a.cu = b->cu_rows;
  a.lens = b->lens;
  a.table = b->table;
  a.table_stride = b->table_stride;
  a.q_row = q->row_stride;
  a.q_head = q->head_stride;
  a.o_row = out->row_stride;
  a.o_head = out->head_stride;
  a.scale_log2 = (float)(scale * 1.4426950408889634074);
  a.seqs = b->seqs;
  a.rows = b->rows;
  a.max_rows = b->max_rows;
  a.max_len = b->max_len;
  a.num_blocks = c->num_blocks;
  a.block_shift = __builtin_ctz(c->block_tokens);
  a.kv_heads = c->kv_heads;
  a.group = q->heads / c->kv_heads;
  a.hd = c->head_dim;
  a.window = window;
  a.q_type = q->type;
  a.q_vec = ops_aligned16(*q);
  a.row_tiles = p.row_tiles;
  a.splits = p.splits;
  a.split_steps = p.split_steps;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(static_cast<float*>(workspace) + (size_t)b->rows * q->heads * p.splits * c->head_dim);
  cudaError_t r = c->head_dim <= 64 ? launch_rows_hd<64>(a, c->code, s) : c->head_dim <= 128 ? launch_rows_hd<128>(a, c->code, s) : launch_rows_hd<256>(a, c->code, s);
  if (r == cudaSuccess && p.splits > 1) {
    const long long warps = (long long)b->seqs * b->max_rows * q->heads;
    r = launch_pdl(gg_kv8_merge_kernel, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, s, a);
  }
  if (r != cudaSuccess) return ops_fail(GG_E_CUDA, "%s: launch: %s", fn, cudaGetErrorString(r));
  return GG_OK;
}
