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
#include "gg_kv8.h"


namespace gg {

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
  const int tok = (int)(x % a.merge_tokens);
  x /= a.merge_tokens;
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
  const long long grid = (long long)a.seqs * a.kv_heads * a.row_tiles * a.splits;
  return launch_big_smem(k, dim3((unsigned)grid), dim3(KV8_WARPS * 32), RowsShape<HD>::SMEM, s, a);
}
template <int HD>
cudaError_t launch_rows_hd(const Kv8Args& a, int code, cudaStream_t s) {
  const bool hilo = a.q_type == GG_T_F32;
  if (code == GG_KV8_INT8) return hilo ? launch_rows<HD, GG_KV8_INT8, true>(a, s) : launch_rows<HD, GG_KV8_INT8, false>(a, s);
  return hilo ? launch_rows<HD, GG_KV8_E4M3, true>(a, s) : launch_rows<HD, GG_KV8_E4M3, false>(a, s);
}

// How a call is cut. Requests with few rows (rows * group up to KV8_FEW) take the kernel above, the
// others the one of gg_kv8_prompt.cu; a call that may hold both launches both, and each skips the
// other's requests.
constexpr int KV8_FEW = 32;

struct Kv8Cut {
  int row_tiles = 0, splits = 0, split_steps = 1;  // row_tiles 0: not launched
  size_t parts = 0;                                // partial results
};
static Kv8Cut kv8_cut(long long items, int tile, long long slots, int least_steps, long long rows, int q_heads,
                      const gg_kv8_cache& c, const gg_kv8_attention_call& b) {
  Kv8Cut p;
  p.row_tiles = (int)((items + tile - 1) / tile);
  // keys that a tile may read: all, or its window with the rows between its first and last
  long long keys = b.max_len;
  if (b.window && keys > (long long)b.window + tile + 2 * KV8_STEP) keys = (long long)b.window + tile + 2 * KV8_STEP;
  const long long steps = (keys + KV8_STEP - 1) / KV8_STEP;
  const long long units = (long long)b.seqs * c.kv_heads * p.row_tiles;
  long long splits = units ? (slots + units - 1) / units : 1;
  const long long most = (steps + least_steps - 1) / least_steps;
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  p.split_steps = (int)((steps + splits - 1) / splits);
  if (p.split_steps < 1) p.split_steps = 1;
  p.splits = (int)((steps + p.split_steps - 1) / p.split_steps);
  if (p.splits < 1) p.splits = 1;
  if (p.splits > 1) p.parts = (size_t)rows * q_heads * p.splits;
  return p;
}
struct Kv8Plan {
  Kv8Cut few, many;
  size_t few_bytes, bytes;
};
static Kv8Plan kv8_plan(const gg_kv8_cache& c, const gg_kv8_attention_call& b) {
  Kv8Plan p;
  const int group = b.q.heads / c.kv_heads;
  const long long items = (long long)b.max_rows * group;
  // few rows: two CTAs fit an SM; four waves of them even out requests of different lengths; at
  // least two steps for each warp. Many rows: one CTA an SM, at least 512 keys.
  p.few = kv8_cut(items < KV8_FEW ? items : KV8_FEW, b.q.type == GG_T_F32 ? 8 : 16, 148 * 2 * 4, 2 * KV8_WARPS, b.rows, b.q.heads, c, b);
  if (items > KV8_FEW) p.many = kv8_cut(items, kv8_prompt_tile(c.head_dim), 148, 32, b.rows, b.q.heads, c, b);
  const auto bytes = [&](const Kv8Cut& k) { return k.parts * c.head_dim * 4 + k.parts * 8; };
  p.few_bytes = bytes(p.few);
  p.bytes = p.few_bytes + bytes(p.many);
  return p;
}

static int kv8_check(const char* fn, const gg_kv8_cache* c, const gg_kv8_attention_call* b) {
  if (int rc = ops_check_cache(fn, c)) return rc;
  if (b->q.type < GG_T_F32 || b->q.type > GG_T_F16) return ops_fail(GG_E_ARG, "%s: q.type %d is none of GG_T_*", fn, b->q.type);
  if (b->q.heads < 1 || b->q.heads > 65535 || b->q.heads % c->kv_heads)
    return ops_fail(GG_E_ARG, "%s: %d query heads over %d key heads", fn, b->q.heads, c->kv_heads);
  if (b->seqs < 0 || b->rows < 0 || b->max_rows < 0 || b->max_len < 0)
    return ops_fail(GG_E_ARG, "%s: seqs %d, rows %d, max_rows %d, max_len %d out of range", fn, b->seqs, b->rows, b->max_rows, b->max_len);
  if (b->window < 0) return ops_fail(GG_E_ARG, "%s: window %d", fn, b->window);
  const Kv8Plan p = kv8_plan(*c, *b);
  for (const Kv8Cut* k : {&p.few, &p.many})
    if ((double)b->seqs * c->kv_heads * k->row_tiles * k->splits >= 2147483647.0)
      return ops_fail(GG_E_ARG, "%s: the batch needs more than 2^31 tiles", fn);
  return GG_OK;
}

}  // namespace gg

extern "C" int gg_kv8_attention_workspace(const gg_kv8_cache* c, const gg_kv8_attention_call* call, size_t* bytes) {
  using namespace gg;
  const char* fn = "gg_kv8_attention_workspace";
  if (!c || !call || !bytes) return ops_fail(GG_E_ARG, "%s: null argument", fn);
  if (int rc = kv8_check(fn, c, call)) return rc;
  *bytes = call->seqs ? kv8_plan(*c, *call).bytes : 0;
  return GG_OK;
}

extern "C" int gg_kv8_attention(const gg_kv8_cache* c, const gg_kv8_attention_call* call, void* stream) {
  using namespace gg;
  const char* fn = "gg_kv8_attention";
  if (!c || !call) return ops_fail(GG_E_ARG, "%s: null argument", fn);
  const gg_kv8_attention_call& b = *call;
  if (int rc = kv8_check(fn, c, call)) return rc;
  if (int rc = ops_check_rows(fn, "q", &b.q, b.rows, c->head_dim)) return rc;
  if (int rc = ops_check_rows(fn, "out", &b.out, b.rows, c->head_dim)) return rc;
  if (b.out.type != b.q.type || b.out.heads != b.q.heads) return ops_fail(GG_E_ARG, "%s: out has another type or number of heads than q", fn);
  if (!b.cu_rows || !b.lens || !b.table) return ops_fail(GG_E_ARG, "%s: null array in the batch", fn);
  if (b.table_stride < ((long long)b.max_len + c->block_tokens - 1) / c->block_tokens)
    return ops_fail(GG_E_ARG, "%s: table_stride %lld holds fewer than max_len %d tokens", fn, (long long)b.table_stride, b.max_len);
  if (!(b.scale >= -1e30 && b.scale <= 1e30)) return ops_fail(GG_E_ARG, "%s: scale is not a number", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int rc = ops_check_stream(fn, s)) return rc;
  if (b.seqs == 0 || b.rows == 0 || b.max_rows == 0) return GG_OK;
  const Kv8Plan p = kv8_plan(*c, b);
  if (p.bytes && (!b.workspace || b.workspace_bytes < p.bytes || (uintptr_t)b.workspace & 15))
    return ops_fail(GG_E_ARG, "%s: needs %zu bytes of 16-byte aligned workspace, got %zu", fn, p.bytes, b.workspace ? b.workspace_bytes : (size_t)0);
  Kv8Args a = {};
  a.kc = static_cast<const uint8_t*>(c->k_codes);
  a.vc = static_cast<const uint8_t*>(c->v_codes);
  a.ks = c->k_scale;
  a.vs = c->v_scale;
  a.q = b.q.data;
  a.out = b.out.data;
  a.lse = b.lse;
  a.cu = b.cu_rows;
  a.lens = b.lens;
  a.table = b.table;
  a.table_stride = b.table_stride;
  a.q_row = b.q.row_stride;
  a.q_head = b.q.head_stride;
  a.o_row = b.out.row_stride;
  a.o_head = b.out.head_stride;
  a.scale_log2 = (float)(b.scale * 1.4426950408889634074);
  a.seqs = b.seqs;
  a.rows = b.rows;
  a.max_rows = b.max_rows;
  a.max_len = b.max_len;
  a.num_blocks = c->num_blocks;
  a.block_shift = __builtin_ctz(c->block_tokens);
  a.kv_heads = c->kv_heads;
  a.group = b.q.heads / c->kv_heads;
  a.hd = c->head_dim;
  a.window = b.window;
  a.q_type = b.q.type;
  a.q_vec = ops_aligned16(b.q);
  a.o_vec = ops_aligned16(b.out);
  cudaError_t r = cudaSuccess;
  for (int many = 0; many < 2 && r == cudaSuccess; many++) {
    const Kv8Cut& k = many ? p.many : p.few;
    if (!k.row_tiles) continue;
    a.row_tiles = k.row_tiles;
    a.splits = k.splits;
    a.split_steps = k.split_steps;
    a.items_lo = many ? KV8_FEW : 0;
    a.items_hi = many ? 0x7fffffff : KV8_FEW;
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(b.workspace) + (many ? p.few_bytes : 0));
    a.part_ml = reinterpret_cast<float2*>(a.part_o + k.parts * c->head_dim);
    r = many ? kv8_launch_prompt(a, c->code, s)
        : c->head_dim <= 64 ? launch_rows_hd<64>(a, c->code, s)
        : c->head_dim <= 128 ? launch_rows_hd<128>(a, c->code, s)
                             : launch_rows_hd<256>(a, c->code, s);
    if (r == cudaSuccess && k.splits > 1) {
      const long long tokens = many ? b.max_rows : (k.row_tiles * (long long)(b.q.type == GG_T_F32 ? 8 : 16) + a.group - 1) / a.group;
      a.merge_tokens = (int)(tokens < b.max_rows ? tokens : b.max_rows);
      r = launch_pdl(gg_kv8_merge_kernel, dim3((unsigned)(((long long)b.seqs * a.merge_tokens * b.q.heads + 3) / 4)), dim3(128), 0, s, a);
    }
  }
  if (r != cudaSuccess) return ops_fail(GG_E_CUDA, "%s: launch: %s", fn, cudaGetErrorString(r));
  return GG_OK;
}
