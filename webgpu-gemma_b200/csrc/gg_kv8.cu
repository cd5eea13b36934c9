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
// in one f16; their weights are rounded to f16 (2^-11 relative at most, and not all the same way; the
// output's own rounding is 2^-8 or 2^-11).
#include "gg_kv8.h"


namespace gg {

// ------------------------------------------------------------------------------ few rows
//
// A unit is one request, one key head and one tile of 8 NT query rows (the `group` heads of a few
// tokens); its keys are steps of 16 (one MMA's depth for the second product, never across a block).
// Each unit is cut into parts of nearly equal steps, one CTA each, so many that the resident CTAs
// fill the GPU once whatever the lengths of the requests are (only the device knows them: every CTA
// sums up the requests and finds its part). Bound by the cache's bytes. Each of the four warps
// streams its own steps through a private cp.async ring (no barriers between warps); the warps'
// results meet in shared memory at the end, the parts of a unit in gg_kv8_merge_kernel. Four requests
// of up to 131072 keys, 8 key heads of 128, bf16: 156 us, 6.0 TB/s of codes and scales; 64 requests of
// up to 8192 keys of one head of 256, f32: 39 us, 3.4 TB/s, of which the start, the first loads and
// the merge take about 15 and the SMs that hold three parts where others hold two some of the rest; one
// request of 641 keys: 10 us, all of it latency.
//
// Both products are transposed, so that the few query rows are the narrow side (N = 8) of an
// m16n8k16 MMA and the accumulators hold nothing else: S^T = K Q^T (16 keys x 8 rows), then
// O^T += V^T P^T (16 dims x 8 rows) -- half the registers and, for f16 and bf16, half the MMAs of
// rows padded to 16. f32 queries and weights take the hi and lo MMAs into the same accumulators.
//
// An MMA cuts the sum it adds to: measured, 0.9 2^-24 of it an MMA, always towards zero (f32 rows lost
// 1.1e-4 over 65536 uncut keys, 2.2e-4 over 131072). For f32 rows each step's two MMAs therefore start from
// zero, and their result is added to O with rounding (64 requests, f32, heads of 256: 39.3 us, 38.3 without). For
// f16 and bf16 rows, 4096 steps of a warp lose 2.2e-4, less than their own rounding, and a part has no
// more (KV8_LONGEST).
//
// Fragments (lane = 4 g + t): keys g and g + 8 of a step are read 16 dims (one 16-byte word) at a time,
// dims 64 j + 16 t .. + 15, whose four 4-byte parts are the operand values of four MMA depth steps;
// q is laid out to match. Weights leave S^T as (key g, rows 2t, 2t + 1) and movmatrix turns them to
// (row g, keys 2t, 2t + 1). For V the lane reads 16 dims of the keys 2t, 2t + 1, 2t + 8, 2t + 9: tile j of
// O^T has dims 16 g + 2 j and 16 g + 2 j + 1 as its rows g and g + 8. The 16-byte words of a key sit at
// swizzled places so that neither read has bank conflicts.
constexpr int KV8_WARPS = 4;
constexpr int KV8_STEP = 16;

template <int HD, bool HILO, int NT>
struct RowsShape {
  static constexpr int STAGES = HD == 256 ? 2 : HD == 128 ? 4 : 8;
  static constexpr int STAGE_BYTES = 2 * KV8_STEP * HD;
  static constexpr int QF_LANE = NT * (HILO ? 16 : 8);  // bytes of a lane's query operands in one depth step
  static constexpr int QF_BYTES = HD / 16 * 32 * QF_LANE;
  static constexpr int RING_BYTES = KV8_WARPS * STAGES * STAGE_BYTES;
  static constexpr int OST = HD + 4;                    // floats of a row of partial outputs
  static constexpr int OUT_BYTES = KV8_WARPS * 8 * NT * OST * 4;
  static constexpr int SMEM = QF_BYTES + RING_BYTES > OUT_BYTES ? QF_BYTES + RING_BYTES : OUT_BYTES;
  static constexpr int CTAS = NT * HD >= 512 ? 2 : 3;   // resident per SM
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
GG_DEV uint32_t transpose8x8(uint32_t x) {  // of f16 pairs: (row g, columns 2t, 2t + 1) -> (column g, rows 2t, 2t + 1)
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}

// Row tiles of a request (0: no rows) and steps of each (the same for its tiles).
struct Kv8Line {
  int tiles, steps, kmin;
};
GG_DEV Kv8Line kv8_line(const Kv8Args& a, const Kv8Seq& q, int RT) {
  Kv8Line n;
  n.tiles = (q.n * a.group + RT - 1) / RT;
  n.kmin = a.window ? (int)min(max(0ll, q.first_pos - a.window + 1), (long long)q.len) & ~(KV8_STEP - 1) : 0;
  n.steps = max(1, (q.len - n.kmin + KV8_STEP - 1) / KV8_STEP);  // a request without keys has one step that sees nothing
  return n;
}
// Steps of a part, for `total` steps in `units` units, so that the parts are not above the resident
// CTAs (a unit rounds its number of parts up): `share` of 0 to 4 quarters of the units counts the
// roundings; 4 is always enough. A step at least for each warp.
GG_DEV int kv8_part_steps(long long total, int units, int resident, int share) {
  if (resident == 0) return 1 << 29;  // units are not cut (steps stay below 2^28)
  const long long c = 2 * units <= resident ? (total + resident - 1) / (resident - share * units / 4) : (2 * total + resident - 1) / resident;
  return (int)min(max(c + 1, (long long)KV8_WARPS), (long long)KV8_LONGEST);
}

template <int HD, int CODE, bool HILO, int NT>
__global__ void __launch_bounds__(KV8_WARPS * 32, RowsShape<HD, HILO, NT>::CTAS) gg_kv8_rows_kernel(const Kv8Args a) {
  typedef RowsShape<HD, HILO, NT> S;
  constexpr int RT = 8 * NT, PER = 4, THREADS = KV8_WARPS * 32;
  extern __shared__ __align__(128) unsigned char kv8_smem[];
  __shared__ float s_mul[RT];
  __shared__ float2 s_ml[KV8_WARPS][RT];
  __shared__ int s_hi[RT];
  __shared__ long long s_sum[KV8_WARPS];
  __shared__ int s_units[KV8_WARPS], s_try[3][KV8_WARPS], s_seq, s_off;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  // ---- this CTA's part: all steps and units first, then the parts before each request
  int steps[PER], units[PER];
  const auto look = [&](int i0) {
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = i0 + tid * PER + k;
      steps[k] = 1;
      units[k] = 0;
      if (i < a.seqs) {
        const Kv8Line n = kv8_line(a, kv8_seq(a, i), RT);
        steps[k] = n.steps;
        units[k] = n.tiles * a.kv_heads;
      }
    }
  };
  long long total = 0;
  int all_units = 0;
  for (int i0 = 0; i0 < a.seqs; i0 += THREADS * PER) {
    look(i0);
#pragma unroll
    for (int k = 0; k < PER; k++) {
      total += (long long)steps[k] * units[k];
      all_units += units[k];
    }
  }
  // (a sum over the warp of numbers below 2^50, in two halves)
  total = (long long)__reduce_add_sync(0xffffffffu, (uint32_t)total & 0xffffffu) + ((long long)__reduce_add_sync(0xffffffffu, (uint32_t)(total >> 24)) << 24);
  all_units = __reduce_add_sync(0xffffffffu, all_units);
  if (lane == 0) {
    s_sum[warp] = total;
    s_units[warp] = all_units;
  }
  if (tid == 0) s_seq = -1;
  __syncthreads();
  total = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
  all_units = s_units[0] + s_units[1] + s_units[2] + s_units[3];
  int part_steps = kv8_part_steps(total, all_units, a.resident, 4);
  // the shortest parts that still fit one wave (sums by a rounded reciprocal: a part too many costs time, nothing else)
  if (a.resident && 2 * all_units <= a.resident && a.seqs <= THREADS * PER && total > (long long)a.resident * KV8_WARPS) {
    int n[3] = {0, 0, 0};
#pragma unroll
    for (int j = 0; j < 3; j++) {
      const int c = kv8_part_steps(total, all_units, a.resident, j + 1);
      const float inv = __fdividef(1.f, (float)c);
#pragma unroll
      for (int k = 0; k < PER; k++) n[j] += units[k] * (int)((float)(steps[k] + c - 1) * inv);
      n[j] = __reduce_add_sync(0xffffffffu, n[j]);
      if (lane == 0) s_try[j][warp] = n[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 2; j >= 0; j--)
      if (s_try[j][0] + s_try[j][1] + s_try[j][2] + s_try[j][3] <= a.resident) part_steps = kv8_part_steps(total, all_units, a.resident, j + 1);
  }
  const bool report = blockIdx.x == 0 && a.pre;  // the merge needs the sums too
  int run = 0;
  for (int i0 = 0; i0 < a.seqs; i0 += THREADS * PER) {
    __syncthreads();
    if (a.seqs > THREADS * PER) look(i0);
    int sum = 0, parts[PER];
#pragma unroll
    for (int k = 0; k < PER; k++) sum += parts[k] = units[k] * ((steps[k] + part_steps - 1) / part_steps);
    int inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += u;
    }
    if (lane == 31) s_units[warp] = inc;
    __syncthreads();
    int before = run + inc - sum;
    for (int w = 0; w < warp; w++) before += s_units[w];
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = i0 + tid * PER + k;
      if (report && i < a.seqs) a.pre[i] = before;
      if (before <= (int)blockIdx.x && (int)blockIdx.x < before + parts[k]) {
        s_seq = i;
        s_off = blockIdx.x - before;
      }
      before += parts[k];
    }
    run += s_units[0] + s_units[1] + s_units[2] + s_units[3];
    if (run > (int)blockIdx.x && !report) break;
  }
  if (report && tid == 0) a.pre[a.seqs] = part_steps;
  __syncthreads();
  const int s = s_seq;
  if (s < 0) return;  // more CTAs than parts
  const int heads = a.kv_heads * a.group;
  const Kv8Seq sq = kv8_seq(a, s);
  const Kv8Line ln = kv8_line(a, sq, RT);
  const int nparts = (ln.steps + part_steps - 1) / part_steps, unit = s_off / nparts, part = s_off % nparts;
  const int st0 = (int)((long long)ln.steps * part / nparts), st1 = (int)((long long)ln.steps * (part + 1) / nparts);
  const int h = unit / ln.tiles, base = (unit % ln.tiles) * RT;
  const bool whole = nparts == 1;
  const int32_t* table = a.table + (long long)s * a.table_stride;
  const int nitems = min(RT, sq.n * a.group - base), kmin = ln.kmin;
  const int first = st0 + warp;
  const int n = sq.len > kmin && st1 > first ? (st1 - first + KV8_WARPS - 1) / KV8_WARPS : 0;
  const auto step_key = [&](int i) { return kmin + (first + i * KV8_WARPS) * KV8_STEP; };

  // ---- the warp's ring
  unsigned char* ring = kv8_smem + S::QF_BYTES + warp * S::STAGES * S::STAGE_BYTES;
  const uint32_t ring_u = smem_u32(ring);
  const auto load_id = [&](int i) { return i < n ? table[step_key(i) >> a.block_shift] : -1; };
  const auto load_scales = [&](int id) {
    const bool in = id >= 0 && id < a.num_blocks;
    const long long at = (long long)(in ? id : 0) * a.kv_heads + h;
    return in ? make_float2(a.ks[at], a.vs[at]) : make_float2(0.f, 0.f);  // a scale of 0 marks a block the cache has not
  };
  int id_even = load_id(lane), id_odd = load_id(32 + lane);  // block ids of an even and of an odd batch of 32 steps, one step per lane
  // the warp's query rows, fetched while the ids are
  constexpr int QR = RT / KV8_WARPS, QP = (HD / 4 + 31) / 32;
  uint4 qv[QR][QP];
  load_raw4(qv, a.q, a.q_type, a.q_vec, [&](int j, int p) {
    const int row = warp + j * KV8_WARPS, it = base + row, tok = it / a.group, d = 4 * (lane + 32 * p);
    return row < nitems && d < a.hd ? (long long)(sq.row0 + tok) * a.q_row + (long long)(h * a.group + it - tok * a.group) * a.q_head + d : -1ll;
  });
  constexpr int W = HD / 16;  // 16-byte words of a key
  const int k_lane = lane / W, w_lane = lane % W;  // (a warp copies 32 / W keys at a time)
  const bool w_in = w_lane * 16 < a.hd;
  const auto issue = [&](int i) {
    if (i < n) {
      const int id = __shfl_sync(0xffffffffu, (i >> 5) & 1 ? id_odd : id_even, i & 31);
      const int key0 = step_key(i);
      const bool ok = w_in && id >= 0 && id < a.num_blocks;
      const long long at = (((long long)(ok ? id : 0) * a.kv_heads + h) << a.block_shift) + (key0 & ((1 << a.block_shift) - 1));
      const int left = ok ? sq.len - key0 : 0;  // keys of this step that exist
      const uint32_t dst = ring_u + (i % S::STAGES) * S::STAGE_BYTES;
      const long long off = at * a.hd + w_lane * 16;
#pragma unroll
      for (int c = 0; c < KV8_STEP * W / 32; c++) {
        const int k = k_lane + c * (32 / W);
        const uint32_t bytes = k < left ? 16 : 0;
        const long long src = k < left ? off + k * a.hd : 0;
        cp_async16(dst + kswz<HD>(k, w_lane), a.kc + src, bytes);
        cp_async16(dst + KV8_STEP * HD + vswz<HD>(k, w_lane), a.vc + src, bytes);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < S::STAGES - 1; i++) issue(i);
  float2 raw = load_scales(n ? id_even : -1);  // scales of the next batch of steps as the cache has them

  // ---- query rows -> f16 operand fragments
  unsigned char* qf = kv8_smem;
#pragma unroll
  for (int j = 0; j < QR; j++) {
    const int row = warp + j * KV8_WARPS;
    const bool live = row < nitems;
    float4 v[QP];
    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < QP; p++) {
      v[p] = widen_raw4(qv[j][p], a.q_type, a.q_vec);
      top = max(max(top, __float_as_uint(v[p].x) & 0x7fffffffu), __float_as_uint(v[p].y) & 0x7fffffffu);
      top = max(max(top, __float_as_uint(v[p].z) & 0x7fffffffu), __float_as_uint(v[p].w) & 0x7fffffffu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    const int ex = min(max((int)(top >> 23) - 127, -100), 127);
    const float up = __uint_as_float((uint32_t)(14 - ex + 127) << 23);
    if (lane == 0) {
      s_mul[row] = __uint_as_float((uint32_t)(ex - 14 + 127) << 23) * a.scale_log2;
      s_hi[row] = live ? (int)min(sq.first_pos + (base + row) / a.group, (long long)sq.len - 1) : -1;
    }
#pragma unroll
    for (int p = 0; p < QP; p++) {
      const int d = 4 * (lane + 32 * p);
      if (d >= HD) break;
      const int ks = 4 * (d >> 6) + ((d >> 2) & 3), tt = (d >> 4) & 3;
      uint32_t* f = reinterpret_cast<uint32_t*>(qf + ((ks * 32) + (row & 7) * 4 + tt) * S::QF_LANE) + (row >> 3) * (HILO ? 4 : 2);
      if constexpr (HILO) {
        split_f16(v[p].x * up, v[p].y * up, f[0], f[2]);
        split_f16(v[p].z * up, v[p].w * up, f[1], f[3]);
      } else {
        f[0] = half2_bits(v[p].x * up, v[p].y * up);
        f[1] = half2_bits(v[p].z * up, v[p].w * up);
      }
    }
  }
  __syncthreads();

  // ---- the lane's rows 2t and 2t + 1 of each tile of eight
  float mul[NT][2], rmax[NT][2], lsum[NT][2];
  int hi_key[NT][2], lo_key[NT][2];
#pragma unroll
  for (int u = 0; u < NT; u++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int row = 8 * u + 2 * t + e;
      mul[u][e] = s_mul[row];
      hi_key[u][e] = s_hi[row];
      lo_key[u][e] = a.window ? (int)max(0ll, sq.first_pos + (base + row) / a.group - a.window + 1) : 0;
      rmax[u][e] = KV8_NEG;
      lsum[u][e] = 0.f;
    }
  constexpr int OT = HD / 16;
  float o[NT][OT][4];
#pragma unroll
  for (int u = 0; u < NT; u++)
#pragma unroll
    for (int i = 0; i < OT; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) o[u][i][j] = 0.f;

  float b_ks = 0.f, b_lv = 0.f, b_iv = 0.f;
  const uint32_t qf_u = smem_u32(qf) + lane * S::QF_LANE;
  for (int i = 0; i < n; i++) {
    if ((i & 31) == 0) {  // this batch's scales: log2 and reciprocal once per step, a lane each
      b_ks = raw.x;
      b_lv = log2f(raw.y);
      b_iv = raw.y == 0.f ? 0.f : 1.f / raw.y;
    }
    cp_async_wait<S::STAGES - 2>();
    __syncwarp();
    issue(i + S::STAGES - 1);
    // the next batch: its ids once those of the batch before are used up, its scales a little later
    if ((i & 31) == 16 && i >= 32 && i + 16 < n) {
      const int id = load_id(i + 16 + lane);
      if ((i >> 5) & 1) id_even = id;
      else id_odd = id;
    }
    if ((i & 31) == 24) raw = load_scales(i + 8 + lane < n ? ((i >> 5) & 1 ? id_even : id_odd) : -1);
    const uint32_t kst = ring_u + (i % S::STAGES) * S::STAGE_BYTES, vst = kst + KV8_STEP * HD;
    const float ks = __shfl_sync(0xffffffffu, b_ks, i & 31), lv = __shfl_sync(0xffffffffu, b_lv, i & 31), iv = __shfl_sync(0xffffffffu, b_iv, i & 31);
    const int key0 = step_key(i);
    // scores, in two accumulators (hi and lo, or odd and even depth steps) to shorten the chains
    float c[NT][2][4] = {};
#pragma unroll
    for (int j = 0; j < HD / 64; j++) {
      const uint4 k0 = lds128(kst + kswz<HD>(g, 4 * j + t)), k1 = lds128(kst + kswz<HD>(g + 8, 4 * j + t));
      const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
      for (int p = 0; p < 4; p++) {
        uint4 ka;
        widen4<CODE>(w0[p], ka.x, ka.z);
        widen4<CODE>(w1[p], ka.y, ka.w);
        const uint32_t qa = qf_u + (4 * j + p) * 32 * S::QF_LANE;
#pragma unroll
        for (int u = 0; u < NT; u++) {
          if constexpr (HILO) {
            const uint4 q = lds128(qa + 16 * u);
            mma_f16(c[u][0], ka, q.x, q.y);
            mma_f16(c[u][1], ka, q.z, q.w);
          } else {
            const uint2 q = lds64(qa + 8 * u);
            mma_f16(c[u][p & 1], ka, q.x, q.y);
          }
        }
      }
    }
    // weights of rows 2t, 2t + 1 at keys key0 + g and key0 + g + 8
    uint32_t pb[NT][HILO ? 4 : 2];
#pragma unroll
    for (int u = 0; u < NT; u++) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const float f = ks * mul[u][e];  // (before it meets the sum: large keys may go with small queries)
        float sc[2], top = KV8_NEG;
        bool seen[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const int key = key0 + g + 8 * k;
          seen[k] = key <= hi_key[u][e] && key >= lo_key[u][e] && iv != 0.f;
          sc[k] = seen[k] ? fmaf(c[u][0][2 * k + e] + c[u][1][2 * k + e], f, lv) : KV8_NEG;
          top = fmaxf(top, sc[k]);
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (__any_sync(0xffffffffu, top > rmax[u][e] + KV8_SLACK)) {
          const float nr = top > rmax[u][e] + KV8_SLACK ? top : rmax[u][e];
          const float down = ex2(rmax[u][e] - nr);  // rmax = KV8_NEG: 2^-huge = 0
          rmax[u][e] = nr;
          lsum[u][e] *= down;
#pragma unroll
          for (int d = 0; d < OT; d++) {
            o[u][d][e] *= down;
            o[u][d][2 + e] *= down;
          }
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
          const float y = seen[k] ? ex2(sc[k] - rmax[u][e]) : 0.f;
          if (seen[k]) lsum[u][e] = fmaf(y, iv, lsum[u][e]);
          w[2 * k + e] = y * KV8_WMUL;
        }
      }
      if constexpr (HILO) {
        uint32_t hi0, lo0, hi1, lo1;
        split_f16(w[0], w[1], hi0, lo0);
        split_f16(w[2], w[3], hi1, lo1);
        pb[u][0] = transpose8x8(hi0);
        pb[u][1] = transpose8x8(hi1);
        pb[u][2] = transpose8x8(lo0);
        pb[u][3] = transpose8x8(lo1);
      } else {
        pb[u][0] = transpose8x8(half2_bits(w[0], w[1]));
        pb[u][1] = transpose8x8(half2_bits(w[2], w[3]));
      }
    }
    const auto product = [&](int tile, const uint32_t (&lo)[4], const uint32_t (&hi)[4]) {  // dims tile * 2 .. of keys 2t, 2t + 1 and 2t + 8, 2t + 9
#pragma unroll
      for (int y = 0; y < 2; y++) {
        const uint4 va = make_uint4(lo[2 * y], lo[2 * y + 1], hi[2 * y], hi[2 * y + 1]);
#pragma unroll
        for (int u = 0; u < NT; u++) {
          if constexpr (HILO) {
            float d[4];
            mma_f16_from_zero(d, va, pb[u][0], pb[u][1]);
            mma_f16(d, va, pb[u][2], pb[u][3]);
            add_f32x2(o[u][tile + y][0], o[u][tile + y][1], d[0], d[1]);
            add_f32x2(o[u][tile + y][2], o[u][tile + y][3], d[2], d[3]);
          } else {
            mma_f16(o[u][tile + y], va, pb[u][0], pb[u][1]);
          }
        }
      }
    };
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
          product(8 * jj + 2 * w, b0, b1);
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
        product(2 * w, b0, b1);
      }
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int u = 0; u < NT; u++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) lsum[u][e] += __shfl_xor_sync(0xffffffffu, lsum[u][e], d);
      if (g == 0) s_ml[warp][8 * u + 2 * t + e] = make_float2(rmax[u][e], lsum[u][e]);
    }
  __syncthreads();  // every warp has left its ring: it becomes [warp][row][OST] f32
  float* so = reinterpret_cast<float*>(kv8_smem);
  constexpr int PD = HD >= 128 ? 16 : 8;  // dims that a lane holds next to each other
#pragma unroll
  for (int u = 0; u < NT; u++)
#pragma unroll
    for (int e = 0; e < 2; e++) {
      if (8 * u + 2 * t + e >= nitems) continue;
      float* dst = so + (warp * RT + 8 * u + 2 * t + e) * S::OST + PD * g;
#pragma unroll
      for (int i = 0; i < OT; i += 2)
        *reinterpret_cast<float4*>(dst + (i * 2 / PD) * 128 + (i * 2) % PD) = make_float4(o[u][i][e], o[u][i][2 + e], o[u][i + 1][e], o[u][i + 1][2 + e]);
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
    const long long pi = (long long)blockIdx.x * RT + row;
    const float inv = whole ? (l == 0.f ? 0.f : (1.f / KV8_WMUL) / l) : 1.f / KV8_WMUL;
    for (int d = 4 * lane; d < a.hd; d += 128) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < KV8_WARPS; w++) {
        const float4 y = *reinterpret_cast<const float4*>(so + (w * RT + row) * S::OST + d);
        v.x = fmaf(f[w], y.x, v.x);
        v.y = fmaf(f[w], y.y, v.y);
        v.z = fmaf(f[w], y.z, v.z);
        v.w = fmaf(f[w], y.w, v.w);
      }
      v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
      if (whole) store_elem4(a.out, a.q_type, ri * a.o_row + (long long)hq * a.o_head + d, v, a.o_vec);
      else *reinterpret_cast<float4*>(a.part_o + pi * a.hd + d) = v;
    }
    if (lane == 0) {
      if (!whole) a.part_ml[pi] = make_float2(r, l);
      else if (a.lse) a.lse[ri * heads + hq] = l == 0.f ? -INFINITY : (r + log2f(l)) * 0.6931471805599453f;
    }
  }
}

// Where the parts of a row stand: of many rows its key ranges, of few rows the CTAs of its unit.
struct Kv8Parts {
  int n;
  long long first, step;
};
GG_DEV Kv8Parts kv8_parts(const Kv8Args& a, const Kv8Seq& sq, int s, int tok, int hq) {
  if (!a.pre) return {a.splits, ((long long)(sq.row0 + tok) * a.kv_heads * a.group + hq) * a.splits, 1};
  const int RT = a.tile_rows, item = tok * a.group + hq % a.group;
  const Kv8Line ln = kv8_line(a, sq, RT);
  const int n = (ln.steps + a.pre[a.seqs] - 1) / a.pre[a.seqs];
  return {n, ((long long)a.pre[s] + ((hq / a.group) * ln.tiles + item / RT) * n) * RT + item % RT, RT};
}
// One CTA per (request, token, query head): the results of the key ranges joined. Bound by latency
// (a few KB per CTA), so the ranges are spread over the threads: `lanes` threads hold four dims each
// and MERGE_THREADS / lanes of them share the ranges; every thread has its loads in flight at once.
constexpr int MERGE_THREADS = 256;
__global__ void __launch_bounds__(MERGE_THREADS) gg_kv8_merge_kernel(const Kv8Args a) {
  __shared__ float4 s_o[MERGE_THREADS];
  __shared__ float s_l[MERGE_THREADS / 32], s_r[MERGE_THREADS / 32];
  pdl_trigger();
  pdl_wait();
  const int t = threadIdx.x;
  const int heads = a.kv_heads * a.group;
  int x = blockIdx.x;
  const int hq = x % heads;
  x /= heads;
  const int tok = x % a.merge_tokens;
  x /= a.merge_tokens;
  const Kv8Seq sq = kv8_seq(a, x);
  if (tok >= sq.n) return;
  const long long ri = sq.row0 + tok;
  const Kv8Parts pt = kv8_parts(a, sq, x, tok, hq);
  const int nparts = pt.n;
  if (a.pre && nparts == 1) return;  // finished by its CTA
  const auto at = [&](int z) { return pt.first + z * pt.step; };
  float r = KV8_NEG;
  for (int z = t; z < nparts; z += MERGE_THREADS) r = fmaxf(r, a.part_ml[at(z)].x);
  const int lanes = a.hd <= 64 ? 16 : a.hd <= 128 ? 32 : 64, parts = MERGE_THREADS / lanes;
  const int d = 4 * (t % lanes), z0 = t / lanes;
  r = warp_max(r);
  if ((t & 31) == 0) s_r[t >> 5] = r;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < MERGE_THREADS / 32; w++) r = fmaxf(r, s_r[w]);
  float l = 0.f;
  for (int z = t; z < nparts; z += MERGE_THREADS) {
    const float2 ml = a.part_ml[at(z)];
    l = fmaf(ex2(ml.x - r), ml.y, l);
  }
  l = warp_sum(l);
  if ((t & 31) == 0) s_l[t >> 5] = l;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (d < a.hd)
#pragma unroll 4
    for (int z = z0; z < nparts; z += parts) {
      const float f = ex2(a.part_ml[at(z)].x - r);
      const float4 y = *reinterpret_cast<const float4*>(a.part_o + at(z) * a.hd + d);
      v.x = fmaf(f, y.x, v.x);
      v.y = fmaf(f, y.y, v.y);
      v.z = fmaf(f, y.z, v.z);
      v.w = fmaf(f, y.w, v.w);
    }
  s_o[t] = v;
  __syncthreads();
  if (t >= lanes || d >= a.hd) return;
  l = 0.f;
#pragma unroll
  for (int w = 0; w < MERGE_THREADS / 32; w++) l += s_l[w];
  for (int p = 1; p < parts; p++) {
    const float4 y = s_o[t + p * lanes];
    v = make_float4(v.x + y.x, v.y + y.y, v.z + y.z, v.w + y.w);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  store_elem4(a.out, a.q_type, ri * a.o_row + (long long)hq * a.o_head + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv), a.o_vec);
  if (t == 0 && a.lse) a.lse[ri * heads + hq] = l == 0.f ? -INFINITY : (r + log2f(l)) * 0.6931471805599453f;
}

// The same by one warp, for rows by the thousand with a few parts each: bound by the parts' bytes.
__global__ void __launch_bounds__(MERGE_THREADS) gg_kv8_merge_rows_kernel(const Kv8Args a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, heads = a.kv_heads * a.group;
  long long x = (long long)blockIdx.x * (MERGE_THREADS / 32) + (threadIdx.x >> 5);
  const int hq = (int)(x % heads);
  x /= heads;
  const int tok = (int)(x % a.merge_tokens);
  x /= a.merge_tokens;
  if (x >= a.seqs) return;
  const Kv8Seq sq = kv8_seq(a, (int)x);
  if (tok >= sq.n) return;
  const long long ri = sq.row0 + tok, p0 = (ri * heads + hq) * a.splits;
  float r = KV8_NEG, l = 0.f;
  for (int z = 0; z < a.splits; z++) r = fmaxf(r, a.part_ml[p0 + z].x);
  for (int z = 0; z < a.splits; z++) l = fmaf(ex2(a.part_ml[p0 + z].x - r), a.part_ml[p0 + z].y, l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int d = 4 * lane; d < a.hd; d += 128) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int z = 0; z < a.splits; z++) {
      const float f = ex2(a.part_ml[p0 + z].x - r);
      const float4 y = *reinterpret_cast<const float4*>(a.part_o + (p0 + z) * a.hd + d);
      v.x = fmaf(f, y.x, v.x);
      v.y = fmaf(f, y.y, v.y);
      v.z = fmaf(f, y.z, v.z);
      v.w = fmaf(f, y.w, v.w);
    }
    store_elem4(a.out, a.q_type, ri * a.o_row + (long long)hq * a.o_head + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv), a.o_vec);
  }
  if (lane == 0 && a.lse) a.lse[ri * heads + hq] = l == 0.f ? -INFINITY : (r + log2f(l)) * 0.6931471805599453f;
}

template <int HD, int CODE, bool HILO, int NT>
cudaError_t launch_rows(const Kv8Args& a, cudaStream_t s) {
  return launch_big_smem<gg_kv8_rows_kernel<HD, CODE, HILO, NT>>(dim3((unsigned)a.few_ctas), dim3(KV8_WARPS * 32), RowsShape<HD, HILO, NT>::SMEM, s, a);
}
template <int HD, int CODE, bool HILO>
cudaError_t launch_rows_nt(const Kv8Args& a, int nt, cudaStream_t s) {
  if (nt == 1) return launch_rows<HD, CODE, HILO, 1>(a, s);
  if constexpr (HD <= 128)
    if (nt == 4) return launch_rows<HD, CODE, HILO, 4>(a, s);
  return launch_rows<HD, CODE, HILO, 2>(a, s);
}
template <int HD>
cudaError_t launch_rows_hd(const Kv8Args& a, int code, int nt, cudaStream_t s) {
  const bool hilo = a.q_type == GG_T_F32;
  if (code == GG_KV8_INT8) return hilo ? launch_rows_nt<HD, GG_KV8_INT8, true>(a, nt, s) : launch_rows_nt<HD, GG_KV8_INT8, false>(a, nt, s);
  return hilo ? launch_rows_nt<HD, GG_KV8_E4M3, true>(a, nt, s) : launch_rows_nt<HD, GG_KV8_E4M3, false>(a, nt, s);
}
// Tiles of eight query rows of a CTA: as many as the call's requests can fill, within the registers
// (a tile more costs 2 head_dim / 16 MMAs a step, a CTA more reads the keys once more).
static int kv8_row_tiles(long long items, int head_dim) { return items <= 8 ? 1 : items <= 16 || head_dim > 128 ? 2 : 4; }

// How a call is cut. Requests with few rows (rows * group up to KV8_FEW) take the kernel above, the
// others the one of gg_kv8_prompt.cu; a call that may hold both launches both, and each skips the
// other's requests. Of calls that kv8_check lets through: seqs * max_rows * heads
// is below 2^31, so row_tiles fits an int.
constexpr int KV8_FEW = 32, KV8_WHOLE = 128 << 10;

struct Kv8Plan {
  // few rows: tiles of eight rows of a CTA, CTAs (-1: too many), how many the GPU holds (0: units are
  // not cut), rows of parts that they may leave
  int nt = 1, few_ctas = 0, resident = 0;
  size_t few_parts = 0;
  // many rows: row tiles of a request and head (0: not launched), key ranges, 16-key steps of a range
  int row_tiles = 0, splits = 1, split_steps = 1;
  size_t many_parts = 0;
  size_t few_bytes = 0, bytes = 0;
};
static Kv8Plan kv8_plan(const gg_kv8_cache& c, const gg_kv8_attention_call& b) {
  Kv8Plan p;
  if (!b.seqs || !b.max_rows) return p;
  const long long items = (long long)b.max_rows * (b.q.heads / c.kv_heads), few = items < KV8_FEW ? items : KV8_FEW;
  // keys that a tile may read: all, or its window with the rows between its first and last
  const auto steps = [&](long long tile) {
    long long keys = b.max_len;
    if (b.window && keys > (long long)b.window + tile + 2 * KV8_STEP) keys = (long long)b.window + tile + 2 * KV8_STEP;
    return (keys + KV8_STEP - 1) / KV8_STEP;
  };
  p.nt = kv8_row_tiles(few, c.head_dim);
  const int rt = 8 * p.nt, hd = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;
  const double units = (double)b.seqs * c.kv_heads * ((few + rt - 1) / rt), line = units * (steps(few) + 1);
  if (line + units >= 2147483647.0) return p.few_ctas = -1, p;
  // Units of at most KV8_WHOLE bytes of codes are not cut: reading them takes less than a second kernel.
  const bool cut = (double)(steps(few) + 1) * 2 * KV8_STEP * c.head_dim > KV8_WHOLE;
  p.resident = cut ? 148 * (p.nt * hd >= 512 ? 2 : 3) : 0;  // RowsShape::CTAS
  const double most = cut ? line / KV8_WARPS : 0;
  p.few_ctas = (int)((most < p.resident ? most : p.resident) + units + line / KV8_LONGEST) + 1;  // parts are at most that many
  p.few_parts = cut ? (size_t)p.few_ctas * rt : 0;
  // One CTA an SM; ranges of at least 512 keys where there are fewer tiles than SMs. Against 256 and 128, merge
  // included: 512 f32 rows of 4 heads over 1 of 256 at position 0 38.9 / 35.7 / 31.2 us, at 1536 45.1 / 40.2 / 44.2;
  // bf16, 32 heads over 8 of 128, 64 rows at 4000 34.2 / 35.1 / 37.1, 256 at 0 20.8 / 20.8 / 27.7, 16 at 2000
  // 27.4 / 24.1 / 23.1. (512 suits the bf16 prompts; f32 ones would gain from shorter ranges.)
  if (items > KV8_FEW) {
    const int tile = kv8_prompt_tile(c.head_dim);
    p.row_tiles = (int)((items + tile - 1) / tile);
    const long long units = (long long)b.seqs * c.kv_heads * p.row_tiles, n = steps(tile), most = (n + 31) / 32;
    long long splits = 148 / units;
    if (splits > most) splits = most;
    const long long least = b.q.type == GG_T_F32 ? 1 : (n + KV8_LONGEST - 1) / KV8_LONGEST;
    if (splits < least) splits = least;
    if (splits < 1) splits = 1;
    p.split_steps = (int)((n + splits - 1) / splits);
    if (p.split_steps < 1) p.split_steps = 1;
    p.splits = (int)((n + p.split_steps - 1) / p.split_steps);
    if (p.splits < 1) p.splits = 1;
    // room for the ranges before they are evened out: a longer max_len never needs less workspace
    if (splits > 1) p.many_parts = (size_t)b.rows * b.q.heads * splits;
  }
  // partial outputs, then their (r, l) pairs; few rows: then the line's prefix sums
  p.few_bytes = p.few_parts ? (p.few_parts * (c.head_dim * 4 + 8) + ((size_t)b.seqs + 1) * 4 + 15) / 16 * 16 : 0;
  p.bytes = p.few_bytes + p.many_parts * (c.head_dim * 4 + 8);
  return p;
}

static int kv8_check(const char* fn, const gg_kv8_cache* c, const gg_kv8_attention_call* b) {
  if (int rc = ops_check_cache(fn, c)) return rc;
  if (b->q.type < GG_T_F32 || b->q.type > GG_T_F16) return ops_fail(GG_E_ARG, "%s: q.type %d is none of GG_T_*", fn, b->q.type);
  if (b->q.heads < 1 || b->q.heads > 65535 || b->q.heads % c->kv_heads)
    return ops_fail(GG_E_ARG, "%s: %d query heads over %d key heads", fn, b->q.heads, c->kv_heads);
  if (b->q.heads / c->kv_heads > 1024) return ops_fail(GG_E_ARG, "%s: more than 1024 query heads to a key head", fn);
  if (b->seqs < 0 || b->rows < 0 || b->max_rows < 0 || b->max_len < 0)
    return ops_fail(GG_E_ARG, "%s: seqs %d, rows %d, max_rows %d, max_len %d out of range", fn, b->seqs, b->rows, b->max_rows, b->max_len);
  if (b->window < 0) return ops_fail(GG_E_ARG, "%s: window %d", fn, b->window);
  const bool rows_fit = (double)b->seqs * b->max_rows * b->q.heads < 2147483647.0;
  const Kv8Plan p = rows_fit ? kv8_plan(*c, *b) : Kv8Plan();
  if (!rows_fit || p.few_ctas < 0 || (double)b->seqs * c->kv_heads * p.row_tiles * p.splits >= 2147483647.0)
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
  return kv8_attention_bounded(c, call, static_cast<cudaStream_t>(stream), nullptr, KV8_TIMEOUT_NS);
}

int kv8_attention_bounded(const gg_kv8_cache* c, const gg_kv8_attention_call* call, cudaStream_t s, uint32_t* err, uint64_t timeout_ns) {
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
  a.err = err;
  a.timeout_ns = timeout_ns;
  cudaError_t r = cudaSuccess;
  const auto merge = [&](int tokens) {
    a.merge_tokens = tokens < b.max_rows ? tokens : b.max_rows;
    const long long n = (long long)b.seqs * a.merge_tokens * b.q.heads;
    // A CTA a row while they fit the GPU at once (148 SMs x 8). 35,776 rows of two parts took 102 us so;
    // a warp a row takes 9.7 us for 10,176 of them, but a chain of loads as long as the parts for a few.
    if (!a.pre && n > 148 * 8)
      return launch_pdl(gg_kv8_merge_rows_kernel, dim3((unsigned)((n + MERGE_THREADS / 32 - 1) / (MERGE_THREADS / 32))), dim3(MERGE_THREADS), 0, s, a);
    return launch_pdl(gg_kv8_merge_kernel, dim3((unsigned)((long long)b.seqs * a.merge_tokens * b.q.heads)), dim3(MERGE_THREADS), 0, s, a);
  };
  const auto parts = [&](size_t offset, size_t n) {
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(b.workspace) + offset);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + n * c->head_dim);
  };
  // requests with few rows
  a.items_lo = 0;
  a.items_hi = KV8_FEW;
  a.splits = 1;
  a.few_ctas = p.few_ctas;
  a.resident = p.resident;
  a.tile_rows = 8 * p.nt;
  parts(0, p.few_parts);
  a.pre = p.few_parts ? reinterpret_cast<int*>(a.part_ml + p.few_parts) : nullptr;
  r = c->head_dim <= 64 ? launch_rows_hd<64>(a, c->code, p.nt, s)
      : c->head_dim <= 128 ? launch_rows_hd<128>(a, c->code, p.nt, s)
                           : launch_rows_hd<256>(a, c->code, p.nt, s);
  if (r == cudaSuccess && p.few_parts) {  // no request has more than max_rows tokens
    const int most = (KV8_FEW + a.group - 1) / a.group;
    r = merge(b.max_rows < most ? b.max_rows : most);
  }
  // requests with many
  if (r == cudaSuccess && p.row_tiles) {
    a.items_lo = KV8_FEW;
    a.items_hi = 0x7fffffff;
    a.row_tiles = p.row_tiles;
    a.splits = p.splits;
    a.split_steps = p.split_steps;
    a.pre = nullptr;
    parts(p.few_bytes, p.many_parts);
    r = kv8_launch_prompt(a, c->code, s);
    if (r == cudaSuccess && p.splits > 1) r = merge(b.max_rows);
  }
  if (r != cudaSuccess) return ops_fail(GG_E_CUDA, "%s: launch: %s", fn, cudaGetErrorString(r));
  return GG_OK;
}
