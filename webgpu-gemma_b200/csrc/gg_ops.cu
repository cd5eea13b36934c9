// gg_ops.cu -- operators on device memory: block plans, rotary positions and the writing side of
// the paged 8-bit KV cache (the reading side is gg_kv8.cu).
#include <cuda_fp8.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include "gg_launch.h"
#include "gg_ops.h"

void gg_set_engineless_error(const char* msg);  // gg_engine.cu: the message gg_last_error(NULL) returns

int ops_fail(int code, const char* fmt, ...) {
  char buf[320];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  gg_set_engineless_error(buf);
  return code;
}

int ops_check_stream(const char* fn, cudaStream_t s) {
  if (!s) return GG_OK;
  // a capturing stream may not be asked for its device: a wrong one fails at the launch instead
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  cudaError_t r = cudaStreamIsCapturing(s, &cap);
  if (r != cudaSuccess) return ops_fail(GG_E_ARG, "%s: cudaStreamIsCapturing: %s", fn, cudaGetErrorString(r));
  if (cap != cudaStreamCaptureStatusNone) return GG_OK;
  int dev = -1, sdev = -1;
  r = cudaGetDevice(&dev);
  if (r != cudaSuccess) return ops_fail(GG_E_CUDA, "%s: cudaGetDevice: %s", fn, cudaGetErrorString(r));
  r = cudaStreamGetDevice(s, &sdev);
  if (r != cudaSuccess) return ops_fail(GG_E_ARG, "%s: cudaStreamGetDevice: %s", fn, cudaGetErrorString(r));
  if (sdev != dev) return ops_fail(GG_E_ARG, "%s: stream belongs to device %d, the current device is %d", fn, sdev, dev);
  return GG_OK;
}

int ops_check_rows(const char* fn, const char* name, const gg_rows* v, int rows, int head_dim) {
  if (!v->data) return ops_fail(GG_E_ARG, "%s: %s.data is null", fn, name);
  if (v->type < GG_T_F32 || v->type > GG_T_F16) return ops_fail(GG_E_ARG, "%s: %s.type %d is none of GG_T_*", fn, name, v->type);
  if (v->heads < 1 || v->heads > 65535) return ops_fail(GG_E_ARG, "%s: %s.heads %d outside 1..65535", fn, name, v->heads);
  if ((uintptr_t)v->data % ops_type_bytes(v->type)) return ops_fail(GG_E_ARG, "%s: %s.data is not aligned to its type", fn, name);
  if (v->row_stride < 0 || v->head_stride < 0) return ops_fail(GG_E_ARG, "%s: %s has a negative stride", fn, name);
  if (v->heads > 1 && v->head_stride < head_dim)
    return ops_fail(GG_E_ARG, "%s: the heads of %s overlap (head_stride %lld, head_dim %d)", fn, name, (long long)v->head_stride, head_dim);
  if (rows > 1 && v->row_stride < head_dim)
    return ops_fail(GG_E_ARG, "%s: the rows of %s overlap (row_stride %lld, head_dim %d)", fn, name, (long long)v->row_stride, head_dim);
  return GG_OK;
}

int ops_check_cache(const char* fn, const gg_kv8_cache* c) {
  if (!c->k_codes || !c->v_codes || !c->k_scale || !c->v_scale) return ops_fail(GG_E_ARG, "%s: null cache array", fn);
  if (((uintptr_t)c->k_codes | (uintptr_t)c->v_codes | (uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 15)
    return ops_fail(GG_E_ARG, "%s: the cache arrays must be 16-byte aligned", fn);
  if (c->block_tokens != 16 && c->block_tokens != 32 && c->block_tokens != 64 && c->block_tokens != 128)
    return ops_fail(GG_E_ARG, "%s: block_tokens %d is not 16, 32, 64 or 128", fn, c->block_tokens);
  if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16)
    return ops_fail(GG_E_ARG, "%s: head_dim %d is not a multiple of 16 up to 256", fn, c->head_dim);
  if (c->kv_heads < 1 || c->kv_heads > 1024) return ops_fail(GG_E_ARG, "%s: kv_heads %d outside 1..1024", fn, c->kv_heads);
  if (c->num_blocks < 1 || (long long)c->num_blocks * c->block_tokens >= (1ll << 31))
    return ops_fail(GG_E_ARG, "%s: num_blocks %d x block_tokens %d outside 1..2^31-1", fn, c->num_blocks, c->block_tokens);
  if (c->code != GG_KV8_INT8 && c->code != GG_KV8_E4M3) return ops_fail(GG_E_ARG, "%s: code %d is none of GG_KV8_*", fn, c->code);
  return GG_OK;
}

namespace gg {

// ------------------------------------------------------------------------------ block plan
//
// One CTA: the whole plan is a few prefix sums over the requests (blocks given back, blocks taken,
// new rows), so it is bound by the latency of its dependent steps -- lengths, scan, stack, table,
// rows -- and not by its bytes. The sums of up to PLAN_CHUNK requests stand in shared memory; blocks
// and rows are then spread one per thread and find their request by a binary search of them, so
// that one long prompt among many single tokens costs no more than the tokens themselves. More
// than PLAN_INLINE_ROWS rows are filled by gg_plan_rows_kernel over all SMs. Up to PLAN_CHUNK requests
// keep their lengths in registers (gg_plan_kernel, 256 threads where that many requests have one
// each: its barriers are cheaper); more go through the chunks three times (gg_plan_many_kernel).
// The code runs once, so instruction fetches count: with its loops unrolled by four 1000 requests
// with 32768 rows took 16.2 us, rolled and with warp reductions 10.8; 64 requests with one row each
// take 2.8 us (6.1 with the chunked kernel), most of it three dependent rounds of loads.
constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_CHUNK = 4096;
constexpr int PLAN_PER = PLAN_CHUNK / PLAN_THREADS;
constexpr int PLAN_INLINE_ROWS = 4096;

struct PlanScan {
  int give[PLAN_CHUNK + 1], take[PLAN_CHUNK + 1], rows[PLAN_CHUNK + 1];  // exclusive, within the chunk
  int warp[3][PLAN_THREADS / 32];
};

// Index i with pre[i] <= k < pre[i + 1] (pre ascending, n + 1 entries, pre[0] <= k < pre[n]).
GG_DEV int find_segment(const int* pre, int n, int k) {
  int lo = 0, hi = n;
#pragma unroll 1
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= k) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Slot of position pos in a block; -1 for an id that no cache has (below 0, or with slots beyond 31 bits).
GG_DEV int plan_slot(int id, int pos, int B) {
  const long long s = (long long)id * B + pos % B;
  return s >= 0 && s <= 0x7fffffff ? (int)s : -1;
}

GG_DEV int plan_blocks_of(int len, int B) { return len > 0 ? (int)((uint32_t)(len - 1) / (uint32_t)B) + 1 : 0; }

// Exclusive prefix sums of the chunk's requests i0 .. i0 + n - 1. Called with a plan that passed
// its checks: every sum fits 32 bits.
GG_DEV void plan_scan(const gg_block_plan& p, int i0, int n, PlanScan& sc) {
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  int v[3][PLAN_PER], sum[3] = {0, 0, 0};
#pragma unroll
  for (int k = 0; k < PLAN_PER; k++) {
    const int i = t * PLAN_PER + k;
    int a = 0, b = 0;
    if (i < n) { a = p.old_len[i0 + i]; b = p.new_len[i0 + i]; }
    const int d = plan_blocks_of(b, p.block_tokens) - plan_blocks_of(a, p.block_tokens);
    v[0][k] = max(-d, 0);
    v[1][k] = max(d, 0);
    v[2][k] = max(b - a, 0);
#pragma unroll
    for (int q = 0; q < 3; q++) sum[q] += v[q][k];
  }
  int inc[3];
#pragma unroll
  for (int q = 0; q < 3; q++) {
    inc[q] = sum[q];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc[q], o);
      if (lane >= o) inc[q] += u;
    }
    if (lane == 31) sc.warp[q][w] = inc[q];
  }
  __syncthreads();
  if (w < 3) {
    int x = sc.warp[w][lane];
    const int own = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += u;
    }
    sc.warp[w][lane] = x - own;
  }
  __syncthreads();
  int* const dst[3] = {sc.give, sc.take, sc.rows};
#pragma unroll
  for (int q = 0; q < 3; q++) {
    int run = sc.warp[q][w] + inc[q] - sum[q];
#pragma unroll
    for (int k = 0; k < PLAN_PER; k++) {
      const int i = t * PLAN_PER + k;
      if (i < n) dst[q][i] = run;
      run += v[q][k];
      if (i == n - 1) dst[q][n] = run;
    }
  }
  __syncthreads();
}

// Sum over the warp of numbers from 0 to 2^50, in two halves.
GG_DEV long long warp_add_long(long long v) {
  return (long long)__reduce_add_sync(0xffffffffu, (uint32_t)v & 0xffffffu) + ((long long)__reduce_add_sync(0xffffffffu, (uint32_t)(v >> 24)) << 24);
}

template <int THREADS, int PER>
__global__ void __launch_bounds__(THREADS) gg_plan_kernel(const gg_block_plan p, int inline_rows) {
  constexpr int WARPS = THREADS / 32;
  extern __shared__ __align__(16) unsigned char plan_smem[];
  PlanScan& sc = *reinterpret_cast<PlanScan*>(plan_smem);
  __shared__ long long s_long[3][WARPS];
  __shared__ uint32_t s_int[3][WARPS];
  __shared__ int s_bad[WARPS];
  pdl_trigger();
  pdl_wait();
  const int t = threadIdx.x, lane = t & 31, w = t >> 5, B = p.block_tokens, n = p.seqs;
  int a[PER], b[PER], flags = 0;
  uint32_t v[3][PER], sum[3] = {0, 0, 0};  // (these sums wrap only where the 64-bit ones refuse the plan)
  long long tot[3] = {0, 0, 0};
  const int count = *p.free_count;
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int i = t * PER + k;
    a[k] = i < n ? p.old_len[i] : 0;
    b[k] = i < n ? p.new_len[i] : 0;
  }
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int ha = plan_blocks_of(max(a[k], 0), B), hb = plan_blocks_of(max(b[k], 0), B);
    if (a[k] < 0 || b[k] < 0 || ha > p.max_blocks) flags |= GG_PLAN_BAD_LENGTH;
    if (hb > p.max_blocks) flags |= GG_PLAN_TOO_LONG;
    const long long d[3] = {max(ha - hb, 0), max(hb - ha, 0), max((long long)b[k] - a[k], 0ll)};
#pragma unroll
    for (int q = 0; q < 3; q++) {
      tot[q] += d[q];
      v[q][k] = (uint32_t)d[q];
      sum[q] += v[q][k];
    }
  }
  uint32_t inc[3];
#pragma unroll
  for (int q = 0; q < 3; q++) {
    inc[q] = sum[q];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, inc[q], o);
      if (lane >= o) inc[q] += u;
    }
    tot[q] = warp_add_long(tot[q]);
    if (lane == 31) {
      s_int[q][w] = inc[q];
      s_long[q][w] = tot[q];
    }
  }
  flags = __reduce_or_sync(0xffffffffu, flags);
  if (lane == 0) s_bad[w] = flags;
  __syncthreads();
  uint32_t before[3];
  flags = __reduce_or_sync(0xffffffffu, lane < WARPS ? s_bad[lane] : 0);
#pragma unroll
  for (int q = 0; q < 3; q++) {
    before[q] = __reduce_add_sync(0xffffffffu, lane < w ? s_int[q][lane] : 0u);
    tot[q] = warp_add_long(lane < WARPS ? s_long[q][lane] : 0);
  }
  if (count < 0 || count > p.free_capacity || count + tot[0] > p.free_capacity) flags |= GG_PLAN_BAD_STACK;
  else if (tot[1] > count + tot[0]) flags |= GG_PLAN_NO_BLOCKS;
  if (tot[2] > p.rows) flags |= GG_PLAN_NO_ROWS;
  const int given = flags ? 0 : (int)tot[0], taken = flags ? 0 : (int)tot[1], total = flags ? 0 : (int)tot[2];
  int* const dst[3] = {sc.give, sc.take, sc.rows};
#pragma unroll
  for (int q = 0; q < 3; q++) {
    uint32_t run = before[q] + inc[q] - sum[q];
#pragma unroll
    for (int k = 0; k < PER; k++) {
      const int i = t * PER + k;
      if (i < n) {
        dst[q][i] = (int)run;
        if (q == 2) {
          p.cu_rows[i] = flags ? 0 : (int)run;
          p.lens[i] = flags ? a[k] : b[k];
        }
      }
      run += v[q][k];
    }
  }
  if (t == 0) {
    *p.status = flags;
    *p.free_count_out = flags ? count : count + given - taken;
    p.cu_rows[n] = total;
    sc.give[n] = given;
    sc.take[n] = taken;
    sc.rows[n] = total;
  }
  __syncthreads();
  if (given > 0) {  // pushed above the current top, which this launch only reads below it
#pragma unroll 1
    for (int k = t; k < given; k += THREADS) {
      const int i = find_segment(sc.give, n, k);
      p.free_list[count + k] = p.table[(long long)i * p.table_stride + plan_blocks_of(p.new_len[i], B) + k - sc.give[i]];
    }
    __syncthreads();
  }
  if (taken > 0) {
#pragma unroll 1
    for (int k = t; k < taken; k += THREADS) {
      const int i = find_segment(sc.take, n, k);
      p.table[(long long)i * p.table_stride + plan_blocks_of(p.old_len[i], B) + k - sc.take[i]] = p.free_list[count + given - 1 - k];
    }
    __syncthreads();  // the rows below read the table entries written above
  }
  if (inline_rows) {
#pragma unroll 1
    for (int r = t; r < total; r += THREADS) {
      const int i = find_segment(sc.rows, n, r), pos = p.old_len[i] + r - sc.rows[i];
      p.row_seq[r] = i;
      p.positions[r] = pos;
      p.slots[r] = plan_slot(p.table[(long long)i * p.table_stride + pos / B], pos, B);
    }
    for (int r = total + t; r < p.rows; r += THREADS) p.row_seq[r] = p.positions[r] = p.slots[r] = -1;
  }
}

__global__ void __launch_bounds__(PLAN_THREADS) gg_plan_many_kernel(const gg_block_plan p, int inline_rows) {
  extern __shared__ __align__(16) unsigned char plan_smem[];
  PlanScan& sc = *reinterpret_cast<PlanScan*>(plan_smem);
  __shared__ long long s_sum[3][PLAN_THREADS / 32];
  __shared__ int s_flags;
  __shared__ long long s_tot[3];
  pdl_trigger();
  pdl_wait();
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int B = p.block_tokens;
  if (t == 0) s_flags = 0;
  __syncthreads();
  // totals and checks, in 64 bits
  long long tot[3] = {0, 0, 0};
  int flags = 0;
  for (int i = t; i < p.seqs; i += PLAN_THREADS) {
    const int a = p.old_len[i], b = p.new_len[i];
    const int ha = plan_blocks_of(max(a, 0), B), hb = plan_blocks_of(max(b, 0), B);
    if (a < 0 || b < 0 || ha > p.max_blocks) flags |= GG_PLAN_BAD_LENGTH;
    if (hb > p.max_blocks) flags |= GG_PLAN_TOO_LONG;
    tot[0] += max(ha - hb, 0);
    tot[1] += max(hb - ha, 0);
    tot[2] += max((long long)b - a, 0ll);
  }
#pragma unroll
  for (int q = 0; q < 3; q++) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tot[q] += __shfl_xor_sync(0xffffffffu, tot[q], o);
    if (lane == 0) s_sum[q][w] = tot[q];
  }
  if (flags) atomicOr(&s_flags, flags);
  const int count = *p.free_count;
  __syncthreads();
  if (w < 3) {
    long long x = s_sum[w][lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (lane == 0) s_tot[w] = x;
  }
  __syncthreads();
  flags = s_flags;
  if (count < 0 || count > p.free_capacity || count + s_tot[0] > p.free_capacity) flags |= GG_PLAN_BAD_STACK;
  else if (s_tot[1] > count + s_tot[0]) flags |= GG_PLAN_NO_BLOCKS;
  if (s_tot[2] > p.rows) flags |= GG_PLAN_NO_ROWS;
  const int given = (int)s_tot[0], taken = (int)s_tot[1], total = flags ? 0 : (int)s_tot[2];
  if (t == 0) *p.status = flags;
  const int chunks = (p.seqs + PLAN_CHUNK - 1) / PLAN_CHUNK;
  if (flags) {
    for (int i = t; i < p.seqs; i += PLAN_THREADS) {
      p.lens[i] = p.old_len[i];
      p.cu_rows[i] = 0;
    }
    if (t == 0) p.cu_rows[p.seqs] = 0;
  } else {
    // blocks given back: pushed above the current top, which this launch only reads below it
    if (given > 0) {
      int base = count;
      for (int c = 0; c < chunks; c++) {
        const int i0 = c * PLAN_CHUNK, n = min(PLAN_CHUNK, p.seqs - i0);
        plan_scan(p, i0, n, sc);
        for (int k = t; k < sc.give[n]; k += PLAN_THREADS) {
          const int i = find_segment(sc.give, n, k);
          const int b = plan_blocks_of(p.new_len[i0 + i], B) + k - sc.give[i];
          p.free_list[base + k] = p.table[(long long)(i0 + i) * p.table_stride + b];
        }
        base += sc.give[n];
        __syncthreads();
      }
    }
    int base_take = 0, base_rows = 0;
    const int top = count + given - 1;
    for (int c = 0; c < chunks; c++) {
      const int i0 = c * PLAN_CHUNK, n = min(PLAN_CHUNK, p.seqs - i0);
      plan_scan(p, i0, n, sc);
      for (int i = t; i < n; i += PLAN_THREADS) {
        p.lens[i0 + i] = p.new_len[i0 + i];
        p.cu_rows[i0 + i] = base_rows + sc.rows[i];
      }
      for (int k = t; k < sc.take[n]; k += PLAN_THREADS) {
        const int i = find_segment(sc.take, n, k);
        const int b = plan_blocks_of(p.old_len[i0 + i], B) + k - sc.take[i];
        p.table[(long long)(i0 + i) * p.table_stride + b] = p.free_list[top - (base_take + k)];
      }
      __syncthreads();  // the rows below read the table entries written above
      if (inline_rows)
        for (int r = t; r < sc.rows[n]; r += PLAN_THREADS) {
          const int i = find_segment(sc.rows, n, r);
          const int pos = p.old_len[i0 + i] + r - sc.rows[i];
          p.row_seq[base_rows + r] = i0 + i;
          p.positions[base_rows + r] = pos;
          p.slots[base_rows + r] = plan_slot(p.table[(long long)(i0 + i) * p.table_stride + pos / B], pos, B);
        }
      base_take += sc.take[n];
      base_rows += sc.rows[n];
      __syncthreads();
    }
    if (t == 0) p.cu_rows[p.seqs] = total;
  }
  if (t == 0) *p.free_count_out = flags ? count : count + given - taken;
  if (inline_rows)
    for (int r = total + t; r < p.rows; r += PLAN_THREADS) p.row_seq[r] = p.positions[r] = p.slots[r] = -1;
}

template <void (*Kernel)(const gg_block_plan, int)>
using PlanKernel = std::integral_constant<void (*)(const gg_block_plan, int), Kernel>;

// The row arrays of a large plan, one row per thread (after gg_plan_kernel).
constexpr int PLAN_ROWS_SMEM = 8192;  // requests whose cu_rows fit this kernel's shared memory
__global__ void __launch_bounds__(256) gg_plan_rows_kernel(const gg_block_plan p) {
  __shared__ int cu[PLAN_ROWS_SMEM + 1];
  pdl_trigger();
  pdl_wait();
  const int total = p.cu_rows[p.seqs];
  const bool in_smem = p.seqs <= PLAN_ROWS_SMEM;
  if (in_smem && (int)(blockIdx.x * blockDim.x) < total)
    for (int i = threadIdx.x; i <= p.seqs; i += blockDim.x) cu[i] = p.cu_rows[i];
  __syncthreads();
  const int* pre = in_smem ? cu : p.cu_rows;
  const int B = p.block_tokens;
  for (long long rr = blockIdx.x * (long long)blockDim.x + threadIdx.x; rr < p.rows; rr += (long long)gridDim.x * blockDim.x) {
    const int r = (int)rr;
    int seq = -1, pos = -1, slot = -1;
    if (r < total) {
      seq = find_segment(pre, p.seqs, r);
      pos = p.old_len[seq] + r - pre[seq];
      slot = plan_slot(p.table[(long long)seq * p.table_stride + pos / B], pos, B);
    }
    p.row_seq[r] = seq;
    p.positions[r] = pos;
    p.slots[r] = slot;
  }
}

// ------------------------------------------------------------------------------ rotary positions
//
// (a, b) -> (a c - b s, b c + a s). Bound by its bytes (each value read and written once). A CTA
// takes a few rows: it forms their (c, s) once in shared memory -- the angle p w in f64 turns,
// reduced to [-1/2, 1/2] before the f32 sincospi, because p w of a far position has no correct
// digits left in f32 -- and applies them to every head of q and k. 8192 rows of 40 heads of 128 in
// bf16: 31.0 us, 5.4 TB/s; 64 rows of 5 heads of 256 in f32: 2.0 us, one round of loads after a launch.
// 2047 rows of 32 heads of 96, interleaved f16: 8.5 us, 3.0 TB/s -- the loads of q and k stand behind the
// barrier that ends the sincospi.
constexpr int ROPE_THREADS = 256;
constexpr int ROPE_CS = 1024;  // (c, s) pairs in shared memory

struct RopeView {
  const void* in;
  void* out;
  long long in_row, in_head, out_row, out_head;
};
struct RopeArgs {
  RopeView q, k;
  const int32_t* pos;
  const double* freqs;
  double mscale;
  int rows, q_heads, heads, hd, rot, rows_per_cta, inverse, interleaved;
};

// Explicit roundings: the result does not depend on which variant of the kernel ran.
GG_DEV void turn(float p, float q, float2 m, float& x, float& y) {
  x = __fmaf_rn(p, m.x, -__fmul_rn(q, m.y));
  y = __fmaf_rn(q, m.x, __fmul_rn(p, m.y));
}

// V consecutive values of a unit: HALF: V values from i and their V partners from i + rot / 2,
// interleaved: V consecutive values (V / 2 pairs; V = 1 stands for one pair). Values behind rot
// are copied V (or 1) at a time.
template <class T, int V, bool INTER>
__global__ void __launch_bounds__(ROPE_THREADS) gg_rope_kernel(const RopeArgs a) {
  __shared__ float2 cs[ROPE_CS];
  pdl_trigger();
  pdl_wait();
  constexpr bool VEC = V > 1;
  constexpr int PER = INTER && !VEC ? 2 : V;  // values of a turned unit (one side of it for HALF)
  const int half = a.rot / 2;
  const int row0 = blockIdx.x * a.rows_per_cta;
  const int nrows = min(a.rows_per_cta, a.rows - row0);
  for (int i = threadIdx.x; i < nrows * half; i += ROPE_THREADS) {
    const int r = i / half, j = i - r * half;
    const int p = a.pos[row0 + r];
    float2 v = make_float2(1.f, 0.f);
    if (p >= 0) {
      const double turns = (double)p * (a.freqs[j] * 0.15915494309189533577);
      const float x = 2.f * (float)(turns - rint(turns));
      float s, c;
      sincospif(x, &s, &c);
      v = make_float2((float)(c * a.mscale), (float)((a.inverse ? -s : s) * a.mscale));
    }
    cs[i] = v;
  }
  __syncthreads();
  const int turned = (INTER ? a.rot : half) / PER;            // turned units of a head
  const int units = turned + (a.hd - a.rot) / V;              // and copied ones behind them
  const int per_row = units * a.heads;
  for (int i = threadIdx.x; i < nrows * per_row; i += ROPE_THREADS) {
    const int r = i / per_row, hu = i - r * per_row;
    const int h = hu / units, u = hu - h * units;
    const bool is_q = h < a.q_heads;
    const RopeView& w = is_q ? a.q : a.k;
    const int hh = is_q ? h : h - a.q_heads;
    const T* in = static_cast<const T*>(w.in) + (long long)(row0 + r) * w.in_row + (long long)hh * w.in_head;
    T* out = static_cast<T*>(w.out) + (long long)(row0 + r) * w.out_row + (long long)hh * w.out_head;
    if (u >= turned) {
      if (in == out) continue;
      const int at = a.rot + (u - turned) * V;
      float x[V];
      load_row<T, V, VEC>(in + at, x);
      store_row<T, V, VEC>(out + at, x);
      continue;
    }
    const float2* c = cs + r * half;
    const bool still = a.pos[row0 + r] < 0;
    if constexpr (INTER) {
      float x[PER];
      load_row<T, PER, VEC>(in + u * PER, x);
      if (!still)
#pragma unroll
        for (int j = 0; j < PER / 2; j++) {
          const float2 m = c[u * (PER / 2) + j];
          const float p = x[2 * j], q = x[2 * j + 1];
          turn(p, q, m, x[2 * j], x[2 * j + 1]);
        }
      store_row<T, PER, VEC>(out + u * PER, x);
    } else {
      float x[V], y[V];
      load_row<T, V, VEC>(in + u * V, x);
      load_row<T, V, VEC>(in + half + u * V, y);
      if (!still)
#pragma unroll
        for (int j = 0; j < V; j++) {
          const float2 m = c[u * V + j];
          const float p = x[j], q = y[j];
          turn(p, q, m, x[j], y[j]);
        }
      store_row<T, V, VEC>(out + u * V, x);
      store_row<T, V, VEC>(out + half + u * V, y);
    }
  }
}

template <class T>
cudaError_t launch_rope(const RopeArgs& a, bool vec, cudaStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  const int half = a.rot / 2;
  const bool fits = vec && (a.interleaved ? a.rot : half) % V == 0 && (a.hd - a.rot) % V == 0;
  const dim3 grid((a.rows + a.rows_per_cta - 1) / a.rows_per_cta), block(ROPE_THREADS);
  if (a.interleaved) return fits ? launch_pdl(gg_rope_kernel<T, V, true>, grid, block, 0, s, a) : launch_pdl(gg_rope_kernel<T, 1, true>, grid, block, 0, s, a);
  return fits ? launch_pdl(gg_rope_kernel<T, V, false>, grid, block, 0, s, a) : launch_pdl(gg_rope_kernel<T, 1, false>, grid, block, 0, s, a);
}

// ------------------------------------------------------------------------------ append
//
// Code and scale of a block: e = min{e >= -60 : max |x| <= Q 2^e}, code = rne(x 2^-e), Q = 127 or
// 448. Bound by its bytes: the new rows read once, a byte per value written. The CTA that finds
// the first row of a block's run takes the whole run, so the block's scale needs no atomics and
// no second launch: one pass for the largest value, one that rounds (the rows stay in registers, as
// they were read; what long runs have above that comes from L1/L2 again). 6300 rows of 8 heads of 128,
// bf16 to e4m3: 11.5 us, 3.4 TB/s (39 us with a search for each row's run and maxima one value at a
// time; 10.8 where skipped rows end a run, but then a block could have two); 64 rows of one head of 256,
// f32 to int8: 2.7 us, all latency.
constexpr int APPEND_THREADS = 128;
constexpr int APPEND_GAP = 128;  // rows of a block stand fewer than this apart, as the tokens of the largest block do
constexpr int KV8_MIN_EXP = -60;

// Smallest e >= KV8_MIN_EXP with |x| <= Q 2^e; bits = the pattern of a finite |x|.
template <int CODE>
GG_DEV int kv8_exponent(uint32_t bits) {
  const int x = (int)(bits >> 23) - 127;
  const uint32_t m = bits & 0x7fffffu;
  // 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8
  const int e = CODE == GG_KV8_INT8 ? x - 6 + (m > 0x7e0000u) : x - 8 + (m > 0x600000u);
  return max(e, KV8_MIN_EXP);  // zero and subnormal values (x = -127) end here too
}
// 2^e for -127 <= e <= 127
GG_DEV float pow2i(int e) { return __uint_as_float(e < -126 ? 0x00400000u : (uint32_t)(e + 127) << 23); }

// Eight values already divided by the scale -> eight codes.
template <int CODE>
GG_DEV uint2 kv8_encode8(const float (&x)[8]) {
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; j++) {
    if constexpr (CODE == GG_KV8_INT8) {
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; i++) b[i] = (uint32_t)__float2int_rn(x[4 * j + i]) & 0xffu;
      w[j] = b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24);
    } else {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * j], x[4 * j + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * j + 2], x[4 * j + 3]), __NV_SATFINITE, __NV_E4M3);
      w[j] = lo | (hi << 16);
    }
  }
  return make_uint2(w[0], w[1]);
}
// One code times 2^-d, rounded to a code again.
template <int CODE>
GG_DEV uint2 kv8_rescale8(uint2 w, float f) {
  float x[8];
  const uint32_t u[2] = {w.x, w.y};
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const uint32_t b = (u[i >> 2] >> (8 * (i & 3))) & 0xffu;
    if constexpr (CODE == GG_KV8_INT8) x[i] = (float)(int8_t)b * f;
    else x[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3))) * f;
  }
  return kv8_encode8<CODE>(x);
}

struct AppendArgs {
  const void* x[2];  // k, v
  uint8_t* codes[2];
  float* scale[2];
  long long row[2], head[2];
  const int32_t* slots;
  int rows, num_slots, block_shift, heads, hd, rows_per_cta;
};

// Eight values of a row as they were read, widened when they are used.
template <class T, bool VEC>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
  GG_DEV void load(const T* p) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; i++) w[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      T* e = reinterpret_cast<T*>(w);
#pragma unroll
      for (int i = 0; i < 8; i++) e[i] = p[i];
    }
  }
  GG_DEV void get(float (&v)[8]) const {
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = to_f32(e[i]);
  }
  // The largest |pattern| so far, of a 16-bit type two at a time; NaN is above all.
  GG_DEV void raise(uint32_t& m) const {
    const uint32_t* e = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
    for (int i = 0; i < 2 * (int)sizeof(T); i++)
      m = sizeof(T) == 2 ? __vmaxu2(m, e[i] & 0x7fff7fffu) : max(m, e[i] & 0x7fffffffu);
  }
};
// The same as the pattern of an f32.
template <class T>
GG_DEV uint32_t top_pattern(uint32_t m) {
  if constexpr (sizeof(T) == 4) return m;
  const uint16_t u = (uint16_t)max(m & 0xffffu, m >> 16);
  return __float_as_uint(to_f32(*reinterpret_cast<const T*>(&u)));
}

template <class T, int CODE, bool VEC>
__global__ void __launch_bounds__(APPEND_THREADS) gg_append_kernel(const AppendArgs a) {
  constexpr int KEEP = 16 / (int)sizeof(T);  // groups of eight values a thread keeps between the two passes
  __shared__ uint32_t s_max;
  pdl_trigger();
  pdl_wait();
  const int t = threadIdx.x, lane = t & 31;
  const int h = blockIdx.y >> 1, which = blockIdx.y & 1;
  const int B = 1 << a.block_shift;
  const int groups = a.hd / 8;
  const uint32_t gmagic = (65536u + groups - 1) / groups;  // i / groups for i < 2048
  const T* x = static_cast<const T*>(which ? a.x[1] : a.x[0]) + (long long)h * (which ? a.head[1] : a.head[0]);
  const long long xrow = which ? a.row[1] : a.row[0];
  const auto slot_of = [&](int r) { const int s = r >= 0 && r < a.rows ? a.slots[r] : -1; return s >= 0 && s < a.num_slots ? s : -1; };
  // the rows of this CTA's tile (at most 32) that begin a block's run; the others belong to earlier ones
  const int r0 = blockIdx.x * a.rows_per_cta;
  const int s_here = lane < a.rows_per_cta ? slot_of(r0 + lane) : -1, s_prev = slot_of(r0 + lane - 1);
  uint32_t leaders = __ballot_sync(0xffffffffu, s_here >= 0 && (s_prev < 0 || (s_prev >> a.block_shift) != (s_here >> a.block_shift)));
  // The nearest row with a slot among the APPEND_GAP - 1 from r on (step 1) or back from r (step -1): its
  // distance from r, or -1, and its slot.
  const auto nearest = [&](int r, int step, int& slot) {
    int s[APPEND_GAP / 32];
#pragma unroll
    for (int c = 0; c < APPEND_GAP / 32; c++) s[c] = 32 * c + lane < APPEND_GAP - 1 ? slot_of(r + step * (32 * c + lane)) : -1;
    int at = -1;
#pragma unroll
    for (int c = APPEND_GAP / 32 - 1; c >= 0; c--) {
      const uint32_t in = __ballot_sync(0xffffffffu, s[c] >= 0);
      if (!in) continue;
      at = 32 * c + __ffs(in) - 1;
      slot = __shfl_sync(0xffffffffu, s[c], at & 31);
    }
    return at;
  };
  for (; leaders; leaders &= leaders - 1) {
    const int r = r0 + __ffs(leaders) - 1;
    const int s0 = __shfl_sync(0xffffffffu, s_here, r - r0);
    const int blk = s0 >> a.block_shift;
    // behind skipped rows: the continuation of an earlier row's run?
    int other = -1;
    if (r > 0 && __shfl_sync(0xffffffffu, s_prev, r - r0) < 0 && nearest(r - 1, -1, other) >= 0 && other >> a.block_shift == blk) continue;
    // the run: rows r .. r + m - 1, of this block or skipped; each warp finds it alone
    int m = 0, first = B;
    bool ascending = true;
    for (;;) {
      const int s = slot_of(r + m + lane);
      const bool in = s >= 0 && (s >> a.block_shift) == blk;
      const uint32_t out = __ballot_sync(0xffffffffu, !in);
      const int n = out ? __ffs(out) - 1 : 32;
      first = min(first, (int)__reduce_min_sync(0xffffffffu, lane < n ? (uint32_t)(s & (B - 1)) : (uint32_t)B));
      ascending &= __all_sync(0xffffffffu, lane >= n || s == s0 + m + lane);
      const int seen = m + 32;
      m += n;
      if (n == 32) continue;
      // ended by a row of another block or the last row; behind skipped rows the block may go on
      if (r + m >= a.rows || __shfl_sync(0xffffffffu, s, n) >= 0) break;
      if (r + seen >= a.rows && !(__ballot_sync(0xffffffffu, s >= 0) >> n)) break;
      const int ahead = nearest(r + m, 1, other);
      if (ahead < 0 || other >> a.block_shift != blk) break;
      m += ahead;
      ascending = false;
    }
    const auto row_of = [&](int i) { return i < 2048 ? (int)((i * gmagic) >> 16) : i / groups; };
    const auto fetch = [&](int i, Raw8<T, VEC>& v) {
      const int j = row_of(i);
      v.load(x + (long long)(r + j) * xrow + (i - j * groups) * 8);
    };
    // skipped, or not the last of the rows with its slot (a run in ascending order has no such rows)
    const auto replaced = [&](int j) {
      const int s = slot_of(r + j);
      if (s < 0) return true;
      for (int k = j + 1; k < m; k++)
        if (a.slots[r + k] == s) return true;
      return false;
    };
    if (t == 0) s_max = 0;
    __syncthreads();
    const int items = m * groups;
    float* scale = (which ? a.scale[1] : a.scale[0]) + (long long)blk * a.heads + h;
    const float before = first > 0 ? *scale : 0.f;
    Raw8<T, VEC> keep[KEEP];
    uint32_t top = 0;
    if (ascending) {
#pragma unroll
      for (int k = 0; k < KEEP; k++)
        if (t + k * APPEND_THREADS < items) fetch(t + k * APPEND_THREADS, keep[k]);
#pragma unroll
      for (int k = 0; k < KEEP; k++)
        if (t + k * APPEND_THREADS < items) keep[k].raise(top);
    }
#pragma unroll 1
    for (int i = t + (ascending ? KEEP * APPEND_THREADS : 0); i < items; i += APPEND_THREADS) {
      Raw8<T, VEC> v;
      fetch(i, v);
      if (ascending || !replaced(row_of(i))) v.raise(top);
    }
    top = __reduce_max_sync(0xffffffffu, top_pattern<T>(top));
    if (lane == 0 && top) atomicMax(&s_max, top);
    __syncthreads();  // (everyone has read the old scale, too)
    top = s_max;
    bool finite = top < 0x7f800000u;
    int e = finite ? kv8_exponent<CODE>(top) : 0;
    float shrink = 1.f;  // what the codes of earlier tokens are multiplied by
    if (first > 0) {
      const uint32_t ob = __float_as_uint(before);
      // the smallest exponent that holds the old scale, which need not be a power of two; 128 where no
      // f32 does (or the block was poisoned before)
      const int old = (int)(ob >> 23) - 127 + ((ob & 0x7fffffu) != 0);
      if (old > 127) finite = false;
      if (finite) {
        e = max(e, old);
        shrink = before * pow2i(-e);  // exact, or 0 where every code becomes 0
      }
    }
    if (t == 0) *scale = finite ? pow2i(e) : __uint_as_float(0x7fffffffu);
    uint8_t* codes = (which ? a.codes[1] : a.codes[0]) + ((long long)blk * a.heads + h) * B * a.hd;
    if (shrink != 1.f)
#pragma unroll 1
      for (int i = t; i < first * groups; i += APPEND_THREADS) {
        uint2* w = reinterpret_cast<uint2*>(codes) + i;
        *w = kv8_rescale8<CODE>(*w, shrink);
      }
    const float inv = pow2i(-e);
    const auto encode = [&](const Raw8<T, VEC>& raw) {
      float y[8];
      raw.get(y);
#pragma unroll
      for (int q = 0; q < 8; q++) y[q] *= inv;
      return finite ? kv8_encode8<CODE>(y) : make_uint2(0, 0);
    };
    uint2* dst = reinterpret_cast<uint2*>(codes);
    if (ascending) {
      // consecutive rows fill consecutive slots: item i of the run is item i of the block from its first slot on
#pragma unroll
      for (int k = 0; k < KEEP; k++)
        if (t + k * APPEND_THREADS < items) dst[first * groups + t + k * APPEND_THREADS] = encode(keep[k]);
    }
#pragma unroll 1
    for (int i = t + (ascending ? KEEP * APPEND_THREADS : 0); i < items; i += APPEND_THREADS) {
      const int j = row_of(i);
      if (!ascending && replaced(j)) continue;
      Raw8<T, VEC> v;
      fetch(i, v);
      dst[(ascending ? first + j : a.slots[r + j] & (B - 1)) * groups + i - j * groups] = encode(v);
    }
    __syncthreads();  // s_max is reused by the next run
  }
}

template <class T>
cudaError_t launch_append(const AppendArgs& a, int code, bool vec, dim3 grid, cudaStream_t s) {
  const dim3 block(APPEND_THREADS);
  if (code == GG_KV8_INT8)
    return vec ? launch_pdl(gg_append_kernel<T, GG_KV8_INT8, true>, grid, block, 0, s, a)
               : launch_pdl(gg_append_kernel<T, GG_KV8_INT8, false>, grid, block, 0, s, a);
  return vec ? launch_pdl(gg_append_kernel<T, GG_KV8_E4M3, true>, grid, block, 0, s, a)
             : launch_pdl(gg_append_kernel<T, GG_KV8_E4M3, false>, grid, block, 0, s, a);
}

}  // namespace gg

// ------------------------------------------------------------------------------ entry points

extern "C" int gg_plan_blocks(const gg_block_plan* plan, void* stream) {
  using namespace gg;
  const char* fn = "gg_plan_blocks";
  if (!plan) return ops_fail(GG_E_ARG, "%s: null plan", fn);
  const gg_block_plan& p = *plan;
  if (!p.old_len || !p.new_len || !p.table || !p.free_list || !p.free_count || !p.cu_rows || !p.lens || !p.row_seq ||
      !p.positions || !p.slots || !p.free_count_out || !p.status)
    return ops_fail(GG_E_ARG, "%s: null array", fn);
  if (p.seqs < 1 || p.max_blocks < 1 || p.rows < 0 || p.free_capacity < 0)
    return ops_fail(GG_E_ARG, "%s: seqs %d, max_blocks %d, rows %d, free_capacity %d out of range", fn, p.seqs, p.max_blocks, p.rows, p.free_capacity);
  if (p.table_stride < p.max_blocks) return ops_fail(GG_E_ARG, "%s: table_stride %lld below max_blocks %d", fn, (long long)p.table_stride, p.max_blocks);
  if (p.block_tokens < 1) return ops_fail(GG_E_ARG, "%s: block_tokens %d", fn, p.block_tokens);
  if (p.lens == p.old_len || p.lens == p.new_len) return ops_fail(GG_E_ARG, "%s: lens must not be old_len or new_len", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int rc = ops_check_stream(fn, s)) return rc;
  const int inline_rows = p.rows <= PLAN_INLINE_ROWS;
  static_assert(sizeof(PlanScan) > 48 * 1024 && sizeof(PlanScan) < 64 * 1024, "opt-in shared memory");
  const auto launch = [&](auto kernel, int threads) {
    return launch_big_smem<kernel.value>(dim3(1), dim3(threads), sizeof(PlanScan), s, p, inline_rows);
  };
  cudaError_t r = p.seqs <= 256            ? launch(PlanKernel<gg_plan_kernel<256, 1>>(), 256)
                  : p.seqs <= PLAN_THREADS ? launch(PlanKernel<gg_plan_kernel<PLAN_THREADS, 1>>(), PLAN_THREADS)
                  : p.seqs <= PLAN_CHUNK   ? launch(PlanKernel<gg_plan_kernel<PLAN_THREADS, PLAN_PER>>(), PLAN_THREADS)
                                           : launch(PlanKernel<gg_plan_many_kernel>(), PLAN_THREADS);
  if (r == cudaSuccess && !inline_rows) {
    const int grid = (int)(((long long)p.rows + 255) / 256);
    r = launch_pdl(gg_plan_rows_kernel, dim3(grid < 1184 ? grid : 1184), dim3(256), 0, s, p);
  }
  if (r != cudaSuccess) return ops_fail(GG_E_CUDA, "%s: launch: %s", fn, cudaGetErrorString(r));
  return GG_OK;
}

extern "C" int gg_rope(const gg_rope_call* call, void* stream) {
  using namespace gg;
  const char* fn = "gg_rope";
  if (!call || !call->positions || !call->freqs || !call->k.data != !call->k_out.data) return ops_fail(GG_E_ARG, "%s: null argument", fn);
  const gg_rows *q = &call->q, *q_out = &call->q_out, *k = call->k.data ? &call->k : nullptr, *k_out = &call->k_out;
  const int rows = call->rows, head_dim = call->head_dim, rot_dim = call->rot_dim, layout = call->layout;
  if (rows < 0 || head_dim < 1 || head_dim > 4096) return ops_fail(GG_E_ARG, "%s: rows %d or head_dim %d out of range", fn, rows, head_dim);
  if (rot_dim < 2 || rot_dim > head_dim || rot_dim % 2 || rot_dim / 2 > ROPE_CS)
    return ops_fail(GG_E_ARG, "%s: rot_dim %d is not an even number from 2 to min(head_dim %d, %d)", fn, rot_dim, head_dim, 2 * ROPE_CS);
  if (layout != GG_ROPE_HALF && layout != GG_ROPE_INTERLEAVED) return ops_fail(GG_E_ARG, "%s: layout %d is none of GG_ROPE_HALF, GG_ROPE_INTERLEAVED", fn, layout);
  const gg_rows* views[4] = {q, q_out, k, k_out};
  const char* names[4] = {"q", "q_out", "k", "k_out"};
  bool vec = true;
  for (int i = 0; i < (k ? 4 : 2); i++) {
    if (int rc = ops_check_rows(fn, names[i], views[i], rows, head_dim)) return rc;
    if (views[i]->type != q->type) return ops_fail(GG_E_ARG, "%s: %s has another type than q", fn, names[i]);
    vec &= ops_aligned16(*views[i]);
  }
  if (q_out->heads != q->heads || (k && k_out->heads != k->heads)) return ops_fail(GG_E_ARG, "%s: an output has another number of heads than its input", fn);
  if (q->heads + (k ? k->heads : 0) > 65535) return ops_fail(GG_E_ARG, "%s: too many heads", fn);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int rc = ops_check_stream(fn, s)) return rc;
  if (rows == 0) return GG_OK;
  RopeArgs a = {};
  a.q = {q->data, q_out->data, q->row_stride, q->head_stride, q_out->row_stride, q_out->head_stride};
  if (k) a.k = {k->data, k_out->data, k->row_stride, k->head_stride, k_out->row_stride, k_out->head_stride};
  a.pos = call->positions;
  a.freqs = call->freqs;
  a.mscale = call->mscale;
  a.rows = rows;
  a.q_heads = q->heads;
  a.heads = q->heads + (k ? k->heads : 0);
  a.hd = head_dim;
  a.rot = rot_dim;
  a.inverse = call->inverse != 0;
  a.interleaved = layout == GG_ROPE_INTERLEAVED;
  // rows of a CTA: enough that the angles keep its threads busy once there are rows for every SM
  int per = 1;
  while (per < 8 && 2 * per * (rot_dim / 2) <= ROPE_CS && (long long)rows >= 2ll * per * 148 * 4 && per * (rot_dim / 2) < ROPE_THREADS) per *= 2;
  a.rows_per_cta = per;
  const cudaError_t r = q->type == GG_T_F32 ? launch_rope<float>(a, vec, s) : q->type == GG_T_BF16 ? launch_rope<__nv_bfloat16>(a, vec, s) : launch_rope<__half>(a, vec, s);
  if (r != cudaSuccess) return ops_fail(GG_E_CUDA, "%s: launch: %s", fn, cudaGetErrorString(r));
  return GG_OK;
}

extern "C" int gg_rope_freqs(int scaling, int rot_dim, double theta, double factor, double trained, double low, double high,
                             double* freqs, double* mscale) {
  const char* fn = "gg_rope_freqs";
  if (!freqs || !mscale) return ops_fail(GG_E_ARG, "%s: null output", fn);
  if (rot_dim < 2 || rot_dim % 2 || rot_dim > 4096) return ops_fail(GG_E_ARG, "%s: rot_dim %d is not an even number from 2 to 4096", fn, rot_dim);
  if (scaling < GG_ROPE_NONE || scaling > GG_ROPE_YARN) return ops_fail(GG_E_ARG, "%s: scaling %d is none of GG_ROPE_*", fn, scaling);
  if (!(theta > 1.0) || !std::isfinite(theta)) return ops_fail(GG_E_ARG, "%s: theta must be above 1", fn);
  if (scaling != GG_ROPE_NONE && (!(factor > 0.0) || !std::isfinite(factor))) return ops_fail(GG_E_ARG, "%s: factor must be above 0", fn);
  if (scaling >= GG_ROPE_BANDS && (!(trained > 0.0) || !(low > 0.0) || !(low < high) || !std::isfinite(trained) || !std::isfinite(high)))
    return ops_fail(GG_E_ARG, "%s: needs trained > 0 and 0 < low < high", fn);
  const double tau = 6.283185307179586476925286766559;
  const int n = rot_dim / 2;
  // the pair that turns `turns` times in the trained positions: trained w_i = turns 2 pi
  const auto pair = [&](double turns) { return rot_dim * std::log(trained / (turns * tau)) / (2 * std::log(theta)); };
  double first = 0, last = 0;
  if (scaling == GG_ROPE_YARN) {
    first = std::fmax(std::floor(pair(high)), 0.0);
    last = std::fmin(std::ceil(pair(low)), rot_dim - 1.0);
    if (last - first < 0.001) last = first + 0.001;
  }
  *mscale = scaling == GG_ROPE_YARN && factor > 1.0 ? 0.1 * std::log(factor) + 1.0 : 1.0;
  for (int i = 0; i < n; i++) {
    const double w = std::pow(theta, -2.0 * i / rot_dim);
    double keep = 1.0;  // share of the unscaled frequency
    if (scaling == GG_ROPE_LINEAR) keep = 0.0;
    if (scaling == GG_ROPE_BANDS) keep = (trained * w / tau - low) / (high - low);
    if (scaling == GG_ROPE_YARN) keep = 1.0 - (i - first) / (last - first);
    keep = std::fmin(std::fmax(keep, 0.0), 1.0);
    freqs[i] = scaling == GG_ROPE_NONE ? w : w * keep + w * (1.0 - keep) / factor;
  }
  return GG_OK;
}

extern "C" int gg_kv8_append(const gg_kv8_cache* c, const gg_kv8_append_call* call, void* stream) {
  using namespace gg;
  const char* fn = "gg_kv8_append";
  if (!c || !call || !call->slots) return ops_fail(GG_E_ARG, "%s: null argument", fn);
  const gg_rows *k = &call->k, *v = &call->v;
  const int32_t* slots = call->slots;
  const int rows = call->rows;
  if (rows < 0) return ops_fail(GG_E_ARG, "%s: rows %d", fn, rows);
  if (int rc = ops_check_cache(fn, c)) return rc;
  if (int rc = ops_check_rows(fn, "k", k, rows, c->head_dim)) return rc;
  if (int rc = ops_check_rows(fn, "v", v, rows, c->head_dim)) return rc;
  if (k->type != v->type) return ops_fail(GG_E_ARG, "%s: k and v have different types", fn);
  if (k->heads != c->kv_heads || v->heads != c->kv_heads)
    return ops_fail(GG_E_ARG, "%s: k has %d and v %d heads, the cache %d", fn, k->heads, v->heads, c->kv_heads);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (int rc = ops_check_stream(fn, s)) return rc;
  if (rows == 0) return GG_OK;
  AppendArgs a = {};
  a.x[0] = k->data;
  a.x[1] = v->data;
  a.codes[0] = static_cast<uint8_t*>(c->k_codes);
  a.codes[1] = static_cast<uint8_t*>(c->v_codes);
  a.scale[0] = c->k_scale;
  a.scale[1] = c->v_scale;
  a.row[0] = k->row_stride;
  a.row[1] = v->row_stride;
  a.head[0] = k->head_stride;
  a.head[1] = v->head_stride;
  a.slots = slots;
  a.rows = rows;
  a.block_shift = __builtin_ctz(c->block_tokens);
  a.num_slots = c->num_blocks << a.block_shift;
  a.heads = c->kv_heads;
  a.hd = c->head_dim;
  // rows that a CTA looks through for the first of a run: every row of a decode step starts one, a
  // prompt's rows one in block_tokens, and CTAs that find none still cost their launch
  int per = 1;
  while (per < 32 && (long long)rows * c->kv_heads * 2 > 148ll * 8 * per) per *= 2;
  a.rows_per_cta = per;
  const dim3 grid((rows + per - 1) / per, 2 * c->kv_heads);
  const bool vec = ops_aligned16(*k) && ops_aligned16(*v);
  const cudaError_t r = k->type == GG_T_F32 ? launch_append<float>(a, c->code, vec, grid, s)
                        : k->type == GG_T_BF16 ? launch_append<__nv_bfloat16>(a, c->code, vec, grid, s)
                                               : launch_append<__half>(a, c->code, vec, grid, s);
  if (r != cudaSuccess) return ops_fail(GG_E_CUDA, "%s: launch: %s", fn, cudaGetErrorString(r));
  return GG_OK;
}
