// gg_kv8_prompt.cu -- attention over the paged 8-bit KV cache for many query rows (prompts and
// prompt chunks). The mathematics and the exponent arithmetic are those of gg_kv8.cu.
//
// Bound by the tensor cores: 4 hd operations for each (row, key) pair. One CTA takes NQ tiles of
// 128 query rows (the heads that share a key head, token by token) and one range of keys, KT at a
// time; both products run as tcgen05 kind::f16 with f32 accumulators in TMEM:
//   converter warps  codes from global memory through registers (one tile ahead), widened to f16
//                    (exact) and stored as SW128 tiles: K (K-major B operand of Q K^T) and V, the
//                    same bytes read MN-major as the B operand of P V, so V is never transposed
//   MMA warps        S = Q K^T into TMEM, then O += P V with P read from TMEM; two warps, one for
//                    each query tile or, with one query tile, one for each product
//   softmax warps    four per query tile, a thread per row: S from TMEM, weights in registers (no
//                    shuffles), f16 weights back over S's columns as the A operand of P V
// S is double-buffered, so that the tensor cores work on the next key tile during the softmax of this
// one; hd <= 128 leaves TMEM for two query tiles, which share each converted key tile. (128 keys a
// tile and one S buffer a query tile took 656 us where this took 517: each query tile then waits for
// its own products.) f32 queries make both products twice, for the hi and the lo half of q and of
// the weights, into the same accumulators. The running maximum r is kept an integer and raised only
// when a weight would pass 2^KV8_SLACK, so the accumulator in TMEM is rarely rescaled (first tile,
// then now and then).
//
// Measured with 2005 and 1804 rows over 7058 and 5134 keys, 32 query heads over 8 of 128, int8, bf16:
// 405 us, 800 TFLOP/s. A step of 64 keys takes about 2250 cycles: the MMAs 1850 (61 cycles for N = 64,
// 75 for N = 128, both as slow from TMEM as from shared memory), the softmax about as long and the
// conversion of the codes almost so (without widening the step falls by an eighth, and without the
// exponentials by a twelfth; with queries of zeros by a seventh, at 975 W the operands count). Before
// and after its steps a CTA takes 10 us: query rows, output rows, and the next CTA's start.
//
// The tensor cores cut the f32 sums they hold: measured, a sum loses 6e-10 of itself a key and
// product, always downwards (1e-5 after 8192 keys with both products of f32 queries). For f16 and
// bf16 outputs that stays below their own rounding up to 2^18 keys, the most that a range has
// (KV8_LONGEST). For f32 ones O is added to an f32 row in memory (the row of the output itself) every PROMPT_FLUSH tiles and starts again from zero.
#include "gg_kv8.h"
#include "gg_tc.cuh"

namespace gg {

template <int HD, bool HILO>
struct PromptShape {
  static constexpr int NQ = HD == 256 ? 1 : 2;                       // query tiles of 128 rows
  static constexpr int KT = 64;                                      // keys of a tile
  static constexpr int ST = HD == 256 ? (HILO ? 1 : 2) : HILO ? 2 : 4;  // ring stages of K and of V
  static constexpr bool EARLY_K = ST <= 2;
  static constexpr int Q_BYTES = 128 * HD * 2 * (HILO ? 2 : 1);      // per query tile
  static constexpr int KV_BYTES = KT * HD * 2;
  static constexpr int GROUPS = 256;                                 // 16-key groups in the scale ring
  static constexpr int OFF_K = NQ * Q_BYTES;
  static constexpr int OFF_V = OFF_K + ST * KV_BYTES;
  static constexpr int OFF_META = OFF_V + ST * KV_BYTES;
  static constexpr int OFF_MUL = OFF_META + GROUPS * 16;
  static constexpr int OFF_BAR = OFF_MUL + NQ * 128 * 4;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;  // + alignment of the operand tiles
  static constexpr int SOFT_WARPS = 4 * NQ, CONV_WARPS = HD == 256 ? 8 : 4;
  static constexpr int THREADS = (SOFT_WARPS + CONV_WARPS + 2) * 32;  // and two that issue MMAs
  static constexpr int TMEM_S = KT;               // columns of one S buffer: two for each query tile
  static constexpr int TMEM_O = 2 * NQ * KT;      // first column of O
  static_assert(2 * NQ * KT + NQ * HD <= 512, "TMEM columns");
};

// MN-major operand, 128-byte swizzle: rows of 64 values of the N index, 8 rows (K index) to an
// atom of 1024 B; the next 8 rows follow 1024 B on, the next 64 values of N `slab` bytes on.
GG_DEV uint64_t umma_desc_sw128_mn(uint32_t saddr, uint32_t slab) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)((slab >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// kind::f16 with f16 operands and f32 sums, M = 128, N = n; B MN-major if b_mn.
GG_DEV uint32_t umma_idesc_f16_m128(int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// D(tmem) (+)= A x B, A from shared memory (descriptor) or TMEM, issued by the lanes with `on` set
// (one of them). The whole warp runs the code around them, so that addresses and descriptors stay
// in uniform registers: issued from a branch that one lane takes, each MMA first moves seven
// registers there (150 instead of 80 cycles an MMA).
GG_DEV void umma_f16_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
GG_DEV void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
GG_DEV void umma_commit_on(uint64_t* bar, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "setp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)), "r"(on)
      : "memory");
}
GG_DEV void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
GG_DEV void tmem_ld_done() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
GG_DEV void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
GG_DEV void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
GG_DEV void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two f32 at a time, each rounded to nearest as the single operations are.
GG_DEV uint64_t pack2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
GG_DEV void fma2(uint32_t& a, uint32_t& b, uint64_t f, uint64_t c) {  // (a, b) = (a, b) f + c
  asm("{\n\t.reg .b64 x;\n\tmov.b64 x, {%0, %1};\n\tfma.rn.f32x2 x, x, %2, %3;\n\tmov.b64 {%0, %1}, x;\n\t}" : "+r"(a), "+r"(b) : "l"(f), "l"(c));
}
GG_DEV void add2(uint64_t& s, float a, float b) { asm("{\n\t.reg .b64 x;\n\tmov.b64 x, {%1, %2};\n\tadd.rn.f32x2 %0, %0, x;\n\t}" : "+l"(s) : "f"(a), "f"(b)); }
GG_DEV float sum2(uint64_t s) {
  float a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(s));
  return a + b;
}
GG_DEV float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// In tiles of 64 keys. With 64 rows of positive values lose 4.4e-6 of a sum (6.1e-6 at most), and 2048 f32 rows
// behind 6000 keys, 32 heads over 8 of 128, take 444 us; with 32 2.2e-6 and 483 us, with 16 1.1e-6 and 562 us.
constexpr int PROMPT_FLUSH = 64;

// Wait for an mbarrier phase; after timeout_ns (or when another warp gave up) sets *abort and *err and
// returns false: the CTA then drains its MMAs and leaves NaN in its rows.
GG_DEV bool prompt_wait(uint64_t* bar, uint32_t parity, volatile int* abort, uint32_t* err, unsigned long long timeout_ns) {
#pragma unroll 1
  for (int it = 0; it < 64; ++it)
    if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
#pragma unroll 1
  for (;;) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort) return false;
    if (global_timer_ns() - t0 > timeout_ns) {
      *abort = 1;
      if (err) atomicOr(err, GG_ERR_WAIT_MBAR);
      return false;
    }
  }
}

// The same for a whole warp: all lanes agree on the outcome.
GG_DEV bool prompt_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort, uint32_t* err, unsigned long long timeout_ns) {
  return __all_sync(0xffffffffu, prompt_wait(bar, parity, abort, err, timeout_ns));
}

__global__ void gg_kv8_wait_probe_kernel(uint32_t* err, unsigned long long timeout_ns) {
  __shared__ uint64_t bar;
  __shared__ int abort;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    mbar_fence_init();
    abort = 0;
  }
  __syncthreads();
  (void)prompt_wait_warp(&bar, 0, &abort, err, timeout_ns);
}

template <int HD, int CODE, bool HILO>
__global__ void __launch_bounds__(PromptShape<HD, HILO>::THREADS, 1) gg_kv8_prompt_kernel(const Kv8Args a) {
  typedef PromptShape<HD, HILO> S;
  constexpr int NQ = S::NQ, KT = S::KT, ST = S::ST, GT = KT / 16;
  extern __shared__ unsigned char prompt_smem[];
  unsigned char* sm = prompt_smem + ((1024 - (smem_u32(prompt_smem) & 1023)) & 1023);
  float4* meta = reinterpret_cast<float4*>(sm + S::OFF_META);  // per 16-key group: ks, log2 vs, 1 / vs
  float* s_mul = reinterpret_cast<float*>(sm + S::OFF_MUL);
  uint64_t* kfull = reinterpret_cast<uint64_t*>(sm + S::OFF_BAR);
  // kfull, vfull, kdone: by ring stage; sfull, pfull: [query tile][parity of the key tile]; odone:
  // [query tile][key tile mod 4], so that a parity always tells a phase from the one before
  uint64_t *vfull = kfull + 4, *sfull = kfull + 8, *pfull = kfull + 12, *odone = kfull + 16, *kdone = kfull + 24, *drain = kfull + 26;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(kfull + 28);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const auto wait = [&](uint64_t* bar, uint32_t parity) { return prompt_wait_warp(bar, parity, abort, a.err, a.timeout_ns); };
  constexpr int MMA_WARP = S::SOFT_WARPS + S::CONV_WARPS;

  pdl_wait();
  int x = blockIdx.x;
  const int split = x % a.splits;
  x /= a.splits;
  const int h = x % a.kv_heads;
  x /= a.kv_heads;
  const int s = x % a.seqs, rt = a.row_tiles - 1 - x / a.seqs;  // every request's tiles with the most keys first
  const Kv8Seq sq = kv8_seq(a, s);
  const int items = sq.n * a.group, base = rt * (NQ * 128);
  const int nitems = max(min(NQ * 128, items - base), 0);
  const int heads = a.kv_heads * a.group;
  if (!nitems) {
    pdl_trigger();
    return;
  }
  // TMEM is taken after the wait for earlier kernels and before later ones may become resident: none
  // that waits for this one can hold the columns this one needs
  if (warp == MMA_WARP) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
    if (lane == 0) {
      for (int i = 0; i < 4; i++) {
        mbar_init(&kfull[i], S::CONV_WARPS);
        mbar_init(&vfull[i], S::CONV_WARPS);
        mbar_init(&odone[i], 1);
        mbar_init(&odone[4 + i], 1);
        mbar_init(&pfull[i], 4);
        mbar_init(&sfull[i], 1);
      }
      for (int i = 0; i < 2; i++) {
        mbar_init(&kdone[i], NQ);
        mbar_init(&drain[i], 1);
      }
      *abort = 0;
      mbar_fence_init();
    }
  }
  const long long pos_lo = sq.first_pos + base / a.group, pos_hi = sq.first_pos + (base + nitems - 1) / a.group;
  const int kmax = (int)min((long long)sq.len, pos_hi + 1);
  const int kmin = a.window ? (int)max(0ll, pos_lo - a.window + 1) & ~15 : 0;
  const int k00 = (int)min(kmin + 16ll * split * a.split_steps, (long long)kmax);  // first key of this range
  const int kend = (int)min((long long)kmax, k00 + (long long)a.split_steps * 16);
  const int nt = kend > k00 ? (kend - k00 + KT - 1) / KT : 0;

  // ---- query rows -> f16 tiles, each row times its own power of two
  if (nt) {
    // a warp takes QB rows at a time, all their loads in flight together; token and head of a row
    // within the tile: y / group for y < 1280 by a multiplication (with divisions: 527 us, not 517)
    const int tok0 = base / a.group, rem0 = base - tok0 * a.group;
    const uint32_t gmagic = (1u << 22) / a.group + 1;
    const long long q0 = (long long)(sq.row0 + tok0) * a.q_row + (long long)h * a.group * a.q_head;
    constexpr int WARPS = S::THREADS / 32, QB = 5 * NQ, PER = (HD / 4 + 31) / 32;
    const auto fill = [&](int type, int vec) {
      for (int row0 = warp; row0 < NQ * 128; row0 += WARPS * QB) {
        uint4 raw[QB][PER];
        load_raw4(raw, a.q, type, vec, [&](int j, int p) {
          const int row = row0 + j * WARPS, d = 4 * (lane + 32 * p), y = rem0 + row, tok = (int)(((uint32_t)y * gmagic) >> 22);
          return row < nitems && d < a.hd ? q0 + tok * a.q_row + (long long)(y - tok * a.group) * a.q_head + d : -1ll;
        });
#pragma unroll
        for (int j = 0; j < QB; j++) {
          const int row = row0 + j * WARPS;  // (no branch on it: the rows' instructions interleave)
          float4 v[PER];
          uint32_t top = 0;
#pragma unroll
          for (int p = 0; p < PER; p++) {
            v[p] = widen_raw4(raw[j][p], type, vec);
            top = max(max(top, __float_as_uint(v[p].x) & 0x7fffffffu), __float_as_uint(v[p].y) & 0x7fffffffu);
            top = max(max(top, __float_as_uint(v[p].z) & 0x7fffffffu), __float_as_uint(v[p].w) & 0x7fffffffu);
          }
          top = __reduce_max_sync(0xffffffffu, top);
          const int ex = min(max((int)(top >> 23) - 127, -100), 127);
          const float up = __uint_as_float((uint32_t)(14 - ex + 127) << 23);
          if (lane == 0 && row < NQ * 128) s_mul[row] = __uint_as_float((uint32_t)(ex - 14 + 127) << 23) * a.scale_log2;
          unsigned char* qt = sm + (row >> 7) * S::Q_BYTES;
          const int r = row & 127;
#pragma unroll
          for (int p = 0; p < PER; p++) {
            const int d = 4 * (lane + 32 * p);
            if (d >= HD || row >= NQ * 128) continue;
            uint2* dst = reinterpret_cast<uint2*>(qt + (d >> 6) * (128 * 128) + sw128_offset(r, d & 63));
            if constexpr (HILO) {
              uint2 hi, lo;
              split_f16(v[p].x * up, v[p].y * up, hi.x, lo.x);
              split_f16(v[p].z * up, v[p].w * up, hi.y, lo.y);
              *dst = hi;
              *reinterpret_cast<uint2*>(reinterpret_cast<unsigned char*>(dst) + S::Q_BYTES / 2) = lo;
            } else {
              *dst = make_uint2(half2_bits(v[p].x * up, v[p].y * up), half2_bits(v[p].z * up, v[p].w * up));
            }
          }
        }
      }
    };
    // one loop for each type, whose branches are not taken row by row
    if (HILO && a.q_vec) fill(GG_T_F32, 1);
    else if (!HILO && a.q_vec && a.q_type == GG_T_BF16) fill(GG_T_BF16, 1);
    else if (!HILO && a.q_vec && a.q_type == GG_T_F16) fill(GG_T_F16, 1);
    else fill(a.q_type, 0);
    fence_proxy_async_smem();
  }

  // ---- block ids and scales of 16-key groups, 64 groups (two to a lane) at a time
  const int32_t* table = a.table + (long long)s * a.table_stride;
  const auto load_id = [&](int group) {  // group of this range; -1 for a block the cache has not
    const long long key = k00 + 16ll * group;
    if (key >= kend) return -1;
    const int id = table[key >> a.block_shift];
    return id >= 0 && id < a.num_blocks ? id : -1;
  };
  const auto load_scales = [&](int id) {
    return id < 0 ? make_float2(0.f, 1.f) : make_float2(a.ks[(long long)id * a.kv_heads + h], a.vs[(long long)id * a.kv_heads + h]);
  };
  const auto put_group = [&](int group, int id, float2 sc) {
    // no block: scores of 0 under an exponent of -huge, rows of zeros in V, nothing added to l. A NaN
    // scale reaches l through the weights of the rows that see it, not through 1 / vs.
    meta[group & (S::GROUPS - 1)] = id < 0 ? make_float4(0.f, KV8_NEG, 0.f, 0.f) : make_float4(sc.x, log2f(sc.y), sc.y == sc.y ? 1.f / sc.y : 1.f, 0.f);
  };
  if (nt && tid < 64) {
    const int id = load_id(tid);
    put_group(tid, id, load_scales(id));
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;

  if (nt && warp >= S::SOFT_WARPS && warp < MMA_WARP) {
    // ------------------------------------------------------------------ converter warps
    // A thread keeps one 16-byte word of a key row and takes every KS-th key; a warp takes KPW keys
    // at once, all of one 16-key group, so block ids are the same for all its lanes. Eight lanes
    // hold four words of one 64-value slab of two neighbouring keys: their f16 chunks fall on
    // eight different bank groups.
    const int ct = tid - S::SOFT_WARPS * 32;
    constexpr int WP = HD / 16, KPW = 32 / WP, KS = S::CONV_WARPS * KPW, WORDS = KT / KS;
    const int k0 = (ct >> 5) * KPW + ((lane >> 2) & (KPW - 1)), w = (lane / (4 * KPW)) * 4 + (lane & 3);
    const bool mine = w * 16 < a.hd;
    constexpr int TB = 64 / GT;  // tiles of a batch of 64 groups
    const long long block_bytes = (long long)a.kv_heads * a.hd << a.block_shift;
    const int tok_mask = (1 << a.block_shift) - 1;
    const auto group_at = [&](int group, int id) {  // offset of a group's first key in its head's codes; -1: none
      return id < 0 ? -1ll : id * block_bytes + (long long)((k00 + 16 * group) & tok_mask) * a.hd;
    };
    // the groups of this batch and the next one's: two of each to a lane
    int nxt[2] = {load_id(lane), load_id(lane + 32)};
    long long nxt_at[2] = {group_at(lane, nxt[0]), group_at(lane + 32, nxt[1])}, cur_at[2] = {nxt_at[0], nxt_at[1]};
    static_assert(KS % 16 == 0 && KPW <= 8, "keys of a thread have the same place in their groups and the same swizzle");
    const long long lane_at = ((long long)h * a.hd << a.block_shift) + (k0 & 15) * a.hd + w * 16;
    const uint8_t *kc = a.kc + lane_at, *vc = a.vc + lane_at;
    const int left = mine ? min(sq.len, kend) - k00 - k0 : 0;
    long long at[WORDS];
    const auto locate = [&](int tile, int batch) {  // this thread's words of a tile, for K and for V
      const bool now = tile / TB == batch;
      const long long lo = now ? cur_at[0] : nxt_at[0], hi = now ? cur_at[1] : nxt_at[1];
#pragma unroll
      for (int i = 0; i < WORDS; i++) {
        const int k = k0 + KS * i, group = (tile * GT + (k >> 4)) & 63;
        at[i] = __shfl_sync(0xffffffffu, group & 32 ? hi : lo, group & 31);
        if (tile * KT + KS * i >= left) at[i] = -1;
      }
    };
    const auto fetch = [&](const uint8_t* codes, uint4 (&r)[WORDS]) {
#pragma unroll
      for (int i = 0; i < WORDS; i++) {
        r[i] = make_uint4(0, 0, 0, 0);
        if (at[i] >= 0) r[i] = __ldg(reinterpret_cast<const uint4*>(codes + at[i]));
      }
    };
    const uint32_t row0 = (w >> 2) * (KT * 128) + (k0 >> 3) * 1024 + (k0 & 7) * 128;
    const uint32_t at0 = row0 + ((((w & 3) * 2) ^ (k0 & 7)) << 4), at1 = row0 + ((((w & 3) * 2 + 1) ^ (k0 & 7)) << 4);
    const auto put = [&](unsigned char* tile, const uint4 (&r)[WORDS]) {
      if (mine) {
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
          uint4 lo, hi;
          widen4<CODE>(r[i].x, lo.x, lo.y);
          widen4<CODE>(r[i].y, lo.z, lo.w);
          widen4<CODE>(r[i].z, hi.x, hi.y);
          widen4<CODE>(r[i].w, hi.z, hi.w);
          *reinterpret_cast<uint4*>(tile + at0 + i * (KS * 128)) = lo;
          *reinterpret_cast<uint4*>(tile + at1 + i * (KS * 128)) = hi;
        }
      }
      fence_proxy_async_smem();
    };
    const auto products_done = [&](int i) {  // P V of key tile i, every query tile's
      bool ok = true;
      for (int q = 0; q < NQ; q++) ok = ok && wait(&odone[4 * q + i % 4], (i >> 2) & 1);
      return ok;
    };
    uint4 rk[WORDS], rv[WORDS];
    float2 sc[2] = {};
    locate(0, 0);
    fetch(kc, rk);
    fetch(vc, rv);
    for (int i = 0; i < nt; i++) {
      const int st = i % ST, par = (i / ST) & 1, b = i / TB, q = i % TB;
      // the next batch of groups: ids, then (one warp) scales, then shared memory, a quarter batch apart
      if (q == 0) {
        for (int j = 0; j < 2; j++) {
          const int group = (b + 1) * 64 + lane + 32 * j;
          cur_at[j] = nxt_at[j];
          nxt[j] = load_id(group);
          nxt_at[j] = group_at(group, nxt[j]);
        }
      }
      if (ct < 32 && q == TB / 4)
        for (int j = 0; j < 2; j++) sc[j] = load_scales(nxt[j]);
      if (ct < 32 && q == TB / 2)
        for (int j = 0; j < 2; j++) put_group((b + 1) * 64 + lane + 32 * j, nxt[j], sc[j]);
      // A stage is free once both products of the tile that had it are done; with few stages its K
      // is waited for, and handed back, by itself once the scores are.
      if (i >= ST && !(S::EARLY_K ? wait(&kdone[st], par ^ 1) : products_done(i - ST))) break;
      put(sm + S::OFF_K + st * S::KV_BYTES, rk);
      __syncwarp();
      if (lane == 0) mbar_arrive(&kfull[st]);
      locate(i + 1, b);
      fetch(kc, rk);
      if (S::EARLY_K && i >= ST && !products_done(i - ST)) break;
      put(sm + S::OFF_V + st * S::KV_BYTES, rv);
      __syncwarp();
      if (lane == 0) mbar_arrive(&vfull[st]);
      fetch(vc, rv);
    }
  } else if (nt && warp >= MMA_WARP) {
    // ------------------------------------------------------------------ MMA issue (lane 0's MMAs)
    // a warp for each query tile; with one query tile, a warp for each product
    const int q = NQ == 2 ? warp - MMA_WARP : 0;
    const bool for_s = NQ == 2 || warp == MMA_WARP, for_o = NQ == 2 || warp != MMA_WARP;
    const uint32_t on = lane == 0;
    // the same in every lane, which the compiler sees of a shuffle's result but not of a load's
    const int tiles = __shfl_sync(0xffffffffu, nt, 0);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const int steps = a.hd >> 4;
    const uint32_t idesc_s = umma_idesc_f16_m128(KT, false), idesc_o = umma_idesc_f16_m128(a.hd, true);
    const uint64_t qd = umma_desc_sw128(smem_u32(sm)), kd = umma_desc_sw128(smem_u32(sm + S::OFF_K));
    const uint64_t vd = umma_desc_sw128_mn(smem_u32(sm + S::OFF_V), KT * 128);
    // descriptors count 16-byte units; the address field does not overflow (227 KB of shared memory)
    const auto scores = [&](int i) {  // S buffer = Q tile q x K tile i
      const int buf = 2 * q + (i & 1);
      const uint64_t kb = kd + (uint32_t)(i % ST) * (S::KV_BYTES / 16);
#pragma unroll
      for (int part = 0; part < (HILO ? 2 : 1); part++)
#pragma unroll
        for (int k = 0; k < HD / 16; k++)
          if (k < steps)
            umma_f16_ss(tm + buf * S::TMEM_S, qd + (uint32_t)q * (S::Q_BYTES / 16) + part * (S::Q_BYTES / 32) + (k >> 2) * (128 * 128 / 16) + (k & 3) * 2,
                        kb + (k >> 2) * (KT * 128 / 16) + (k & 3) * 2, idesc_s, part > 0 || k > 0, on);
      umma_commit_on(&sfull[buf], on);
      if (S::EARLY_K) umma_commit_on(&kdone[i % ST], on);
    };
    const auto outputs = [&](int i) {  // O tile q += P x V tile i
      const uint32_t d = tm + S::TMEM_O + q * HD, p = tm + (2 * q + (i & 1)) * S::TMEM_S;
      const uint64_t vb = vd + (uint32_t)(i % ST) * (S::KV_BYTES / 16);
#pragma unroll
      for (int k = 0; k < KT / 16; k++)
#pragma unroll
        for (int part = 0; part < (HILO ? 2 : 1); part++)
          umma_f16_ts(d, p + part * 32 + k * 8, vb + k * (2048 / 16), idesc_o, (HILO ? i % PROMPT_FLUSH != 0 : i > 0) || k > 0 || part > 0, on);
      umma_commit_on(&odone[4 * q + (i & 3)], on);
    };
    // Scores run two key tiles ahead of their weights, so that the softmax warps hardly wait for
    // them. They overwrite the weights of two tiles before, once the product that reads those is
    // complete (MMAs with different accumulators are not ordered). Each wait costs the issuing warp
    // about 100 cycles even when it is over, and the tensor pipe runs dry meanwhile: hence two warps,
    // whose waits the other's products cover (427 us, one warp: 517). Each commit takes the pipe as long as
    // an MMA of N = 64 (62 cycles), hence few of them.
    bool ok = true;
    const auto scores_of = [&](int i) {  // when K is there and the buffer is free
      if (!for_s || !ok || i >= tiles) return;
      ok = wait(&kfull[i % ST], (i / ST) & 1);
      if (i > 1) ok = ok && wait(&odone[4 * q + (i - 2) % 4], ((i - 2) >> 2) & 1);
      if (!ok) return;
      tc_fence_after();
      scores(i);
    };
    scores_of(0);
    scores_of(1);
    for (int i = 0; ok && i < tiles; i++) {
      if (for_o) {  // when V and the weights are there
        ok = wait(&vfull[i % ST], (i / ST) & 1) && wait(&pfull[2 * q + (i & 1)], (i >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        outputs(i);
      }
      scores_of(i + 2);
    }
    if (!ok) {  // everything issued so far has finished before TMEM is freed
      uint64_t* mine = &drain[warp - MMA_WARP];
      umma_commit_on(mine, on);
      for (int it = 0; it < 1000000 && !mbar_try_wait(mine, 0); ++it) {
      }
    }
  } else if (warp < S::SOFT_WARPS) {
    // ------------------------------------------------------------------ softmax warps
    const int q = warp >> 2;
    const int row = q * 128 + (warp & 3) * 32 + lane;
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16), to = tl + S::TMEM_O + q * HD;
    const bool live = row < nitems;
    const int it = base + (live ? row : 0), tok = it / a.group, hq = h * a.group + it % a.group;
    const long long pos = sq.first_pos + tok;
    const int hi_key = live ? (int)min(pos, (long long)kend - 1) : -1;
    const int lo_key = a.window ? (int)max(0ll, pos - a.window + 1) : 0;
    // keys that every row of the CTA sees (dead rows see what they like: nothing of theirs is stored)
    const int all_hi = (int)min(pos_lo, (long long)kend - 1), all_lo = a.window ? (int)max(0ll, pos_hi - a.window + 1) : 0;
    const float mul = nt ? s_mul[row] : 0.f;
    float r = KV8_NEG, l = 0.f;
    bool ok = true;
    const long long ri = (long long)sq.row0 + tok, pi = (ri * heads + hq) * a.splits + split;
    // f32: the row in memory that takes O now and then, and r as it was the last time
    float* sum = nullptr;
    float sum_r = KV8_NEG;
    bool summed = false;
    const int sum_vec = a.splits > 1 || a.o_vec;
    if constexpr (HILO) sum = a.splits > 1 ? a.part_o + pi * a.hd : static_cast<float*>(a.out) + ri * a.o_row + (long long)hq * a.o_head;
    // O's columns c .. c + 31 and what memory has of them
    const auto gather = [&](int c, float keep, uint32_t (&v)[32]) {
      tmem_ld32(to + c, v);
      tmem_ld_done();
      if (HILO && summed && live) {
        const int n = min(32, a.hd - c);
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          if (e < n) {
            const float4 y = sum_vec ? *reinterpret_cast<const float4*>(sum + c + e) : make_float4(sum[c + e], sum[c + e + 1], sum[c + e + 2], sum[c + e + 3]);
            v[e] = __float_as_uint(fmaf(y.x, keep, __uint_as_float(v[e])));
            v[e + 1] = __float_as_uint(fmaf(y.y, keep, __uint_as_float(v[e + 1])));
            v[e + 2] = __float_as_uint(fmaf(y.z, keep, __uint_as_float(v[e + 2])));
            v[e + 3] = __float_as_uint(fmaf(y.w, keep, __uint_as_float(v[e + 3])));
          }
      }
    };
    for (int i = 0; i < nt; i++) {
      if (HILO && i > 0 && i % PROMPT_FLUSH == 0) {
        if (!(ok = wait(&odone[4 * q + (i - 1) % 4], ((i - 1) >> 2) & 1))) break;
        tc_fence_after();
        const float keep = ex2(sum_r - r);
        for (int c = 0; c < a.hd; c += 32) {
          uint32_t v[32];
          gather(c, keep, v);
          if (live) {
            const int n = min(32, a.hd - c);
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (e < n)
                store_elem4(sum, GG_T_F32, c + e, make_float4(__uint_as_float(v[e]), __uint_as_float(v[e + 1]), __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])), sum_vec);
          }
        }
        sum_r = r;
        summed = true;
      }
      const int buf = 2 * q + (i & 1);
      if (!(ok = wait(&sfull[buf], (i >> 1) & 1))) break;
      tc_fence_after();
      const uint32_t ts = tl + buf * S::TMEM_S;
      const int key0 = k00 + i * KT;
      const bool whole = key0 + 63 <= all_hi && key0 >= all_lo;
      const float4* mt = meta + ((i * GT) & (S::GROUPS - 1));
      uint32_t v[2][32];
      float top;
      // x = t - r + 7 in place of the scores: weights are 2^x = 2^7 w
      const auto exponents = [&](float from) {
        tmem_ld32(ts, v[0]);
        tmem_ld_done();
        tmem_ld32(ts + 32, v[1]);
        float tops[8];
#pragma unroll
        for (int g = 0; g < 4; g++) {
          if (g == 2) tmem_ld_done();
          const float4 m = mt[g];
          const float f = m.x * mul, c = m.y - from;
          const uint64_t f2 = pack2(f, f), c2 = pack2(c, c);
#pragma unroll
          for (int e = 0; e < 16; e += 2) fma2(v[g >> 1][(g & 1) * 16 + e], v[g >> 1][(g & 1) * 16 + e + 1], f2, c2);
        }
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 64; e++) {
            const int key = key0 + e;
            if (key > hi_key || key < lo_key) v[e >> 5][e & 31] = __float_as_uint(KV8_NEG);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) tops[e] = KV8_NEG;
#pragma unroll
        for (int e = 0; e < 64; e += 2) tops[(e >> 1) & 7] = max3(tops[(e >> 1) & 7], __uint_as_float(v[e >> 5][e & 31]), __uint_as_float(v[e >> 5][(e & 31) + 1]));
        top = max3(max3(tops[0], tops[1], tops[2]), max3(tops[3], tops[4], tops[5]), fmaxf(tops[6], tops[7]));
      };
      uint32_t ph[16], pl[16];
      // 32 keys: 16 columns of weights (HILO: and 16 of what they leave); returns their part of l
      const auto weights = [&](int g2) {
        float add = 0.f;
#pragma unroll
        for (int g = 0; g < 2; g++) {
          uint64_t sum = 0;  // (0, 0)
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float w0 = ex2(__uint_as_float(v[g2][g * 16 + 2 * e])), w1 = ex2(__uint_as_float(v[g2][g * 16 + 2 * e + 1]));
            add2(sum, w0, w1);
            if constexpr (HILO) split_f16(w0, w1, ph[g * 8 + e], pl[g * 8 + e]);
            else ph[g * 8 + e] = half2_bits(w0, w1);
          }
          add = fmaf(sum2(sum), mt[2 * g2 + g].z, add);
        }
        return add;
      };
      const auto store = [&](int g2) {
        tmem_st16(ts + g2 * 16, ph);
        if constexpr (HILO) tmem_st16(ts + 32 + g2 * 16, pl);
      };
      exponents(r - 7.f);
      float dl = weights(0);  // ahead of the vote, whose latency it covers
      if (__any_sync(0xffffffffu, top > 7.f + KV8_SLACK)) {
        const bool raise = top > 7.f + KV8_SLACK;
        exponents(0.f);
        const float nr = raise ? ceilf(top) : r;
        const float f = ex2(r - nr);  // 0 for the first keys of a row, else a power of two
        l *= f;
        if (HILO ? i % PROMPT_FLUSH != 0 : i > 0) {  // O is rescaled once the previous tile's product is in it
          if (!(ok = wait(&odone[4 * q + (i - 1) % 4], ((i - 1) >> 2) & 1))) break;
          tc_fence_after();
          for (int c = 0; c < a.hd; c += 32) {
            tmem_ld32(to + c, v[0]);
            tmem_ld_done();
#pragma unroll
            for (int e = 0; e < 32; e++) v[0][e] = __float_as_uint(__uint_as_float(v[0][e]) * f);
            tmem_st32(to + c, v[0]);
          }
        }
        tmem_st_done();
        r = nr;
        exponents(r - 7.f);
        dl = weights(0);
      }
      l += dl;
      store(0);
      l += weights(1);
      store(1);
      tmem_st_done();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pfull[buf]);
    }
    if (ok && nt) {
      ok = wait(&odone[4 * q + (nt - 1) % 4], ((nt - 1) >> 2) & 1);
      tc_fence_after();
    }
    l *= 1.f / KV8_WMUL;
    const float keep = ex2(sum_r - r);
    const float nan = __uint_as_float(0x7fffffffu);
    const float inv = !ok ? nan : a.splits > 1 ? 1.f / KV8_WMUL : l == 0.f ? 0.f : (1.f / KV8_WMUL) / l;
    // A warp's rows pass through the shared memory of its query rows, which no product reads any more, so
    // that they leave as whole rows and not 16 bytes of each at a time (2.9 us a
    // CTA instead of 3.6). Words are swizzled by row.
    constexpr int ES = HILO ? 4 : 2, WORDS_OUT = HD * ES / 16;
    unsigned char* turned = sm + q * S::Q_BYTES + (warp & 3) * (S::Q_BYTES / 4);
    const auto word_at = [&](int r, int w) { return reinterpret_cast<uint4*>(turned + r * (HD * ES) + ((w ^ (r & 7)) << 4)); };
    const long long oi = ri * a.o_row + (long long)hq * a.o_head;
    for (int c = 0; c < a.hd; c += 32) {
      uint32_t v[32];
      if (nt && ok) {
        gather(c, keep, v);
      } else {
#pragma unroll
        for (int e = 0; e < 32; e++) v[e] = 0;
      }
      if (live) {
        const int n = min(32, a.hd - c);
#pragma unroll
        for (int e = 0; e < 32; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * inv);
        if (a.splits > 1) {
          float* dst = a.part_o + pi * a.hd + c;
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (e < n) *reinterpret_cast<uint4*>(dst + e) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        } else {
          if (!a.o_vec) {
#pragma unroll
            for (int e = 0; e < 32; e++)
              if (e < n) store_elem(a.out, a.q_type, oi + c + e, __uint_as_float(v[e]));
          } else if constexpr (HILO) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) *word_at(lane, (c + e) / 4) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          } else {
            const bool bf = a.q_type == GG_T_BF16;
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; j++) {
                const float y0 = __uint_as_float(v[e + 2 * j]), y1 = __uint_as_float(v[e + 2 * j + 1]);
                w[j] = bf ? pack_bf16x2(__float2bfloat16_rn(y0), __float2bfloat16_rn(y1)) : half2_bits(y0, y1);
              }
              *word_at(lane, (c + e) / 8) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
      }
    }
    if (a.splits == 1 && a.o_vec) {
      __syncwarp();
      const uint32_t rows_live = __ballot_sync(0xffffffffu, live);
      const int words = a.hd * ES / 16;
#pragma unroll 4
      for (int k = 0; k < WORDS_OUT; k++) {
        const int x = k * 32 + lane, from = x / WORDS_OUT, w = x % WORDS_OUT;
        const long long at = __shfl_sync(0xffffffffu, oi, from);
        if ((rows_live >> from & 1) && w < words) reinterpret_cast<uint4*>(static_cast<unsigned char*>(a.out) + at * ES)[w] = *word_at(from, w);
      }
    }
    if (live) {
      if (a.splits > 1) a.part_ml[pi] = make_float2(r, ok ? l : nan);
      else if (a.lse) a.lse[ri * heads + hq] = !ok ? nan : l == 0.f ? -INFINITY : (r + log2f(l)) * 0.6931471805599453f;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD, int CODE, bool HILO>
static cudaError_t launch_prompt(const Kv8Args& a, cudaStream_t s) {
  typedef PromptShape<HD, HILO> S;
  const long long grid = (long long)a.seqs * a.kv_heads * a.row_tiles * a.splits;
  return launch_big_smem<gg_kv8_prompt_kernel<HD, CODE, HILO>>(dim3((unsigned)grid), dim3(S::THREADS), S::SMEM, s, a);
}
template <int HD>
static cudaError_t launch_prompt_hd(const Kv8Args& a, int code, cudaStream_t s) {
  const bool hilo = a.q_type == GG_T_F32;
  if (code == GG_KV8_INT8) return hilo ? launch_prompt<HD, GG_KV8_INT8, true>(a, s) : launch_prompt<HD, GG_KV8_INT8, false>(a, s);
  return hilo ? launch_prompt<HD, GG_KV8_E4M3, true>(a, s) : launch_prompt<HD, GG_KV8_E4M3, false>(a, s);
}

cudaError_t kv8_wait_probe(uint32_t* err, unsigned long long timeout_ns, cudaStream_t s) {
  gg_kv8_wait_probe_kernel<<<1, 32, 0, s>>>(err, timeout_ns);
  return cudaGetLastError();
}

int kv8_prompt_tile(int head_dim) { return head_dim <= 128 ? 256 : 128; }

cudaError_t kv8_launch_prompt(const Kv8Args& a, int code, cudaStream_t s) {
  return a.hd <= 64 ? launch_prompt_hd<64>(a, code, s) : a.hd <= 128 ? launch_prompt_hd<128>(a, code, s) : launch_prompt_hd<256>(a, code, s);
}

}  // namespace gg
