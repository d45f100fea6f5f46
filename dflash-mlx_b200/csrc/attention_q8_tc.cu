// Attention over the 8-bit K/V cache on the 5th-generation tensor cores (tcgen05, accumulators and
// softmax weights in TMEM), for long key chunks. Same work split, masks, scales and partial-result
// format as attn_q8_kernel (attention_q8.cu); same independence of a row from its tile.
//
// One CTA per (run tile of up to 64 (token, head) rows, kv head, key chunk). The 128-row MMA tile
// holds the rows twice: copy 0 (TMEM lanes 0-63) takes keys 0-31 of every 64-key block, copy 1
// (lanes 64-127) keys 32-63, so that all four softmax warps have work; the copies are merged at the
// end. Per block:
//   S = Q K^T      M = 128, N = 64, K = hd, both operands fp16 in shared memory
//   w = e vs       one thread per (row, copy), 32 keys each; fp16, over S's own TMEM columns, the
//                  other copy's keys zero
//   O += w V       A = w from TMEM, B = V as [key][dim] in shared memory (MN-major), N = hd
// Warps 0-3 softmax and epilogue, 4-7 convert codes to fp16 tiles, 8 issues the MMAs.
// The converters load codes straight into registers, one block ahead of the one they convert, with
// the blocks after it prefetched into L2 by bulk prefetches: raw codes never pass shared memory, whose
// bandwidth (fp16 tiles written once and read once by the MMA: 8 bytes per code) is what this form
// is closest to.
// A row's exponent base M follows its maximum lazily: sums, weights and O are rescaled only when
// M would grow by more than 4 (log2), so weights stay below 2^15 in fp16 and those down to 2^-25 of the
// largest keep all their bits (those below are rounded to multiples of 2^-35 of it).
// Every wait is bounded (device error 350-359).
#include "attention_q8.cuh"
#include "tcgen05.cuh"

namespace dfl {

constexpr int QT_KB = 64;       // keys per block
constexpr int QT_ROWS = 64;     // (token, head) rows per tile
constexpr int QT_THREADS = 288;
constexpr int QT_SCALES = 4;    // scale ring: block i's are read until its weights are written
constexpr int QT_AHEAD = 4;     // blocks prefetched into L2
constexpr float QT_BASE = 10.f, QT_LAZY = 4.f;

template <int HD>
struct QtLayout {
  static constexpr int UNITS = HD / 64;  // 64-dim (128-byte) units of an fp16 row
  static constexpr int TILE = QT_KB * HD * 2;
  static constexpr int OFF_K = 0;               // 2 stages
  static constexpr int OFF_V = 2 * TILE;        // 2 stages; the epilogue reuses K and V for O
  static constexpr int OFF_Q = 4 * TILE;        // [units][128 rows][128 B]
  static constexpr int OFF_S = OFF_Q + 128 * HD * 2;  // scales [4][2][64]
  static constexpr int OFF_R = OFF_S + QT_SCALES * 2 * QT_KB * 4;  // row factor, limit, (M, l) of both copies
  static constexpr int OFF_BAR = OFF_R + QT_ROWS * 8 + 128 * 8;
  static constexpr int N_BAR = 2 * 4 + 2 * 3 + QT_SCALES;
  static constexpr int SMEM = OFF_BAR + N_BAR * 8 + 16 + 1024;
  static constexpr uint32_t COLS = HD == 256 ? 512 : 256;  // S / weights 2 x 64, O hd
  static_assert(4 * TILE >= 128 * HD * 4, "O of both copies fits the K and V stages");
};

__device__ __forceinline__ void tc_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(acc));
}

__device__ __forceinline__ void tc_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tc_st16_nowait(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// 16-byte chunk c of row r of a [rows][128 B] 128-byte-swizzled unit
__device__ __forceinline__ uint32_t qt_sw(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// kind::f16, A = B = fp16, D = fp32, M = 128; B K-major (S) or MN-major (O)
__host__ __device__ constexpr uint32_t qt_idesc(int n, bool mn) {
  return (1u << 4) | (mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

template <int HD, bool E4M3>
__global__ void __launch_bounds__(QT_THREADS, HD == 256 ? 1 : 2) attn_q8_tc_kernel(const __grid_constant__ AttnQ8Args a) {
  using L = QtLayout<HD>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* s_sc = reinterpret_cast<float*>(smem + L::OFF_S);  // [ring][K, V][64]
  float* s_rowf = reinterpret_cast<float*>(smem + L::OFF_R);
  int* s_lim = reinterpret_cast<int*>(smem + L::OFF_R) + QT_ROWS;
  float2* s_ml = reinterpret_cast<float2*>(smem + L::OFF_R + QT_ROWS * 8);  // [128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* k_full = bars;        // [2] 128 converter arrivals
  uint64_t* k_empty = bars + 2;   // [2] MMA commit
  uint64_t* v_full = bars + 4;    // [2] 128 converter arrivals
  uint64_t* v_empty = bars + 6;   // [2] MMA commit
  uint64_t* s_full = bars + 8;    // [2] MMA commit
  uint64_t* p_full = bars + 10;   // [2] 128 softmax arrivals: weights written (and S consumed)
  uint64_t* pv_done = bars + 12;  // [2] MMA commit: O holds the block
  uint64_t* sc_full = bars + 14;  // [QT_SCALES] 128 converter arrivals
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L::N_BAR);
  __shared__ int s_tok_lim[QT_ROWS], s_tok_ok[QT_ROWS];

  grid_dependency_wait();
  const int run = blockIdx.x / a.run_tiles, tile = blockIdx.x % a.run_tiles, kvh = blockIdx.y, chunk = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = run * a.run_rows + tile * a.tile_toks;
  const int ntok = min(min(a.tile_toks, a.run_rows - tile * a.tile_toks), a.M - m0);
  if (ntok <= 0) return;
  int seq = -1;  // of the tile's first row with a position
  for (int i = 0; i < ntok && seq < 0; ++i)
    if (a.pos[m0 + i] >= 0) seq = a.row_seq ? a.row_seq[m0 + i] : 0;
  if (seq < 0 || seq >= a.c.n_seqs) {
    if (seq >= 0 && threadIdx.x == 0) q8_error(a.err, Q8_ERR_SEQ);
    return;
  }
  if (threadIdx.x < ntok) {
    const int m = m0 + threadIdx.x, p = a.pos[m];
    int lim = 0, ok = p >= 0;
    if (ok && a.row_seq && a.row_seq[m] != seq) {
      q8_error(a.err, Q8_ERR_SEQ);
      ok = 0;
    }
    if (ok) lim = q8_row_limit(a, m, p, seq, chunk == 0 && kvh == 0 ? a.err : nullptr);
    s_tok_lim[threadIdx.x] = lim;
    s_tok_ok[threadIdx.x] = ok;
  }
  __syncthreads();
  int lim_max = 0, lim_min = 0x7fffffff;
  for (int i = 0; i < ntok; ++i) {
    const int lim = s_tok_lim[i];
    lim_max = max(lim_max, lim);
    if (lim > 0) lim_min = min(lim_min, lim);
  }
  const int k_begin = chunk * a.key_chunk;
  if (k_begin >= lim_max && a.n_chunks > 1) return;
  const int k_end = min(k_begin + a.key_chunk, lim_max);
  const int n_blocks = (max(k_end - k_begin, 0) + QT_KB - 1) / QT_KB;

  if (threadIdx.x == 256) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&k_full[s], 128);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 128);
      mbar_init(&v_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 128);
      mbar_init(&pv_done[s], 1);
    }
    for (int s = 0; s < QT_SCALES; ++s) mbar_init(&sc_full[s], 128);
    fence_barrier_init();
  }
  if (warp == 8) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)),
                 "n"(L::COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
  }
  // Q rows to scaled fp16, twice (softmax warps); a row's factor undoes its power of two
  if (warp < 4) {
    constexpr int VEC = HD / 32;
    for (int r = warp; r < QT_ROWS; r += 4) {
      const int tok = r / a.G, hg = r % a.G;
      const bool ok = tok < ntok && s_tok_lim[min(tok, ntok - 1)] > 0;
      const __nv_bfloat16* src = a.q + ((long long)(ok ? m0 + tok : m0) * a.Hq + kvh * a.G + (ok ? hg : 0)) * HD;
      uint32_t u[VEC / 2];
      if constexpr (VEC == 2) {
        u[0] = reinterpret_cast<const uint32_t*>(src)[lane];
      } else if constexpr (VEC == 4) {
        const uint2 w = reinterpret_cast<const uint2*>(src)[lane];
        u[0] = w.x, u[1] = w.y;
      } else {
        const uint4 w = reinterpret_cast<const uint4*>(src)[lane];
        u[0] = w.x, u[1] = w.y, u[2] = w.z, u[3] = w.w;
      }
      float x[VEC], mx = 0.f;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        x[j] = !ok ? 0.f : __uint_as_float(j & 1 ? u[j / 2] & 0xffff0000u : u[j / 2] << 16);
        mx = fmaxf(mx, fabsf(x[j]));
      }
      mx = warp_max(mx);
      int sh = 0;
      if (mx > 0.f && mx < INFINITY) sh = min(14 - ((int)(__float_as_uint(mx) >> 23) - 127), 120);
      const float f = __uint_as_float((uint32_t)(sh + 127) << 23) * a.q_sign;
#pragma unroll
      for (int j = 0; j < VEC; j += 2) {
        const int d = lane * VEC + j;
        const __half2 h = __floats2half2_rn(x[j] * f, x[j + 1] * f);
        unsigned char* dst = smem + L::OFF_Q + (d >> 6) * 16384 + ((d & 7) << 1);
        *reinterpret_cast<__half2*>(dst + qt_sw(r, (d & 63) >> 3)) = h;
        *reinterpret_cast<__half2*>(dst + qt_sw(r + QT_ROWS, (d & 63) >> 3)) = h;
      }
      if (lane == 0) {
        s_rowf[r] = a.scale_log2 * __uint_as_float((uint32_t)(127 - sh) << 23);
        s_lim[r] = ok ? s_tok_lim[tok] : 0;
      }
    }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dependency_launch_dependents();  // after the TMEM allocation: a dependent's must not come before it
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_o = tmem + 128;  // S / weights: columns 0-63, 64-127

  if (warp >= 4 && warp < 8) {
    // ---------------- converters ----------------
    constexpr int NC = HD / 16;                 // 16-code chunks per key
    constexpr int PER = QT_KB * NC / 128;       // chunks per thread and matrix
    const int ct = threadIdx.x - 128;
    const unsigned char* Kh = a.c.k + kvh * a.c.head_stride;
    const unsigned char* Vh = a.c.v + kvh * a.c.head_stride;
    const float* Sh = (ct < QT_KB ? a.c.ks : a.c.vs) + kvh * a.c.s_head_stride;
    // Lane bits: two of the chunk, one of the row, the rest of the chunk, the rest of the row: the eight
    // lanes of a 16-byte store phase write two rows' chunks of one unit, eight different bank groups.
    auto place = [&](int u, int& r, int& c) {
      const int idx = ct + u * 128;
      constexpr int HI = NC / 4;  // units
      c = (idx & 3) | (((idx >> 3) & (HI - 1)) << 2);
      r = ((idx >> 2) & 1) | ((idx / (8 * HI)) << 1);
    };
    struct Block {
      uint4 k[PER], v[PER];
      float s;
    };
    auto locate = [&](int i, long long& page, int& row) -> bool {
      return q8_place(a.c, seq, k_begin + i * QT_KB, ct == 0 ? a.err : nullptr, page, row);
    };
    auto prefetch = [&](int i) {  // both matrices' rows of block i, one bulk prefetch each
      long long page;
      int row;
      if (i >= n_blocks || ct >= 2 || !locate(i, page, row)) return;
      const int n = min(QT_KB, k_end - (k_begin + i * QT_KB));
      const unsigned char* p = (ct ? Vh : Kh) + page * a.c.seq_stride + (long long)row * HD;
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" ::"l"(p), "r"(n * HD) : "memory");
    };
    auto fetch = [&](int i, Block& b) {
      long long page;
      int row;
      const bool ok = locate(i, page, row);
      const int n = ok ? min(QT_KB, k_end - (k_begin + i * QT_KB)) : 0;
      const long long off = ok ? page * a.c.seq_stride + (long long)row * HD : 0;
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        int r, c;
        place(u, r, c);
        b.k[u] = b.v[u] = make_uint4(0, 0, 0, 0);
        if (r < n) {
          b.k[u] = __ldg(reinterpret_cast<const uint4*>(Kh + off + r * HD + c * 16));
          b.v[u] = __ldg(reinterpret_cast<const uint4*>(Vh + off + r * HD + c * 16));
        }
      }
      b.s = (ct & 63) < n ? __ldg(Sh + page * a.c.s_seq_stride + row + (ct & 63)) : 0.f;
    };
    auto convert = [&](const uint4& w, unsigned char* dst, int r, int c) {
      const uint32_t x[4] = {w.x, w.y, w.z, w.w};
      uint32_t h[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) q8_to_half<E4M3, true>(x[q], h[2 * q], h[2 * q + 1]);
      unsigned char* d = dst + (c >> 2) * (QT_KB * 128);
      *reinterpret_cast<uint4*>(d + qt_sw(r, (c & 3) * 2)) = make_uint4(h[0], h[1], h[2], h[3]);
      *reinterpret_cast<uint4*>(d + qt_sw(r, (c & 3) * 2 + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
    };
    Block nxt;
    for (int i = 1; i <= QT_AHEAD; ++i) prefetch(i);
    if (n_blocks > 0) fetch(0, nxt);
    for (int i = 0; i < n_blocks; ++i) {
      const int s = i & 1;
      const Block cur = nxt;
      if (i + 1 < n_blocks) {
        prefetch(i + 1 + QT_AHEAD);
        fetch(i + 1, nxt);
      }
      if (!mbar_wait(&k_empty[s], ((i >> 1) & 1) ^ 1, 350, a.err)) break;
      s_sc[(i & (QT_SCALES - 1)) * 2 * QT_KB + ct] = cur.s;
      mbar_arrive(&sc_full[i & (QT_SCALES - 1)]);
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        int r, c;
        place(u, r, c);
        convert(cur.k[u], smem + L::OFF_K + s * L::TILE, r, c);
      }
      fence_proxy_async_smem();
      mbar_arrive(&k_full[s]);
      if (!mbar_wait(&v_empty[s], ((i >> 1) & 1) ^ 1, 351, a.err)) break;
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        int r, c;
        place(u, r, c);
        convert(cur.v[u], smem + L::OFF_V + s * L::TILE, r, c);
      }
      fence_proxy_async_smem();
      mbar_arrive(&v_full[s]);
    }
  } else if (warp == 8) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      const uint32_t q0 = smem_u32(smem + L::OFF_Q);
      auto pv = [&](int j) -> bool {
        const int s = j & 1;
        if (!mbar_wait(&p_full[s], (j >> 1) & 1, 352, a.err)) return false;
        if (!mbar_wait(&v_full[s], (j >> 1) & 1, 353, a.err)) return false;
        tc_fence_after();
        const uint32_t vb = smem_u32(smem + L::OFF_V + s * L::TILE);
#pragma unroll
        for (int kk = 0; kk < QT_KB / 16; ++kk)
          tc_mma_ts(t_o, tmem + s * 64 + kk * 8, sw128_mn_desc(vb + kk * 2048, QT_KB * 128, 1024), qt_idesc(HD, true),
                    j > 0 || kk > 0 ? 1u : 0u);
        tc_commit(&v_empty[s]);
        tc_commit(&pv_done[s]);
        return true;
      };
      bool ok = true;
      for (int i = 0; i < n_blocks && ok; ++i) {
        const int s = i & 1;
        if (!mbar_wait(&k_full[s], (i >> 1) & 1, 354, a.err)) {
          ok = false;
          break;
        }
        tc_fence_after();
        // S of block i overwrites the weights of block i - 2, whose product was issued before it
        const uint32_t kt = smem_u32(smem + L::OFF_K + s * L::TILE);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          tc_mma(tmem + s * 64, sw128_desc(q0 + (kk >> 2) * 16384) + 2 * (kk & 3),
                 sw128_desc(kt + (kk >> 2) * (QT_KB * 128)) + 2 * (kk & 3), qt_idesc(QT_KB, false), kk > 0 ? 1u : 0u);
        tc_commit(&k_empty[s]);
        tc_commit(&s_full[s]);
        if (i > 0) ok = pv(i - 1);
      }
      if (ok && n_blocks > 0) pv(n_blocks - 1);
    }
    __syncwarp();
  } else if (warp < 4) {
    // ---------------- softmax: thread = (row, copy) ----------------
    const int row = threadIdx.x & 63, half = threadIdx.x >> 6;
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    const int lim = s_lim[row];
    const float rowf = s_rowf[row];
    float m = -INFINITY, mu_used = -INFINITY, l = 0.f;
    int er = -90;
    bool ok = true;
    for (int i = 0; i < n_blocks && ok; ++i) {
      const int s = i & 1;
      const float* sc = s_sc + (i & (QT_SCALES - 1)) * 2 * QT_KB + half * 32;
      const int kb = k_begin + i * QT_KB + half * 32;
      ok = mbar_wait(&sc_full[i & (QT_SCALES - 1)], (i / QT_SCALES) & 1, 355, a.err) &&
           mbar_wait(&s_full[s], (i >> 1) & 1, 356, a.err);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float sv[32];
      tc_ld32(tmem + lane_base + (uint32_t)(s * 64 + half * 32), sv);
      const bool full = kb + 32 <= lim_min;
      float mx = -INFINITY;
      uint32_t vm = 0;
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const float4 ks = *reinterpret_cast<const float4*>(sc + c);
        sv[c] *= ks.x;
        sv[c + 1] *= ks.y;
        sv[c + 2] *= ks.z;
        sv[c + 3] *= ks.w;
      }
      if (full) {
        const uint32_t b = __float_as_uint(sc[QT_KB + lane]) & 0x7fffffffu;
        vm = __reduce_max_sync(0xffffffffu, b < 0x7f800000u ? b : 0u);
      } else {
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const bool seen = kb + c < lim;
          sv[c] = seen ? sv[c] : -INFINITY;
          const uint32_t b = __float_as_uint(sc[QT_KB + c]) & 0x7fffffffu;
          if (seen && b < 0x7f800000u) vm = max(vm, b);
        }
      }
#pragma unroll
      for (int c = 0; c < 32; ++c) mx = fmaxf(mx, sv[c]);
      m = fmaxf(m, mx * rowf);
      er = max(er, (int)(vm >> 23) - 127);
      const float M = m + ((float)er - QT_BASE);
      const bool grow = M > mu_used + QT_LAZY || (mu_used == -INFINITY && M > -INFINITY);
      const float fac = grow ? exp2f(mu_used - M) : 1.f;
      if (grow) {
        mu_used = M;
        l *= fac;
      }
      if (i > 0 && __any_sync(0xffffffffu, grow)) {  // a factor of 1 is exact
        ok = mbar_wait(&pv_done[(i - 1) & 1], ((i - 1) >> 1) & 1, 357, a.err);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < HD; c += 16) {
          float ov[16];
          tc_ld16(t_o + lane_base + (uint32_t)c, ov);
#pragma unroll
          for (int e = 0; e < 16; ++e) ov[e] *= fac;
          tc_st16(t_o + lane_base + (uint32_t)c, ov);
        }
      }
      const float mu = mu_used == -INFINITY ? 0.f : mu_used;
      float ps0 = 0.f, ps1 = 0.f;
      uint32_t w[16];
#pragma unroll
      for (int c = 0; c < 32; c += 4) {
        const float4 vs = *reinterpret_cast<const float4*>(sc + QT_KB + c);
        const float e0 = exp2f(__fmaf_rn(sv[c], rowf, -mu)), e1 = exp2f(__fmaf_rn(sv[c + 1], rowf, -mu));
        const float e2 = exp2f(__fmaf_rn(sv[c + 2], rowf, -mu)), e3 = exp2f(__fmaf_rn(sv[c + 3], rowf, -mu));
        ps0 += e0 + e1;
        ps1 += e2 + e3;
        float w0 = e0 * vs.x, w1 = e1 * vs.y, w2 = e2 * vs.z, w3 = e3 * vs.w;
        if (!full) {
          w0 = kb + c < lim ? w0 : 0.f;
          w1 = kb + c + 1 < lim ? w1 : 0.f;
          w2 = kb + c + 2 < lim ? w2 : 0.f;
          w3 = kb + c + 3 < lim ? w3 : 0.f;
        }
        const __half2 h0 = __floats2half2_rn(w0, w1), h1 = __floats2half2_rn(w2, w3);
        w[c / 2] = *reinterpret_cast<const uint32_t*>(&h0);
        w[c / 2 + 1] = *reinterpret_cast<const uint32_t*>(&h1);
      }
      l += ps0 + ps1;
      const uint32_t t_w = tmem + lane_base + (uint32_t)(s * 64);
      tc_st16_nowait(t_w + half * 16, w);
#pragma unroll
      for (int c = 0; c < 16; ++c) w[c] = 0;
      tc_st16_nowait(t_w + (half ^ 1) * 16, w);
      tc_wait_st();
      tc_fence_before();
      mbar_arrive(&p_full[s]);
    }
    // ---- O of both copies through shared memory, then merged, row by row ----
    const int nb1 = n_blocks - 1;
    if (ok && n_blocks > 0) ok = mbar_wait(&pv_done[nb1 & 1], (nb1 >> 1) & 1, 358, a.err);
    ok = __all_sync(0xffffffffu, ok);
    constexpr int CH = HD / 4;  // float4 chunks per row
    float4* s_o = reinterpret_cast<float4*>(smem);
    if (ok && n_blocks > 0) {
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < HD; c += 16) {
        float ov[16];
        tc_ld16(t_o + lane_base + (uint32_t)c, ov);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s_o[threadIdx.x * CH + ((c / 4 + e) ^ (threadIdx.x & 7))] =
              make_float4(ov[4 * e], ov[4 * e + 1], ov[4 * e + 2], ov[4 * e + 3]);
      }
      tc_fence_before();
    }
    s_ml[threadIdx.x] = make_float2(mu_used, l);
    asm volatile("bar.sync 1, 128;\n" ::: "memory");
    constexpr int RPW = CH >= 32 ? 1 : 32 / CH;  // rows a warp writes at a time
    for (int r0 = warp * RPW; r0 < ntok * a.G && ok; r0 += 4 * RPW) {
      const int r = r0 + lane / (32 / RPW), c0 = lane % (32 / RPW);
      const int tok = r / a.G, hg = r % a.G;
      if (tok >= ntok || !s_tok_ok[tok]) continue;
      const int lm = s_lim[r];
      if (a.n_chunks > 1 && lm <= k_begin) continue;
      const float2 x0 = s_ml[r], x1 = s_ml[r + QT_ROWS];
      const float mm = fmaxf(x0.x, x1.x), mu = mm == -INFINITY ? 0.f : mm;
      const float w0 = exp2f(x0.x - mu), w1 = exp2f(x1.x - mu);
      const float den = w0 * x0.y + w1 * x1.y;
      const int mrow = m0 + tok, head = kvh * a.G + hg;
      const long long base = ((long long)chunk * a.M + mrow) * a.Hq + head;
#pragma unroll
      for (int c = c0; c < CH; c += 32) {
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        if (n_blocks > 0) {
          const float4 o0 = s_o[r * CH + (c ^ (r & 7))], o1 = s_o[(r + QT_ROWS) * CH + (c ^ (r & 7))];
          y = make_float4(w0 * o0.x + w1 * o1.x, w0 * o0.y + w1 * o1.y, w0 * o0.z + w1 * o1.z, w0 * o0.w + w1 * o1.w);
        }
        if (a.n_chunks > 1) {
          *reinterpret_cast<float4*>(a.part_o + base * HD + c * 4) = y;
        } else {
          const float inv = lm > 0 ? 1.f / den : 0.f;
          float f[4] = {y.x * inv, y.y * inv, y.z * inv, y.w * inv};
          if (a.gate) {
            const __nv_bfloat16* gr = a.gate + (long long)mrow * a.ldg + (long long)head * a.gate_hs + c * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = f[e] / (1.f + __expf(-bf2f(gr[e])));
          }
          *reinterpret_cast<uint2*>(a.out + (long long)mrow * a.ldo + (long long)head * HD + c * 4) =
              make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
        }
      }
      if (a.n_chunks > 1 && c0 == 0) a.part_ml[base] = make_float2(mm, den);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "n"(L::COLS));
  }
}

template <int HD, bool E4M3>
static int launch_qt(const AttnQ8Args& a, int tiles, cudaStream_t st) {
  using L = QtLayout<HD>;
  static bool opted[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !opted[dev]) {
    if (cudaFuncSetAttribute(attn_q8_tc_kernel<HD, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM) !=
        cudaSuccess) {
      cudaGetLastError();
      set_error("dfl_attention_q8: cannot opt in to %d bytes of shared memory", L::SMEM);
      return DFL_ERR_UNSUPPORTED;
    }
    if (dev >= 0 && dev < 64) opted[dev] = true;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles, a.c.Hkv, a.n_chunks);
  cfg.blockDim = dim3(QT_THREADS);
  cfg.dynamicSmemBytes = L::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_q8_tc_kernel<HD, E4M3>, a);
  if (e != cudaSuccess) {
    set_error("dfl_attention_q8: launch failed: %s", cudaGetErrorString(e));
    return DFL_ERR_CUDA;
  }
  return DFL_OK;
}

int launch_attention_q8_tc(const AttnQ8Args& a, int hd, bool e4m3, int tiles, cudaStream_t st) {
  switch (hd) {
    case 64: return e4m3 ? launch_qt<64, true>(a, tiles, st) : launch_qt<64, false>(a, tiles, st);
    case 128: return e4m3 ? launch_qt<128, true>(a, tiles, st) : launch_qt<128, false>(a, tiles, st);
    default: return e4m3 ? launch_qt<256, true>(a, tiles, st) : launch_qt<256, false>(a, tiles, st);
  }
}

}  // namespace dfl
