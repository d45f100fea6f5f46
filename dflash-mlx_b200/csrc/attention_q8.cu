// Grouped-query attention over the 8-bit K/V cache (dfl_kv_q8).
//
//   x_j = scale * ks_j * (q . Kc_j)            Kc, Vc codes; ks, vs their scales; j < lim(row)
//   o   = sum_j e_j vs_j Vc_j / sum_j e_j      e_j = exp(x_j - max x)
//
// Work split: one CTA per (run tile, kv head, key chunk). A run is the rows of one sequence; its
// tile's rows are (token, query head of the group) pairs packed without gaps, so a single token
// with G heads fills G rows of one 16-row MMA tile. Small calls take tiles of 16 rows (more CTAs, lower latency),
// large ones 32 or 64 (a 16-token verify block with G = 4), which read K and V once for all of them. The four
// warps of a row group are four strands: strand s takes the 32-key blocks s, s + 4, ... of the chunk with its own
// running maximum and sum, and the strands are merged in order at the end. Chunks are merged in order by
// a second kernel (one chunk: written directly). A row's arithmetic depends on the chunk size and
// on its own query and keys alone, whatever the tile's other rows, row groups or masks are: the
// rows of a verify block and of single-token decode agree bit for bit.
//
// Single tokens are bound by memory: 64 sequences of 512 to 4096 keys (e4m3) 62 us, 80 % of the copy rate; 4 of up to
// 131k keys (int8) 165 us, 87 %. Small calls are bound by latency, 8 us for one token at 1536 keys, 9.4 for 16 at
// 1024: two dependent launches, and in each positions, then codes, then the strands' merge.
//
// Codes go to fp16 exactly (int8 by placing the biased byte into 1024 + u and subtracting 1152;
// e4m3 by the conversion instruction) and the products run on mma.sync m16n8k16 with fp32
// accumulators. Both products contract over permuted dims / keys so that no byte is moved to be
// transposed: a K register of four codes holds four consecutive dims, so Q is stored in that
// order, and a V register read by ldmatrix.trans holds two keys of two adjacent dims, so even and
// odd dims go to two accumulator tiles.
//  * q is scaled by a power of two per row to [2^14, 2^15) at its largest element: every bf16 value
//    down to 2^-29 of it stays exact in fp16.
//  * The V scale goes into the weight, w_j = e_j vs_j, which is rounded to fp16 (2^-11 relative).
//    e_j is taken relative to a base M that follows the largest x_j + floor(log2 vs_j) that the row has seen (or up
//    to 4 more: attention_q8.cuh), less 4; it is raised, and sums and accumulators rescaled, only when it has fallen
//    behind by more than 10. So w_j < 2^15 whatever the scales are, and weights down to 2^-14 of the largest keep all
//    their bits, down to 2^-18 where the V scales are alike (those below are rounded to multiples of 2^-24, of 2^-28
//    of it); the sum of e_j uses the same M, which cancels in the quotient.
// Rows' statistics, sums and accumulators are fp32. Masked keys are selected away (their scales
// and query products may be anything), so infinities and NaN there do not reach the row; codes are
// numbers (a weight of 0 times e4m3's NaN code would not be 0; the append writes none).
#include "attention_q8.cuh"

#include <type_traits>

namespace dfl {

constexpr int Q8_KB = 32;       // keys per block
constexpr int Q8_STRANDS = 4;   // blocks in flight per chunk, each a warp of every row group
constexpr int Q8_CHUNK_UNIT = Q8_KB * Q8_STRANDS;

// ---- fp16 fragments ------------------------------------------------------------------
__device__ __forceinline__ void mma_f16_16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// byte offset of 16-byte chunk c of key row r in a stage's [32][HD]-byte tile: ldmatrix reads the
// same chunk of eight consecutive rows, which then lie in eight different 16-byte bank groups
template <int HD>
__device__ __forceinline__ int q8_swz(int r, int c) {
  return r * HD + ((HD == 64 ? c ^ ((r >> 1) & 3) : c ^ (r & 7)) << 4);
}

template <int HD, int MT, int RG, int ST>
struct AttnQ8Layout {
  static constexpr int ROWS = 16 * MT * RG;
  static constexpr int STAGE = 2 * Q8_KB * HD + 3 * Q8_KB * 4;  // K and V codes; K scales, V scales, V exponents
  static constexpr int RING = Q8_STRANDS * ST * STAGE;
  static constexpr int MERGE = Q8_STRANDS * ROWS * HD * 4 + Q8_STRANDS * ROWS * 8;
  static constexpr int BASE = RING > MERGE ? RING : MERGE;  // the merge reuses the ring
  static constexpr int OFF_Q = BASE;
  static constexpr int OFF_F = OFF_Q + ROWS * HD * 2;  // row factors, row limits
  static constexpr int SMEM = OFF_F + ROWS * 8;
};

template <int HD, int MT, int RG, int ST, bool E4M3>
// single tokens at head_dim <= 128: three CTAs an SM (12 warps; 10 % faster than two at a 3-stage ring)
__global__ void __launch_bounds__(32 * Q8_STRANDS * RG, MT == 1 && HD <= 128 ? 3 : 1) attn_q8_kernel(const __grid_constant__ AttnQ8Args a) {
  using L = AttnQ8Layout<HD, MT, RG, ST>;
  constexpr int NC = HD / 16;
  constexpr int NWARPS = Q8_STRANDS * RG;
  extern __shared__ __align__(128) unsigned char smem[];
  __half* sQ = reinterpret_cast<__half*>(smem + L::OFF_Q);
  float* s_rowf = reinterpret_cast<float*>(smem + L::OFF_F);
  int* s_lim = reinterpret_cast<int*>(smem + L::OFF_F) + L::ROWS;
  __shared__ int s_tok_lim[L::ROWS], s_tok_ok[L::ROWS];

  grid_dependency_wait();
  grid_dependency_launch_dependents();  // the merge kernel relies on this order

  const Q8Tile at = q8_tile(a);
  const int run = at.run, tile = at.tile, kvh = at.kvh, chunk = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int strand = warp % Q8_STRANDS, rg = warp / Q8_STRANDS;
  const int g = lane >> 2, t = lane & 3;
  const int m0 = run * a.run_rows + tile * a.tile_toks;
  const int ntok = min(min(a.tile_toks, a.run_rows - tile * a.tile_toks), a.M - m0);
  if (ntok <= 0) return;

  // the tile's rows, two a lane, by every warp alike: their positions and sequences, the run's sequence
  // (that of the first row with a position), limits
  int pos2[2], sq2[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = lane + 32 * k;
    pos2[k] = i < ntok ? a.pos[m0 + i] : -1;
    sq2[k] = i < ntok && a.row_seq ? a.row_seq[m0 + i] : 0;
  }
  // this warp's Q rows, on their way while positions and limits are looked up
  constexpr int VEC = HD / 32, NI = L::ROWS / NWARPS;
  uint32_t qu[NI][VEC / 2];
  {
    const float inv_g = 1.f / (float)a.G;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = warp + i * NWARPS;
      const int tok = (int)(((float)r + 0.5f) * inv_g);  // r / G: at least 1 / 32 from an integer
      const uint32_t* src = reinterpret_cast<const uint32_t*>(
          a.q + ((long long)(m0 + min(tok, ntok - 1)) * a.Hq + kvh * a.G + (r - tok * a.G)) * HD) + lane * (VEC / 2);
      if constexpr (VEC == 2) {
        qu[i][0] = src[0];
      } else if constexpr (VEC == 4) {
        const uint2 w = *reinterpret_cast<const uint2*>(src);
        qu[i][0] = w.x, qu[i][1] = w.y;
      } else {
        const uint4 w = *reinterpret_cast<const uint4*>(src);
        qu[i][0] = w.x, qu[i][1] = w.y, qu[i][2] = w.z, qu[i][3] = w.w;
      }
    }
  }
  const unsigned v0 = __ballot_sync(0xffffffffu, pos2[0] >= 0), v1 = __ballot_sync(0xffffffffu, pos2[1] >= 0);
  if (!(v0 | v1)) return;
  const int seq = __shfl_sync(0xffffffffu, v0 ? sq2[0] : sq2[1], __ffs(v0 ? v0 : v1) - 1);
  if (seq < 0 || seq >= a.c.n_seqs) {  // a row that names no sequence of the cache is left as it is
    if (threadIdx.x == 0) q8_error(a.err, Q8_ERR_SEQ);
    return;
  }
  int lim_max = 0, lim_min = 0x7fffffff;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int i = lane + 32 * k;
    const bool ok = pos2[k] >= 0 && sq2[k] == seq;
    if (warp == 0 && pos2[k] >= 0 && !ok) q8_error(a.err, Q8_ERR_SEQ);
    const int lim = ok ? q8_row_limit(a, m0 + i, pos2[k], seq, warp == 0 && chunk == 0 && kvh == 0 ? a.err : nullptr) : 0;
    if (warp == 0 && i < L::ROWS) {
      s_tok_lim[i] = lim;
      s_tok_ok[i] = ok;
    }
    lim_max = max(lim_max, lim);
    if (lim > 0) lim_min = min(lim_min, lim);
  }
  lim_max = __reduce_max_sync(0xffffffffu, lim_max);
  lim_min = __reduce_min_sync(0xffffffffu, lim_min);
  const int k_begin = chunk * a.key_chunk;
  if (k_begin >= lim_max && a.n_chunks > 1) return;  // the merge kernel writes rows without keys
  const int k_end = min(k_begin + a.key_chunk, lim_max);

  // ---- K/V blocks of this strand into its ring ----
  unsigned char* ring = smem + strand * ST * L::STAGE;
  const unsigned char* Kh = a.c.k + kvh * a.c.head_stride;
  const unsigned char* Vh = a.c.v + kvh * a.c.head_stride;
  const float* KSh = a.c.ks + kvh * a.c.s_head_stride;
  const float* VSh = a.c.vs + kvh * a.c.s_head_stride;
  const int n_blocks = (max(k_end - k_begin, 0) + Q8_KB - 1) / Q8_KB;
  const int my_n = n_blocks > strand ? (n_blocks - strand + Q8_STRANDS - 1) / Q8_STRANDS : 0;
  // Thread `first` of the strand copies 16-byte chunks first, first + T, ... of a block, which is contiguous in
  // the cache: chunk u * T + first lies in row r0 + u * SR, whose swizzle is r0's with SR * u's low bits flipped.
  constexpr int T = 32 * RG, SR = T / NC;
  const int first = rg * 32 + lane, r0c = first / NC;
  const uint32_t dst0 = smem_u32(ring) + q8_swz<HD>(r0c, first % NC);
  // the page of the next block to load, looked up one block ahead; -1 when it is refused
  auto page_of = [&](int i) -> int {
    long long page = -1;
    int row;
    if (i < my_n && !q8_place(a.c, seq, k_begin + (strand + i * Q8_STRANDS) * Q8_KB, lane == 0 ? a.err : nullptr, page, row))
      page = -1;
    return (int)page;
  };
  int next_page = page_of(0);
  auto load = [&](int i) {  // block i of the strand
    const int kb = k_begin + (strand + i * Q8_STRANDS) * Q8_KB;
    unsigned char* st = ring + (i % ST) * L::STAGE;
    const bool ok = next_page >= 0;
    const long long page = max(next_page, 0);
    const int row = !ok ? 0 : a.c.page_table ? kb & ((1 << a.c.page_shift) - 1) : kb;
    next_page = page_of(i + 1);
    const unsigned char* kp = Kh + (page * a.c.seq_stride + (long long)row * HD) + first * 16;
    const unsigned char* vp = Vh + (page * a.c.seq_stride + (long long)row * HD) + first * 16;
    const long long soff = page * a.c.s_seq_stride + row;
    const int n = ok ? min(Q8_KB, k_end - kb) : 0;  // rows of the block that hold keys
    const uint32_t d = dst0 + (i % ST) * L::STAGE;
#pragma unroll
    for (int u = 0; u < Q8_KB * NC / T; ++u) {
      const uint32_t du = (HD == 64 ? d : d ^ ((u * SR & 7) << 4)) + u * SR * HD;
      if (n == Q8_KB) {
        cp_async16(du, kp + u * T * 16, 16);
        cp_async16(du + Q8_KB * HD, vp + u * T * 16, 16);
      } else {  // rows behind the last key read as zeros
        const bool in = r0c + u * SR < n;
        cp_async16(du, in ? kp + u * T * 16 : Kh, in ? 16 : 0);
        cp_async16(du + Q8_KB * HD, in ? vp + u * T * 16 : Vh, in ? 16 : 0);
      }
    }
    if (rg == 0) {
      float* sc = reinterpret_cast<float*>(st + 2 * Q8_KB * HD);
      if (lane < n) {
        cp_async4(smem_u32(sc + lane), KSh + soff + lane);
        cp_async4(smem_u32(sc + Q8_KB + lane), VSh + soff + lane);
      } else {
        sc[lane] = 0.f;
        sc[Q8_KB + lane] = 0.f;
      }
    }
  };
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) {
    if (i < my_n) load(i);
    cp_async_commit();
  }

  __syncthreads();  // the rows' limits
  // ---- Q rows to scaled fp16, dims permuted within 16 to the order of a K register ----
  bool q_ok[NI];
  float q_max[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int tok = (warp + i * NWARPS) / a.G;
    q_ok[i] = tok < ntok && s_tok_lim[min(tok, ntok - 1)] > 0;
    q_max[i] = 0.f;
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
      if (!q_ok[i]) qu[i][j] = 0;
      q_max[i] = fmaxf(q_max[i], fmaxf(fabsf(__uint_as_float(qu[i][j] << 16)), fabsf(__uint_as_float(qu[i][j] & 0xffff0000u))));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < NI; ++i) q_max[i] = fmaxf(q_max[i], __shfl_xor_sync(0xffffffffu, q_max[i], o));
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = warp + i * NWARPS;
    const float mx = q_max[i];
    // 2^(14 - floor(log2 mx)), within fp32's normal powers of two; 1 for zero or non-finite rows
    int sh = 0;
    if (mx > 0.f && mx < INFINITY) sh = min(14 - ((int)(__float_as_uint(mx) >> 23) - 127), 120);
    const float f = __uint_as_float((uint32_t)(sh + 127) << 23);
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
      const int d = lane * VEC + j;
      const int c = d >> 4, dd = d & 15;
      const int kp = 2 * (dd >> 2) + (dd & 2) * 4;  // place of dims (dd, dd + 1) among the 16
      const int cc = 2 * c + (kp >> 3);
      const __half2 h = __floats2half2_rn(__uint_as_float(qu[i][j / 2] << 16) * f * a.q_sign,
                                          __uint_as_float(qu[i][j / 2] & 0xffff0000u) * f * a.q_sign);
      *reinterpret_cast<__half2*>(sQ + r * HD + ((cc ^ (r & 7)) << 3) + (kp & 7)) = h;
    }
    if (lane == 0) {
      s_rowf[r] = q8_row_factor(a.scale_log2, sh);
      s_lim[r] = q_ok[i] ? s_tok_lim[r / a.G] : 0;
    }
  }
  __syncthreads();

  const int r0 = rg * MT * 16;  // this warp's rows: r0 + mt * 16 + g (+ 8)
  float rowf[MT][2], Mr[MT][2], mrow[MT][2], lrow[MT][2];  // mrow: largest x_j + exponent of vs_j
  int lim[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      rowf[mt][h] = s_rowf[r0 + mt * 16 + g + 8 * h];
      lim[mt][h] = s_lim[r0 + mt * 16 + g + 8 * h];
      mrow[mt][h] = Mr[mt][h] = -INFINITY;
      lrow[mt][h] = 0.f;
    }
  float o[MT][2 * NC][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int j = 0; j < 2 * NC; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[mt][j][e] = 0.f;

  auto sync_strand = [&]() {
    if (RG == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;\n" ::"r"(1 + strand), "n"(32 * RG) : "memory");
  };

  for (int i = 0; i < my_n; ++i) {
    cp_async_wait<ST - 2>();
    sync_strand();  // block i is there for every warp of the strand; the stage refilled below was read last time
    if (i + ST - 1 < my_n) load(i + ST - 1);
    cp_async_commit();
    unsigned char* sK = ring + (i % ST) * L::STAGE;
    const unsigned char* sV = sK + Q8_KB * HD;
    float* sc = reinterpret_cast<float*>(sK + 2 * Q8_KB * HD);
    const int kb = k_begin + (strand + i * Q8_STRANDS) * Q8_KB;
    const bool full = kb + Q8_KB <= lim_min;  // every row with keys sees the whole block

    float s[MT][4][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mt][j][e] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint32_t af[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int row = r0 + mt * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
        const int cc = 2 * c + (lane >> 4);
        ldmatrix_x4(smem_u32(sQ + row * HD + ((cc ^ (row & 7)) << 3)), af[mt][0], af[mt][1], af[mt][2], af[mt][3]);
      }
      uint32_t kr[4];  // keys 0-7, 8-15, 16-23, 24-31: dims 16 c + 4 t .. + 3 of key g
      ldmatrix_x4(smem_u32(sK + q8_swz<HD>(lane, c)), kr[0], kr[1], kr[2], kr[3]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t b0, b1;
        q8_to_half<E4M3, true>(kr[j], b0, b1);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) mma_f16_16816(s[mt][j], af[mt], b0, b1);
      }
    }

    uint32_t pf[MT][2][4];  // weights, as A fragments of the two 16-key steps
    auto softmax = [&](auto full_c) {
      constexpr bool FULL = decltype(full_c)::value;
      float2 ks[4], vs[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ks[j] = *reinterpret_cast<const float2*>(sc + j * 8 + 2 * t);
        vs[j] = *reinterpret_cast<const float2*>(sc + Q8_KB + j * 8 + 2 * t);
      }
      const int e = q8_exponent(sc[Q8_KB + lane]);
      const int e_max = __reduce_max_sync(0xffffffffu, e);
      const bool near = e_max - __reduce_min_sync(0xffffffffu, e) <= Q8_NEAR;
      if (!FULL || !near) {
        sc[2 * Q8_KB + lane] = (float)e;  // by every warp of the strand alike
        __syncwarp();
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float fac[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int lm = lim[mt][h];
          float mx = -INFINITY;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = kb + j * 8 + 2 * t;
            float t0 = s[mt][j][2 * h] * ks[j].x, t1 = s[mt][j][2 * h + 1] * ks[j].y;
            if (!FULL) {
              t0 = key < lm ? t0 : -INFINITY;
              t1 = key + 1 < lm ? t1 : -INFINITY;
            }
            s[mt][j][2 * h] = t0;
            s[mt][j][2 * h + 1] = t1;
            mx = fmaxf(mx, fmaxf(t0, t1));
          }
          mx = __fmaf_rn(mx, rowf[mt][h], (float)e_max);
          if (!FULL || !near) {
            float z = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 ex = *reinterpret_cast<const float2*>(sc + 2 * Q8_KB + j * 8 + 2 * t);
              z = fmaxf(z, fmaxf(__fmaf_rn(s[mt][j][2 * h], rowf[mt][h], ex.x),
                                 __fmaf_rn(s[mt][j][2 * h + 1], rowf[mt][h], ex.y)));
            }
            if (!near || kb + Q8_KB > lm) mx = z;
          }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          mrow[mt][h] = fmaxf(mrow[mt][h], mx);
          const float Mn = mrow[mt][h] - Q8_BASE;  // -inf while the row has seen no key
          const bool grow = Mn > Mr[mt][h] + Q8_LAZY || (Mr[mt][h] == -INFINITY && Mn > -INFINITY);
          const float root = grow ? q8_exp2(0.5f * (Mr[mt][h] - Mn)) : 1.f;
          fac[h] = root * root;
          if (grow) Mr[mt][h] = Mn;
          const float mu = Mr[mt][h] == -INFINITY ? 0.f : Mr[mt][h];
          float ps = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = kb + j * 8 + 2 * t;
            const float e0 = q8_exp2(__fmaf_rn(s[mt][j][2 * h], rowf[mt][h], -mu));
            const float e1 = q8_exp2(__fmaf_rn(s[mt][j][2 * h + 1], rowf[mt][h], -mu));
            ps += e0 + e1;
            float w0 = e0 * vs[j].x, w1 = e1 * vs[j].y;
            if (!FULL) {
              w0 = key < lm ? w0 : 0.f;
              w1 = key + 1 < lm ? w1 : 0.f;
            }
            const __half2 w = __floats2half2_rn(w0, w1);
            pf[mt][j >> 1][(j & 1) * 2 + h] = *reinterpret_cast<const uint32_t*>(&w);
          }
          lrow[mt][h] = __fmaf_rn(ps, Q8_SUM_UNIT, lrow[mt][h] * root * root);
        }
        if (__any_sync(0xffffffffu, fac[0] != 1.f || fac[1] != 1.f)) {  // a factor of 1 is exact
#pragma unroll
          for (int j = 0; j < 2 * NC; ++j) {
            o[mt][j][0] *= fac[0];
            o[mt][j][1] *= fac[0];
            o[mt][j][2] *= fac[1];
            o[mt][j][3] *= fac[1];
          }
        }
      }
    };
    if (full) softmax(std::true_type{});
    else softmax(std::false_type{});

#pragma unroll
    for (int c = 0; c < NC; ++c) {
      uint32_t vr[4];  // keys (2 t, 2 t + 1) + 0, 8, 16, 24 of dims 16 c + 2 g, + 1
      ldmatrix_x4_trans(smem_u32(sV + q8_swz<HD>(lane, c)), vr[0], vr[1], vr[2], vr[3]);
      uint32_t ev[4], od[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) q8_to_half<E4M3, false>(vr[u], ev[u], od[u]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        mma_f16_16816(o[mt][2 * c], pf[mt][0], ev[0], ev[1]);
        mma_f16_16816(o[mt][2 * c + 1], pf[mt][0], od[0], od[1]);
        mma_f16_16816(o[mt][2 * c], pf[mt][1], ev[2], ev[3]);
        mma_f16_16816(o[mt][2 * c + 1], pf[mt][1], od[2], od[3]);
      }
    }
  }
  cp_async_wait<0>();

  // ---- merge the strands in order: every warp writes its accumulators (the same lane holds the
  // same elements in all four), then strand s finishes a quarter of the dims ----
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      lrow[mt][h] += __shfl_xor_sync(0xffffffffu, lrow[mt][h], 1);
      lrow[mt][h] += __shfl_xor_sync(0xffffffffu, lrow[mt][h], 2);
    }
  __syncthreads();  // the rings are read no more
  float4* s_o = reinterpret_cast<float4*>(smem);
  float2* s_ml = reinterpret_cast<float2*>(smem + Q8_STRANDS * L::ROWS * HD * 4);  // [strand][row]
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        s_o[((((rg * MT + mt) * NC + c) * Q8_STRANDS + strand) * 2 + h) * 32 + lane] =
            make_float4(o[mt][2 * c][2 * h], o[mt][2 * c + 1][2 * h], o[mt][2 * c][2 * h + 1], o[mt][2 * c + 1][2 * h + 1]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (t == 0) s_ml[strand * L::ROWS + r0 + mt * 16 + g + 8 * h] = make_float2(Mr[mt][h], lrow[mt][h]);
  }
  __syncthreads();
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r0 + mt * 16 + g + 8 * h;
      const int tok = r / a.G, hg = r % a.G;
      if (tok >= ntok || !s_tok_ok[tok]) continue;
      const int lm = s_lim[r];
      if (a.n_chunks > 1 && lm <= k_begin) continue;
      float2 ml[Q8_STRANDS];
      float mm = -INFINITY;
#pragma unroll
      for (int u = 0; u < Q8_STRANDS; ++u) {
        ml[u] = s_ml[u * L::ROWS + r];
        mm = fmaxf(mm, ml[u].x);
      }
      const float mu = mm == -INFINITY ? 0.f : mm;
      float w[Q8_STRANDS], den = 0.f;
#pragma unroll
      for (int u = 0; u < Q8_STRANDS; ++u) {
        const float root = exp2f(0.5f * (ml[u].x - mu));
        w[u] = root * root;
        den += root * ml[u].y * root;
      }
      const int m = m0 + tok, head = kvh * a.G + hg;
      const long long base = ((long long)chunk * a.M + m) * a.Hq + head;
#pragma unroll
      for (int cq = 0; cq < NC / Q8_STRANDS; ++cq) {
        const int c = strand * (NC / Q8_STRANDS) + cq;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < Q8_STRANDS; ++u) {
          const float4 v = s_o[((((rg * MT + mt) * NC + c) * Q8_STRANDS + u) * 2 + h) * 32 + lane];
          y.x += w[u] * v.x;
          y.y += w[u] * v.y;
          y.z += w[u] * v.z;
          y.w += w[u] * v.w;
        }
        const int d = c * 16 + 4 * t;
        if (a.n_chunks > 1) {
          *reinterpret_cast<float4*>(a.part_o + base * HD + d) = y;
        } else {
          const float inv = lm > 0 ? Q8_SUM_UNIT / den : 0.f;
          // + 0: a zero of the sum is positive, as it is behind the merge kernel, whose sum starts at +0
          float f[4] = {(y.x + 0.f) * inv, (y.y + 0.f) * inv, (y.z + 0.f) * inv, (y.w + 0.f) * inv};
          if (a.gate) {
            const __nv_bfloat16* gr = a.gate + (long long)m * a.ldg + (long long)head * a.gate_hs + d;
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = f[e] / (1.f + __expf(-bf2f(gr[e])));
          }
          *reinterpret_cast<uint2*>(a.out + (long long)m * a.ldo + (long long)head * HD + d) =
              make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
        }
      }
      if (a.n_chunks > 1 && strand == 0 && t == 0) a.part_ml[base] = make_float2(mm, den);
    }
}

// Merges the chunk partials of one (row, head) in chunk order: one warp each, hd / 32 dims a lane. What it needs
// to know of the row is read before it waits for the chunk kernel, which lets it start only after what came before
// both; behind the wait the first partials are loaded together with their maxima and sums.
template <int HD>
__global__ void __launch_bounds__(256) attn_q8_merge_kernel(const __grid_constant__ AttnQ8Args a) {
  grid_dependency_launch_dependents();
  constexpr int VEC = HD / 32;
  constexpr int FL = 8;  // chunks' loads in flight
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * (blockDim.x >> 5) + warp;
  bool live = item < (long long)a.M * a.Hq;
  const int m = live ? (int)(item / a.Hq) : 0, h = (int)(item - (long long)m * a.Hq);
  const int p = __ldcg(a.pos + m), seq = a.row_seq ? __ldcg(a.row_seq + m) : 0;
  live = live && p >= 0 && seq >= 0 && seq < a.c.n_seqs;
  if (live && a.row_seq && a.run_rows > 1) {  // a row that is not of its tile's sequence was refused
    const int run0 = m / a.run_rows * a.run_rows;
    int first = run0 + (m - run0) / a.tile_toks * a.tile_toks;
    while (__ldcg(a.pos + first) < 0) ++first;  // ends at m at the latest
    live = __ldcg(a.row_seq + first) == seq;
  }
  const int lim = live ? q8_row_limit(a, m, p, seq, nullptr) : 0;
  const int nch = lim > 0 ? min((lim - 1) / a.key_chunk + 1, a.n_chunks) : 0;
  grid_dependency_wait();
  if (!live) return;
  const long long cstride = (long long)a.M * a.Hq;
  const float2* ml = a.part_ml + item;
  const float* po = a.part_o + item * HD + lane * VEC;
  float v[FL][VEC];
  auto fetch = [&](int c) {  // the partials of chunks c .. c + FL - 1
#pragma unroll
    for (int u = 0; u < FL; ++u) {
      const float* src = po + (long long)(c + u) * cstride * HD;
      if constexpr (VEC == 2) {
        const float2 y = c + u < nch ? *reinterpret_cast<const float2*>(src) : make_float2(0.f, 0.f);
        v[u][0] = y.x;
        v[u][1] = y.y;
      } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
          const float4 y = c + u < nch ? *reinterpret_cast<const float4*>(src + i) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[u][i] = y.x;
          v[u][i + 1] = y.y;
          v[u][i + 2] = y.z;
          v[u][i + 3] = y.w;
        }
      }
    }
  };
  float2 x = lane < nch ? ml[lane * cstride] : make_float2(-INFINITY, 0.f);
  fetch(0);
  float mmax = x.x;
  for (int c = lane + 32; c < nch; c += 32) mmax = fmaxf(mmax, ml[c * cstride].x);
  mmax = warp_max(mmax);
  const float mu = mmax == -INFINITY ? 0.f : mmax;
  float acc[VEC], den = 0.f;
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  for (int c0 = 0; c0 < nch; c0 += 32) {
    if (c0 > 0) x = c0 + lane < nch ? ml[(c0 + lane) * cstride] : make_float2(-INFINITY, 0.f);
    const float root = exp2f(0.5f * (x.x - mu)), w = root * root;
    den += warp_sum(root * x.y * root);
    const int n = min(32, nch - c0);
    for (int j0 = 0; j0 < n; j0 += FL) {
      if (c0 + j0 > 0) fetch(c0 + j0);
#pragma unroll
      for (int u = 0; u < FL; ++u) {
        const float wj = __shfl_sync(0xffffffffu, w, (j0 + u) & 31);
        if (j0 + u < n) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[i] += wj * v[u][i];
        }
      }
    }
  }
  const float inv = lim > 0 ? Q8_SUM_UNIT / den : 0.f;
  __nv_bfloat16* dst = a.out + (long long)m * a.ldo + (long long)h * HD + lane * VEC;
  float y[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) y[i] = acc[i] * inv;
  if (a.gate) {
    const __nv_bfloat16* gr = a.gate + (long long)m * a.ldg + (long long)h * a.gate_hs + lane * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) y[i] = y[i] / (1.f + __expf(-bf2f(gr[i])));
  }
#pragma unroll
  for (int i = 0; i < VEC; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pack_bf16x2(y[i], y[i + 1]);
}

template <int HD>
static int launch_attn_q8_merge(const AttnQ8Args& a, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(((long long)a.M * a.Hq + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_q8_merge_kernel<HD>, a);
  if (e != cudaSuccess) {
    set_error("dfl_attention_q8: merge launch failed: %s", cudaGetErrorString(e));
    return DFL_ERR_CUDA;
  }
  return DFL_OK;
}

template <int HD, int MT, int RG, int ST, bool E4M3>
static int launch_attn_q8(const AttnQ8Args& a, int tiles, cudaStream_t st) {
  using L = AttnQ8Layout<HD, MT, RG, ST>;
  static bool opted[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !opted[dev]) {
    if (cudaFuncSetAttribute(attn_q8_kernel<HD, MT, RG, ST, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             L::SMEM) != cudaSuccess) {
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
  cfg.gridDim = dim3(tiles * a.c.Hkv, a.n_chunks);
  cfg.blockDim = dim3(32 * Q8_STRANDS * RG);
  cfg.dynamicSmemBytes = L::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_q8_kernel<HD, MT, RG, ST, E4M3>, a);
  if (e != cudaSuccess) {
    set_error("dfl_attention_q8: launch failed: %s", cudaGetErrorString(e));
    return DFL_ERR_CUDA;
  }
  return DFL_OK;
}

template <int HD, bool E4M3>
static int launch_attn_q8_rows(const AttnQ8Args& a, int rows, int tiles, cudaStream_t st) {
  if (rows <= 16) return launch_attn_q8<HD, 1, 1, HD == 256 ? 3 : 2, E4M3>(a, tiles, st);
  if constexpr (HD == 256) {
    return launch_attn_q8<HD, 1, 2, 2, E4M3>(a, tiles, st);
  } else {
    if (rows <= 32) return launch_attn_q8<HD, 2, 1, 2, E4M3>(a, tiles, st);
    return launch_attn_q8<HD, 2, 2, 4, E4M3>(a, tiles, st);
  }
}

}  // namespace dfl

using namespace dfl;

static int q8_run_rows(int M, int seq_rows, bool one_seq) {
  return one_seq ? M : seq_rows > 0 ? (seq_rows < M ? seq_rows : M) : 1;
}

// The form, tile rows and keys per chunk of a call.
// Few: runs of at most 16 (token, head) rows, and calls small enough that tiles of 16 rows with 384 keys each
// fit one wave (three CTAs an SM; at head_dim 256 one, of 32 rows where there are more than 16). They take the
// warp form in such tiles, for their latency: one sequence of 1024 keys, 16 tokens of 32 heads of 128, 10.3 us
// when chosen (64-row tiles 15.2, tcgen05 16.2), 9.4 since Q is loaded beside the positions; 4096 keys 16.0
// (20.5, 16.5), now 14.9.
// Others take a tcgen05 form, tc of 64 rows a CTA: four such sequences of 2048 keys 18.3 us (16-row tiles 28.5,
// 64-row 21.3), 64 of 512 to 4096 keys 119 (338 in 64-row tiles); 64 single tokens 107, in the warp form 61.
// Wide, of 256 rows (head_dim 256: 128), for runs that fill more than half of them and calls with a CTA, or 384
// keys, for every SM: 128 rows of 32 heads at 4096 keys 28 us (tc 36), at 1024 27 (16); 8 sequences of 512 to
// 6000 keys, 16 tokens of 24 heads of 256, 46 us (tc 55). Also where tc would take a second wave (25
// sequences of 51 keys, 16 tokens of 32 heads of 256: 15 us, tc 22; 48 of 99, 82 tokens of 8 heads of 64: 14, 20).
// Chunks: as many as keep every CTA in one wave (tc: two an SM, at head_dim 256 and wide one), one more for
// several runs (warp form: that have four and more; tc: unless it makes them two where the CTAs nearly fill the
// wave), as their lengths may differ (those 8 sequences in tc: 55 us with it, 71 without). Runs of one chunk in
// the warp form and half to 1.35 waves: long ones are cut so that their rest fills the SMs at the end, in halves
// up to 0.8 waves (single tokens of 36 sequences of 512 to 4096 keys 55 -> 45 us, all of 4096 76 -> 72), at three
// quarters beyond (64 sequences 72 -> 64, all of 4096 117 -> 104; 52 of 4096 82 -> 86). One chunk needs no merge,
// and each costs the merge and its CTA's start: at least 128 keys, 256 where those make more than 8 chunks (one
// token, 4096 keys: 9.2 us, with 128 11.1; 1536 keys: 8.4 and 8.0, with 16 tokens and a cold L2 18.4 and 20.5),
// in the tcgen05 forms 512, at most 64 chunks (one kv head, 2 tokens at 48k keys: 15 us, in 190 chunks 24), and no
// split of 512 keys where half the SMs have a CTA (four sequences, 16 tokens: 11.1 us, split in two 13.6). At most
// 8192 keys for every full wave, so that the last wave is a small part of the whole: 2048 prompt rows at 65536 keys
// 2.82 ms (uncut 3.03), 64 sequences of 16384, 16 tokens, 0.74 (0.76); and no more chunks than that, as each
// holds its partials in the scratch: 16384 rows at 65536 keys 19.8 ms in one, 19.7 and 2 GB in eight; 256 single
// tokens of 512 to 16384 keys 0.76 ms, 0.80 in two.
struct Q8Plan {
  int form, rows, key_chunk, n_chunks;  // rows: (token, head) pairs a CTA takes
};
static Q8Plan q8_plan(int form, int key_chunk, long long runs, int run_rows, int G, int Hkv, int hd, int max_kv) {
  Q8Plan p;
  const long long want = (long long)run_rows * G, wave = 148 * (hd == 256 ? 1 : 3);
  auto units = [&](int rows) { return runs * Hkv * ((run_rows + rows / G - 1) / (rows / G)); };
  const int small = hd == 256 && want > 16 ? 32 : 16;
  const bool few = want <= 16 || (units(small) <= wave && units(small) * max_kv <= wave * 384);
  const int wide = hd == 256 ? 128 : 256;
  const long long tc_wave = 148 * (hd == 256 ? 1 : 2);
  const bool busy = units(wide) * (max_kv < 384 ? 384 : max_kv) >= 148 * 384LL || units(64) > tc_wave;
  if (form != DFL_Q8_AUTO) p.form = form;
  else if (few) p.form = DFL_Q8_WARP;
  else p.form = want > wide / 2 && busy ? DFL_Q8_WIDE : DFL_Q8_TC;
  const bool tc = p.form >= DFL_Q8_TC;
  p.rows = p.form == DFL_Q8_WIDE ? wide : tc ? 64 : few ? small : want <= 32 || hd == 256 ? 32 : 64;
  if (key_chunk <= 0) {
    const long long slots = tc ? (p.rows == 64 ? tc_wave : 148) : p.rows == 64 ? 148 : wave, u = units(p.rows);
    long long n = slots / u + (runs > 1 && (tc ? slots % u != 0 && 4 * slots >= 5 * u : slots >= 4 * u) ? 1 : 0);
    if (!tc && u > 74 && max_kv <= 512) n = 1;
    if (n > 64) n = 64;
    const long long lo = tc ? 512 : max_kv <= 8 * Q8_CHUNK_UNIT ? Q8_CHUNK_UNIT : 256;
    long long c = n > 1 ? (max_kv + n - 1) / n : max_kv;
    if (!tc && n <= 1 && runs > 1 && max_kv >= 2048 && 20 * u <= 27 * slots)
      c = 5 * u <= 4 * slots ? (max_kv + 1) / 2 : (3LL * max_kv + 3) / 4;
    const long long hi = u < 2 * slots ? 8192 : u < 128 * slots ? 8192 * (u / slots) : 1 << 20;
    c = c < lo ? lo : c > hi ? hi : c;
    key_chunk = (int)((c + Q8_CHUNK_UNIT - 1) / Q8_CHUNK_UNIT * Q8_CHUNK_UNIT);
  }
  p.key_chunk = key_chunk;
  p.n_chunks = (int)(((long long)max_kv + key_chunk - 1) / key_chunk);
  return p;
}

static size_t q8_workspace(int M, int Hq, int hd, int n_chunks) {
  if (n_chunks <= 1) return 0;
  const size_t o = (size_t)n_chunks * M * Hq * hd * sizeof(float);
  return ((o + 255) & ~(size_t)255) + (size_t)n_chunks * M * Hq * sizeof(float2);
}

extern "C" size_t dfl_attention_q8_workspace_bytes(const dfl_kv_q8* cache, int M, int Hq, int seq_rows, int one_seq,
                                                   int max_kv, int form, int key_chunk) {
  if (!cache || M <= 0 || Hq <= 0 || max_kv <= 0 || key_chunk < 0 || key_chunk % Q8_CHUNK_UNIT ||
      cache->n_kv_heads <= 0 || Hq % cache->n_kv_heads || Hq / cache->n_kv_heads > 16 || form < DFL_Q8_AUTO ||
      form > DFL_Q8_WIDE)
    return 0;
  const int rr = q8_run_rows(M, seq_rows, one_seq != 0);
  return q8_workspace(M, Hq, cache->head_dim,
                      q8_plan(form, key_chunk, (M + rr - 1) / rr, rr, Hq / cache->n_kv_heads, cache->n_kv_heads,
                              cache->head_dim, max_kv).n_chunks);
}

extern "C" int dfl_attention_q8(const void* q, const dfl_kv_q8* cache, const int32_t* pos, const int32_t* row_seq,
                                const int32_t* kv_len, int seq_rows, int M, int Hq, int causal, float scale,
                                int max_kv, int form, int key_chunk, void* out, int64_t ldo, const void* gate, int64_t ldg,
                                int gate_head_stride, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "dfl_attention_q8";
  if (M == 0) return DFL_OK;
  AttnQ8Args a;
  if (const int s = q8_cache(cache, who, &a.c)) return s;
  const int hd = cache->head_dim, Hkv = cache->n_kv_heads;
  if (!q || !pos || !out || (!causal && !kv_len) || M < 0 || Hq <= 0 || Hq % Hkv || max_kv <= 0 || seq_rows < 0) {
    set_error("%s: bad arguments (M=%d Hq=%d Hkv=%d max_kv=%d)", who, M, Hq, Hkv, max_kv);
    return DFL_ERR_INVALID;
  }
  const int G = Hq / Hkv;
  if (G > 16) {
    set_error("%s: query heads per kv head must be 1..16 (got %d)", who, G);
    return DFL_ERR_UNSUPPORTED;
  }
  if (form < DFL_Q8_AUTO || form > DFL_Q8_WIDE) {
    set_error("%s: unknown form %d", who, form);
    return DFL_ERR_INVALID;
  }
  if (key_chunk < 0 || key_chunk % Q8_CHUNK_UNIT) {
    set_error("%s: key_chunk %d must be a multiple of %d", who, key_chunk, Q8_CHUNK_UNIT);
    return DFL_ERR_INVALID;
  }
  if (!(scale == scale) || scale - scale != 0.f) {
    set_error("%s: the softmax scale must be finite", who);
    return DFL_ERR_INVALID;
  }
  if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(out) % 8 || ldo % 4 ||
      ldo < (int64_t)Hq * hd) {
    set_error("%s: q must be 16-byte and out 8-byte aligned, ldo a multiple of 4 and at least Hq * hd (ldo=%lld)",
              who, (long long)ldo);
    return DFL_ERR_UNSUPPORTED;
  }
  const int run_rows = q8_run_rows(M, seq_rows, row_seq == nullptr);
  const int runs = (M + run_rows - 1) / run_rows;
  const Q8Plan plan = q8_plan(form, key_chunk, runs, run_rows, G, Hkv, hd, max_kv);
  a.key_chunk = plan.key_chunk;
  a.n_chunks = plan.n_chunks;
  if (a.n_chunks > 65535) {
    set_error("%s: %d key chunks; a larger key_chunk is needed", who, a.n_chunks);
    return DFL_ERR_UNSUPPORTED;
  }
  const size_t need = q8_workspace(M, Hq, hd, a.n_chunks);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)) {
    set_error("%s: workspace missing, misaligned or too small (%zu < %zu)", who, workspace_bytes, need);
    return DFL_ERR_WORKSPACE;
  }
  const bool tc = plan.form >= DFL_Q8_TC;
  const int rows = plan.rows;
  a.run_rows = run_rows;
  a.run_tiles = (run_rows + rows / G - 1) / (rows / G);
  a.tile_toks = (run_rows + a.run_tiles - 1) / a.run_tiles;
  const long long tiles = (long long)runs * a.run_tiles;
  a.runs = runs;
  a.ranked = runs > 1 && runs <= Q8_RANK_RUNS && tiles * Hkv * a.n_chunks > 148;
  if (tiles * Hkv > 0x7fffffffLL) {
    set_error("%s: too many rows (%d)", who, M);
    return DFL_ERR_UNSUPPORTED;
  }
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.pos = pos;
  a.row_seq = row_seq;
  a.kv_len = kv_len;
  a.part_o = static_cast<float*>(workspace);
  const size_t o_bytes = (size_t)a.n_chunks * M * Hq * hd * sizeof(float);
  a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + ((o_bytes + 255) & ~(size_t)255));
  a.out = static_cast<__nv_bfloat16*>(out);
  a.ldo = ldo;
  a.gate = static_cast<const __nv_bfloat16*>(gate);
  a.ldg = ldg;
  a.gate_hs = gate_head_stride > 0 ? gate_head_stride : hd;
  a.M = M;
  a.Hq = Hq;
  a.G = G;
  a.causal = causal;
  a.max_kv = max_kv;
  a.q_sign = scale > 0.f ? 1.f : scale < 0.f ? -1.f : 0.f;
  a.scale_log2 = scale == 0.f ? 1.f : (scale < 0.f ? -scale : scale) * 1.4426950408889634f;
  a.err = device_error_word();
  cudaStream_t st = as_stream(stream);
  const bool e4 = cache->type == DFL_KV_E4M3;
  int status;
  if (tc) {
    status = launch_attention_q8_tc(a, hd, e4, rows, (int)tiles, st);
  } else if (hd == 64) {
    status = e4 ? launch_attn_q8_rows<64, true>(a, rows, (int)tiles, st) : launch_attn_q8_rows<64, false>(a, rows, (int)tiles, st);
  } else if (hd == 128) {
    status = e4 ? launch_attn_q8_rows<128, true>(a, rows, (int)tiles, st) : launch_attn_q8_rows<128, false>(a, rows, (int)tiles, st);
  } else {
    status = e4 ? launch_attn_q8_rows<256, true>(a, rows, (int)tiles, st) : launch_attn_q8_rows<256, false>(a, rows, (int)tiles, st);
  }
  if (status != DFL_OK || a.n_chunks == 1) return status;
  return hd == 64 ? launch_attn_q8_merge<64>(a, st) : hd == 128 ? launch_attn_q8_merge<128>(a, st) : launch_attn_q8_merge<256>(a, st);
}
