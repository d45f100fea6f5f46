// Writing and reading the 8-bit K/V cache.
//
//  * dfl_qkv_rope_append_q8 - per-head q/k RMSNorm, RoPE and the append that quantises each key
//                             and value row as it is written
//  * dfl_kv_read_q8         - cache rows back as bf16
//
// A row of hd values x is held as codes c and one fp32 scale s, x ~ c * s (int8: s = max|x| / 127;
// e4m3: max|x| / 448). Both kernels are bound by memory: per row the append reads the
// projection's (Hq + 2 Hkv) * hd bf16 values and writes Hq * hd bf16 and 2 Hkv (hd + 4) bytes.
#include "kv_q8.cuh"

namespace dfl {

int q8_cache(const dfl_kv_q8* c, const char* who, Q8Cache* out) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) {
    set_error("%s: null cache, codes or scales", who);
    return DFL_ERR_INVALID;
  }
  if (c->type != DFL_KV_INT8 && c->type != DFL_KV_E4M3) {
    set_error("%s: cache type %d is neither DFL_KV_INT8 nor DFL_KV_E4M3", who, c->type);
    return DFL_ERR_INVALID;
  }
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
    set_error("%s: head_dim %d not supported (64, 128, 256)", who, c->head_dim);
    return DFL_ERR_UNSUPPORTED;
  }
  if (c->n_kv_heads <= 0 || c->n_kv_heads > 65535 || c->n_seqs <= 0 || c->cap <= 0 || c->seq_stride < 0 ||
      c->head_stride < 0 || c->scale_seq_stride < 0 || c->scale_head_stride < 0) {
    set_error("%s: bad cache geometry (Hkv=%d n_seqs=%d cap=%d)", who, c->n_kv_heads, c->n_seqs, c->cap);
    return DFL_ERR_INVALID;
  }
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16 || c->seq_stride % 16 ||
      c->head_stride % 16) {
    set_error("%s: cache codes must be 16-byte aligned, with strides that are multiples of 16", who);
    return DFL_ERR_UNSUPPORTED;
  }
  int shift = 0;
  if (c->page_table) {
    if (c->page_size < 64 || (c->page_size & (c->page_size - 1)) || c->pt_stride <= 0 || c->n_pages <= 0) {
      set_error("%s: page_size must be a power of two >= 64 (got %d), with pages and a table stride", who,
                c->page_size);
      return DFL_ERR_INVALID;
    }
    while ((1 << shift) < c->page_size) ++shift;
  }
  out->k = static_cast<unsigned char*>(c->k);
  out->v = static_cast<unsigned char*>(c->v);
  out->ks = c->k_scale;
  out->vs = c->v_scale;
  out->seq_stride = c->seq_stride;
  out->head_stride = c->head_stride;
  out->s_seq_stride = c->scale_seq_stride;
  out->s_head_stride = c->scale_head_stride;
  out->page_table = c->page_table;
  out->pt_stride = c->pt_stride;
  out->page_shift = shift;
  out->n_seqs = c->n_seqs;
  out->n_pages = c->n_pages;
  out->cap = c->cap;
  out->Hkv = c->n_kv_heads;
  return DFL_OK;
}

// ---------------------------------------------------------------------------
// Append. hd / 8 lanes per head, eight values each, so a warp holds 256 / hd heads (a slot) at a time and a
// head's sums take log2(hd / 8) shuffles. A CTA takes ROWS rows: its threads make the rows' (cos, sin)
// tables together, then 8 / ROWS warps walk each row's slots. One row: its slots spread over CTAs (a slot a
// warp, for latency). Two and four: a warp has four slots in flight through shared memory.
// With many rows the issue of instructions bounds it before memory does, so a lane of the rotated dims holds four
// values of the first half and their partners of the second (the rotation needs no other lane), the arithmetic
// runs two values an instruction, and slots of q heads alone have a loop of their own. 16384 rows of
// 32 + 16 heads of 128, int8: 82 us, 4.5 TB/s (eight consecutive values a lane, partners by shuffle, one value an
// instruction, one slot in flight: 135 us; the lane layout and pairs alone: 111; the ring: 97; the q loop: 80; codes
// that are right at a half, two more instructions for four values: 82).
// ---------------------------------------------------------------------------
struct AppendQ8Args {
  const __nv_bfloat16* qkv;
  long long ldqkv;
  int q_stride;
  const int* pos;
  const int* row_seq;
  const __nv_bfloat16* q_norm;
  const __nv_bfloat16* k_norm;
  const float* inv_freq;
  __nv_bfloat16* q_out;
  Q8Cache c;
  int M, Hq, rot_dim;
  int first_head;  // 0, or Hq when the q heads are left out
  int slots_per_cta;
  float eps;
  int* err;
};

constexpr int APPEND_WARPS = 8;
constexpr int APPEND_RING = 4;  // slots a warp has in flight (forms of several rows)

// cos and sin of p * f: the product and its reduction by turns in fp64 (an fp32 product is off by
// 2^-24 p f, 0.008 rad at position 131072), the reduced angle in fp32.
__device__ __forceinline__ float2 rope_cos_sin(int p, float f) {
  const double a = (double)p * (double)f;
  const double turns = rint(a * 0.15915494309189535);  // 1 / (2 pi)
  float s, c;
  sincosf((float)fma(turns, -6.283185307179586, a), &s, &c);
  return make_float2(c, s);
}

// Codes of four values x * (up + lo), rounded to nearest even: int8 by an addition of 1.5 * 2^23, whose sum's low
// byte is the integer (|x * up| <= 127 up to rounding, so none is out of range). lo is what up leaves out of
// TOP / max|x|: bf16 values meet halves of a code often (half of an int8 row's maximum is code 63.5, three quarters
// of an e4m3 row's 336), and up's rounding alone would push one product in two off its half.
template <bool E4M3>
__device__ __forceinline__ uint32_t q8_codes4(uint64_t x01, uint64_t x23, uint64_t up, uint64_t lo) {
  const uint64_t y01 = q8_fma2(x01, up, q8_mul2(x01, lo)), y23 = q8_fma2(x23, up, q8_mul2(x23, lo));
  if constexpr (E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(q8_unpack(y01), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(q8_unpack(y23), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  } else {
    const uint64_t magic = q8_pack(12582912.f, 12582912.f);
    const float2 a = q8_unpack(q8_add2(y01, magic)), b = q8_unpack(q8_add2(y23, magic));
    return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040),
                       __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
  }
}

// two bf16 of a word as two fp32
__device__ __forceinline__ uint64_t q8_bf16x2(uint32_t u) {
  return q8_pack(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

template <int HD, bool E4M3, int ROWS>
__global__ void __launch_bounds__(32 * APPEND_WARPS, ROWS == 1 ? 1 : 4) append_q8_kernel(const __grid_constant__ AppendQ8Args a) {
  grid_dependency_launch_dependents();
  grid_dependency_wait();
  constexpr int LPH = HD / 8;               // lanes per head
  constexpr int HPW = 32 / LPH;             // heads per slot
  constexpr int WPR = APPEND_WARPS / ROWS;  // warps per row
  constexpr bool RINGED = ROWS > 1;
  __shared__ float2 cs[ROWS][HD / 2];
  __shared__ uint4 ring[RINGED ? APPEND_WARPS : 1][APPEND_RING][32];
  const int m0 = blockIdx.x * ROWS;
  const int half = a.rot_dim >> 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m = m0 + warp / WPR;
  const int p = m < a.M ? a.pos[m] : -1;
  const int sub = lane / LPH, l = lane % LPH;  // head within the slot, lane within the head
  const int Hkv = a.c.Hkv;
  const int n_heads = a.Hq + 2 * Hkv;
  // this lane's eight values: i .. i + 3 of both halves of the rotated dims, or eight behind those
  const bool turned = l < half / 4;
  const int d0 = turned ? 4 * l : a.rot_dim + 8 * (l - half / 4), d1 = d0 + (turned ? half : 4);
  const __nv_bfloat16* row = a.qkv + (long long)m * a.ldqkv;
  const long long kv0 = (long long)a.Hq * a.q_stride;
  auto head_at = [&](int h) { return row + (h < a.Hq ? (long long)h * a.q_stride : kv0 + (long long)(h - a.Hq) * HD); };
  auto load = [&](const __nv_bfloat16* x) -> uint4 {
    const uint2 lo = *reinterpret_cast<const uint2*>(x + d0), hi = *reinterpret_cast<const uint2*>(x + d1);
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
  const int slots = (n_heads + HPW - 1) / HPW;
  const int slot0 = a.first_head / HPW + blockIdx.y * a.slots_per_cta;
  const int slot_end = min(slots, slot0 + a.slots_per_cta);
  int slot = slot0 + warp % WPR;
  // one-row form: this warp's slot; four-row form: slot `s`, the i-th of this warp, into its place in the ring
  uint4 nx = make_uint4(0, 0, 0, 0);
  auto fetch = [&](int s, int i) {
    if (p >= 0 && s < slot_end) {
      const __nv_bfloat16* x = head_at(min(s * HPW + sub, n_heads - 1));
      if constexpr (RINGED) {
        cp_async16(smem_u32(&ring[warp][i % APPEND_RING][lane]), x + 8 * l, 16);
      } else {
        nx = load(x);
      }
    }
    if constexpr (RINGED) cp_async_commit();
  };
  if constexpr (RINGED) {
#pragma unroll
    for (int i = 0; i < APPEND_RING - 1; ++i) fetch(slot + i * WPR, i);
  } else {
    fetch(slot, 0);
  }
  // tables: thread t makes entries t, t + 256, ... of the CTA's rows
  for (int i = threadIdx.x; i < ROWS * half; i += 32 * APPEND_WARPS) {
    const int r = ROWS == 1 ? 0 : i / half, k = ROWS == 1 ? i : i - r * half;
    const int pr = m0 + r < a.M ? a.pos[m0 + r] : -1;
    if (pr >= 0) cs[r][k] = rope_cos_sin(pr, a.inv_freq[k]);
  }
  __syncthreads();
  if (p < 0 || slot >= slot_end) return;
  const int seq = a.row_seq ? a.row_seq[m] : 0;
  long long page = 0;
  int prow = 0;
  const bool placed = q8_place(a.c, seq, p, lane == 0 ? a.err : nullptr, page, prow);
  // x' = x cos - partner sin of the first half, x cos + partner sin of the second; other dims: cos 1, sin 0
  uint64_t cr[2], sp[2], sn[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float2 t0 = turned ? cs[warp / WPR][4 * l + 2 * j] : make_float2(1.f, 0.f);
    const float2 t1 = turned ? cs[warp / WPR][4 * l + 2 * j + 1] : make_float2(1.f, 0.f);
    cr[j] = q8_pack(t0.x, t1.x);
    sp[j] = q8_pack(t0.y, t1.y);
    sn[j] = q8_pack(-t0.y, -t1.y);
  }
  uint64_t w[4];  // the norm's weights
  auto weights = [&](const __nv_bfloat16* g) {
    const uint2 lo = *reinterpret_cast<const uint2*>(g + d0), hi = *reinterpret_cast<const uint2*>(g + d1);
    w[0] = q8_bf16x2(lo.x);
    w[1] = q8_bf16x2(lo.y);
    w[2] = q8_bf16x2(hi.x);
    w[3] = q8_bf16x2(hi.y);
  };
  const long long code0 = page * a.c.seq_stride + (long long)prow * HD;
  const long long scale0 = page * a.c.s_seq_stride + prow;
  int i = 0;  // the slot's number among this warp's
  auto take = [&](uint64_t (&x)[4]) {
    if constexpr (RINGED) {
      __syncwarp();  // every lane has read the place that this fetch fills
      fetch(slot + (APPEND_RING - 1) * WPR, i + APPEND_RING - 1);
      cp_async_wait<APPEND_RING - 1>();
      __syncwarp();
      nx = load(reinterpret_cast<const __nv_bfloat16*>(&ring[warp][i % APPEND_RING][sub * LPH]));
    }
    x[0] = q8_bf16x2(nx.x);
    x[1] = q8_bf16x2(nx.y);
    x[2] = q8_bf16x2(nx.z);
    x[3] = q8_bf16x2(nx.w);
  };
  auto inverse_norm = [&](const uint64_t (&x)[4]) -> float {
    uint64_t sq = q8_mul2(x[0], x[0]);
#pragma unroll
    for (int j = 1; j < 4; ++j) sq = q8_fma2(x[j], x[j], sq);
    const float2 s2 = q8_unpack(sq);
    float ss = s2.x + s2.y;
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    return rsqrtf(ss * (1.f / (float)HD) + a.eps);
  };
  auto turn = [&](uint64_t (&x)[4], float inv) {
    const uint64_t inv2 = q8_pack(inv, inv);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = q8_mul2(w[j], q8_mul2(x[j], inv2));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint64_t y = x[j], z = x[2 + j];
      x[j] = q8_fma2(y, cr[j], q8_mul2(z, sn[j]));
      x[2 + j] = q8_fma2(z, cr[j], q8_mul2(y, sp[j]));
    }
  };
  auto put_q = [&](const uint64_t (&x)[4], int h) {
    __nv_bfloat16* o = a.q_out + ((long long)m * a.Hq + h) * HD;
    const float2 f0 = q8_unpack(x[0]), f1 = q8_unpack(x[1]), f2 = q8_unpack(x[2]), f3 = q8_unpack(x[3]);
    *reinterpret_cast<uint2*>(o + d0) = make_uint2(pack_bf16x2(f0.x, f0.y), pack_bf16x2(f1.x, f1.y));
    *reinterpret_cast<uint2*>(o + d1) = make_uint2(pack_bf16x2(f2.x, f2.y), pack_bf16x2(f3.x, f3.y));
  };
  // slots of q heads alone
  if (a.first_head == 0) {
    weights(a.q_norm);
    const int q_end = min(slot_end, a.Hq / HPW);
#pragma unroll 1
    for (; slot < q_end; slot += WPR, ++i) {
      uint64_t x[4];
      take(x);
      turn(x, inverse_norm(x));
      put_q(x, slot * HPW + sub);
    }
  }
  // the others: k and v heads, and a slot that begins with q heads
  if (slot < slot_end) weights(slot * HPW + sub < a.Hq ? a.q_norm : a.k_norm);
#pragma unroll 1
  for (; slot < slot_end; slot += WPR, ++i) {
    uint64_t x[4];
    take(x);
    const int h = slot * HPW + sub;
    const bool is_q = h < a.Hq, is_k = !is_q && h < a.Hq + Hkv;
    const bool live = h >= a.first_head && h < n_heads && (is_q || placed);
    if (slot * HPW < a.Hq + Hkv) {  // some head of the slot is a q or k head: norm and rotation
      const float inv = inverse_norm(x);
      if (is_q || is_k) turn(x, inv);
      if (is_q) {
        if (live) put_q(x, h);
        weights(a.k_norm);
      }
    }
    // the maximum magnitude as an unsigned comparison of the bits, in which a NaN or an
    // infinity is larger than every finite value
    unsigned am = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = q8_unpack(x[j]);
      am = max(am, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
    }
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) am = max(am, __shfl_xor_sync(0xffffffffu, am, o));
    if (!is_q && live) {
      constexpr float TOP = E4M3 ? 448.f : 127.f;
      const bool finite = am < 0x7f800000u;
      const float amax = __uint_as_float(am);
      // below 2^-119 the reciprocal would overflow: such a row is all but zero, and is held as zeros
      const bool some = finite && amax >= 1.5046328e-36f;
      const float up = some ? __fdiv_rn(TOP, amax) : 0.f;
      const float scale = finite ? (some ? __fdiv_rn(amax, TOP) : 0.f) : __uint_as_float(0x7fc00000u);
      const float lo = fmaf(-up, amax, TOP) * (up * (1.f / TOP));  // the remainder is exact, 1 / amax near enough
      const uint64_t up2 = q8_pack(up, up), lo2 = q8_pack(lo, lo);
      const uint32_t c0 = some ? q8_codes4<E4M3>(x[0], x[1], up2, lo2) : 0u;
      const uint32_t c1 = some ? q8_codes4<E4M3>(x[2], x[3], up2, lo2) : 0u;
      const int kh = h - a.Hq - (is_k ? 0 : Hkv);
      unsigned char* codes = (is_k ? a.c.k : a.c.v) + code0 + kh * a.c.head_stride;
      *reinterpret_cast<uint32_t*>(codes + d0) = c0;
      *reinterpret_cast<uint32_t*>(codes + d1) = c1;
      if (l == 0) (is_k ? a.c.ks : a.c.vs)[scale0 + kh * a.c.s_head_stride] = scale;
    }
  }
}

// ---------------------------------------------------------------------------
// Read-back: one thread per 16 codes of a key row and of the value row of the same place.
// Bound by memory: 32 sequences' 588 MB of bf16 rows from 303 MB of codes and scales in 159 us, 86 % of the copy rate.
// ---------------------------------------------------------------------------
struct ReadQ8Args {
  Q8Cache c;
  const int* pos;
  const int* row_seq;
  __nv_bfloat16* k_out;
  __nv_bfloat16* v_out;
  long long n;  // threads with work: M * Hkv * hd / 16
  int* err;
};

template <bool E4M3>
__device__ __forceinline__ void q8_values4(uint32_t w, float (&f)[4]) {
  if (E4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3);
      const float2 v = __half22float2(__half2(h));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(signed char)(w >> (8 * i));
  }
}

template <int HD, bool E4M3>
__global__ void __launch_bounds__(256) read_q8_kernel(const __grid_constant__ ReadQ8Args a) {
  grid_dependency_launch_dependents();
  grid_dependency_wait();
  constexpr int CPR = HD / 16;  // 16-code chunks per row
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.n) return;
  const int c = (int)(i % CPR);
  const long long mh = i / CPR;
  const int h = (int)(mh % a.c.Hkv);
  const int m = (int)(mh / a.c.Hkv);
  const int p = a.pos[m];
  if (p < 0) return;
  long long page;
  int row;
  if (!q8_place(a.c, a.row_seq ? a.row_seq[m] : 0, p, c == 0 && h == 0 ? a.err : nullptr, page, row)) return;
  const long long off = page * a.c.seq_stride + h * a.c.head_stride + (long long)row * HD + c * 16;
  const long long soff = page * a.c.s_seq_stride + h * a.c.s_head_stride + row;
  const uint4 kw = __ldg(reinterpret_cast<const uint4*>(a.c.k + off));
  const uint4 vw = __ldg(reinterpret_cast<const uint4*>(a.c.v + off));
  const float ks = __ldg(a.c.ks + soff), vs = __ldg(a.c.vs + soff);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint4 w = t ? vw : kw;
    const float s = t ? vs : ks;
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    uint32_t o[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float f[4];
      q8_values4<E4M3>(u[q], f);
      o[2 * q] = pack_bf16x2(f[0] * s, f[1] * s);
      o[2 * q + 1] = pack_bf16x2(f[2] * s, f[3] * s);
    }
    uint4* dst = reinterpret_cast<uint4*>((t ? a.v_out : a.k_out) + mh * HD + c * 16);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

template <typename A>
static int launch_q8(void (*kernel)(A), const A& a, dim3 grid, int threads, const char* who, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) {
    set_error("%s: launch failed: %s", who, cudaGetErrorString(e));
    return DFL_ERR_CUDA;
  }
  return DFL_OK;
}

}  // namespace dfl

using namespace dfl;

static bool misaligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

extern "C" int dfl_qkv_rope_append_q8(const void* qkv, int64_t ldqkv, int q_stride, const int32_t* pos,
                                      const int32_t* row_seq, const void* q_norm, const void* k_norm,
                                      const float* inv_freq, void* q_out, const dfl_kv_q8* cache, int M, int Hq,
                                      int rot_dim, float eps, int do_q, void* stream) {
  const char* who = "dfl_qkv_rope_append_q8";
  if (M == 0) return DFL_OK;
  AppendQ8Args a;
  if (const int s = q8_cache(cache, who, &a.c)) return s;
  const int hd = cache->head_dim;
  if (!qkv || !pos || !k_norm || (rot_dim > 0 && !inv_freq) || (do_q && (!q_out || !q_norm)) || M < 0 || Hq < 0) {
    set_error("%s: null pointer or negative size", who);
    return DFL_ERR_INVALID;
  }
  if (rot_dim < 0 || rot_dim > hd || rot_dim % 16) {
    set_error("%s: rot_dim %d must be a multiple of 16, at most head_dim", who, rot_dim);
    return DFL_ERR_UNSUPPORTED;
  }
  if (misaligned16(qkv) || misaligned16(k_norm) || (do_q && (misaligned16(q_norm) || misaligned16(q_out))) ||
      ldqkv % 8 || q_stride % 8 || q_stride < (Hq ? hd : 0) ||
      ldqkv < (int64_t)Hq * q_stride + 2 * (int64_t)cache->n_kv_heads * hd) {
    set_error("%s: rows, norm weights and q_out must be 16-byte aligned and ldqkv cover a row (ldqkv=%lld)", who,
              (long long)ldqkv);
    return DFL_ERR_UNSUPPORTED;
  }
  a.qkv = static_cast<const __nv_bfloat16*>(qkv);
  a.ldqkv = ldqkv;
  a.q_stride = q_stride;
  a.pos = pos;
  a.row_seq = row_seq;
  a.k_norm = static_cast<const __nv_bfloat16*>(k_norm);
  a.q_norm = do_q ? static_cast<const __nv_bfloat16*>(q_norm) : a.k_norm;
  a.inv_freq = inv_freq;
  a.q_out = static_cast<__nv_bfloat16*>(q_out);
  a.M = M;
  a.Hq = Hq;
  a.rot_dim = rot_dim;
  a.first_head = do_q ? 0 : Hq;
  a.eps = eps;
  a.err = device_error_word();
  const int per_slot = 256 / hd;
  const int slots = (Hq + 2 * cache->n_kv_heads + per_slot - 1) / per_slot;
  // Up to about four CTAs an SM: one row each, its slots over CTAs of eight. Beyond: two rows a CTA, with more
  // than 16 rows an SM four, whose tables cost less a row (24 + 8 heads of 256: 256 rows 6.4 us
  // with two, 10.4 with four; 1024 10.5 and 12.4; 16384 105 and 98).
  const int groups = (slots - a.first_head / per_slot + APPEND_WARPS - 1) / APPEND_WARPS;
  const int rows = (long long)M * groups <= 148 * 4 ? 1 : M <= 148 * 16 ? 2 : 4;
  a.slots_per_cta = rows == 1 ? APPEND_WARPS : slots;
  const dim3 grid((M + rows - 1) / rows, rows == 1 ? groups : 1);
  cudaStream_t st = as_stream(stream);
  const int thr = 32 * APPEND_WARPS;
  const bool e4 = cache->type == DFL_KV_E4M3;
#define APPEND_Q8_T(HD, E4)                                                      \
  return launch_q8(rows == 1   ? append_q8_kernel<HD, E4, 1>                    \
                   : rows == 2 ? append_q8_kernel<HD, E4, 2>                    \
                               : append_q8_kernel<HD, E4, 4>,                   \
                   a, grid, thr, who, st)
#define APPEND_Q8(HD)         \
  if (e4) APPEND_Q8_T(HD, true); \
  APPEND_Q8_T(HD, false)
  switch (hd) {
    case 64: APPEND_Q8(64);
    case 128: APPEND_Q8(128);
    default: APPEND_Q8(256);
  }
#undef APPEND_Q8
#undef APPEND_Q8_T
}

extern "C" int dfl_kv_read_q8(const dfl_kv_q8* cache, const int32_t* pos, const int32_t* row_seq, int M, void* k_out,
                              void* v_out, void* stream) {
  const char* who = "dfl_kv_read_q8";
  if (M == 0) return DFL_OK;
  ReadQ8Args a;
  if (const int s = q8_cache(cache, who, &a.c)) return s;
  if (!pos || !k_out || !v_out || M < 0) {
    set_error("%s: null pointer or negative size", who);
    return DFL_ERR_INVALID;
  }
  if (misaligned16(k_out) || misaligned16(v_out)) {
    set_error("%s: outputs must be 16-byte aligned", who);
    return DFL_ERR_UNSUPPORTED;
  }
  const int hd = cache->head_dim;
  a.pos = pos;
  a.row_seq = row_seq;
  a.k_out = static_cast<__nv_bfloat16*>(k_out);
  a.v_out = static_cast<__nv_bfloat16*>(v_out);
  a.n = (long long)M * cache->n_kv_heads * (hd / 16);
  a.err = device_error_word();
  const long long blocks = (a.n + 255) / 256;
  if (blocks > 0x7fffffffLL) {
    set_error("%s: too many rows (%d)", who, M);
    return DFL_ERR_UNSUPPORTED;
  }
  const dim3 grid((unsigned)blocks);
  cudaStream_t st = as_stream(stream);
  const bool e4 = cache->type == DFL_KV_E4M3;
  switch (hd) {
    case 64: return launch_q8(e4 ? read_q8_kernel<64, true> : read_q8_kernel<64, false>, a, grid, 256, who, st);
    case 128: return launch_q8(e4 ? read_q8_kernel<128, true> : read_q8_kernel<128, false>, a, grid, 256, who, st);
    default: return launch_q8(e4 ? read_q8_kernel<256, true> : read_q8_kernel<256, false>, a, grid, 256, who, st);
  }
}
