// The 8-bit K/V cache (dfl_kv_q8) as the kernels see it: argument checks on the host, and on the
// device the place of a (sequence, position), bounds-checked, shared by the append and
// read-back (kv_q8.cu) and the attention (attention_q8.cu).
#pragma once
#include "common.cuh"
#include "tma_util.cuh"

#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace dfl {

constexpr int Q8_ERR_SEQ = 340;   // a row's sequence
constexpr int Q8_ERR_POS = 341;   // a position or key range
constexpr int Q8_ERR_PAGE = 342;  // a page number

struct Q8Cache {
  unsigned char* k;
  unsigned char* v;
  float* ks;
  float* vs;
  long long seq_stride, head_stride, s_seq_stride, s_head_stride;
  const int* page_table;
  long long pt_stride;
  int page_shift, n_seqs, n_pages, cap, Hkv;
};

// Checks a cache descriptor and fills the kernels' form of it; `who` names the entry point.
int q8_cache(const dfl_kv_q8* c, const char* who, Q8Cache* out);

__device__ __forceinline__ void q8_error(int* err, int code) {
  if (err) atomicCAS(err, 0, code);
}

// two fp32 operations an instruction
__device__ __forceinline__ uint64_t q8_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 q8_unpack(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t q8_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t q8_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t q8_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Page (or sequence) and row in it of position p of sequence seq; false, with the error word
// set, when one of them is out of range.
__device__ __forceinline__ bool q8_place(const Q8Cache& c, int seq, int p, int* err, long long& page, int& row) {
  if (seq < 0 || seq >= c.n_seqs) {
    q8_error(err, Q8_ERR_SEQ);
    return false;
  }
  if (p < 0 || p >= c.cap) {
    q8_error(err, Q8_ERR_POS);
    return false;
  }
  if (!c.page_table) {
    page = seq;
    row = p;
    return true;
  }
  page = c.page_table[seq * c.pt_stride + (p >> c.page_shift)];
  row = p & ((1 << c.page_shift) - 1);
  if (page < 0 || page >= c.n_pages) {
    q8_error(err, Q8_ERR_PAGE);
    return false;
  }
  return true;
}

}  // namespace dfl
