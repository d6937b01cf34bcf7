// What the kernels of attention over pages of 4 bits share: the word between portions and single tokens that run beside them, and the second
// kernel where keys are cut, behind the kernel of any number of rows (attention_q4.cu) and the tensor cores' (attention_q4_tc.cu): the parts of
// a row's cuts become its output.
//
// Parts: [token][head][place]: maximum (in powers of two) and sum, and D outputs not yet divided; a place a cut and, with kept first keys,
// one more for those.
#pragma once

#include "attention_combine.cuh"

namespace {

// A step's portions and its single tokens share nothing but what went before both.  The portions' kernel waits for that and lets the single
// tokens' one begin, which may not wait in its turn (its wait is for the portions' end).  What makes the writes before both visible to it is
// therefore this word: 1 is released by the portions' kernel behind its wait and acquired by each block of the single tokens' kernel in front of
// its first dependent read; a block that does not find it waits for the portions' end instead, which is always right.  The single tokens' kernel
// takes the word back behind its own wait (a block of its that begins later finds the portions ended), so that 1 is this launch's and no other's.
__device__ __forceinline__ void release_word(int* word, int value) {
  asm volatile("st.release.gpu.global.s32 [%0], %1;" ::"l"(word), "r"(value) : "memory");
}
__device__ __forceinline__ int acquire_word(const int* word) {
  int value;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(value) : "l"(word) : "memory");
  return value;
}

struct JoinParams {
  const float* ml;
  const float* parts;
  void* out;                  // [tokens, heads, d]
  const int* positions;       // [tokens]
  const int* covered;         // how many tokens belong to entries: rows of others stay as they are
  const float* sink_values;
  const float* gate;
  long long gate_stride;
  int gate_per_head, sink, num_tokens, num_heads, window, keep_first, chunk, num_splits;
};

// A warp a (token, head) row; only places whose keys the row sees were written for it.  28,672 rows of 128 in two cuts (29 MB of parts) take
// 12 us, where a block of 128 threads a row takes 60.
template <int D, typename T>
__global__ void __launch_bounds__(256) attention_q4_join_rows_kernel(const JoinParams p) {
  constexpr int kOwn = D / 32;
  pdl_launch_dependents();
  const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int token = static_cast<int>(min(row / p.num_heads, static_cast<long long>(p.num_tokens))), head = static_cast<int>(row % p.num_heads);
  if (token >= min(p.num_tokens, __ldcg(p.covered))) {     // (in front of the wait: from L2, whatever this multiprocessor has read before)
    if (row == 0) pdl_wait();      // (a grid that finds nothing to do must not end before the kernels ahead)
    return;
  }
  const int position = __ldcg(p.positions + token), visible = first_visible_key(position, p.window);
  const int places = p.num_splits + (p.keep_first > 0 ? 1 : 0);
  const int first = visible / p.chunk, window_last = min(p.num_splits - 1, position / p.chunk);
  const int count = window_last - first + 1 + (min(p.keep_first, visible) > 0 ? 1 : 0);      // the kept keys' place comes last
  const auto place_of = [&](int i) { return row * places + (first + i > window_last ? p.num_splits : first + i); };
  pdl_wait();
  const float2* ml = reinterpret_cast<const float2*>(p.ml);
  float best = -INFINITY;
  for (int i = lane; i < count; i += 32) best = fmaxf(best, ml[place_of(i)].x);
  best = warp_max(best);
  float total = 0.0f, x[kOwn];
#pragma unroll
  for (int c = 0; c < kOwn; ++c) x[c] = 0.0f;
#pragma unroll 4
  for (int i = 0; i < count; ++i) {
    const long long at = place_of(i);
    const float2 part = ml[at];
    const float w = part.x == -INFINITY ? 0.0f : exp2f(part.x - best);      // -inf: a cut that held no key of the row
    const float* from = p.parts + at * D + lane * kOwn;
    total += part.y * w;
    if constexpr (kOwn == 4) {
      const float4 v = *reinterpret_cast<const float4*>(from);
      x[0] += v.x * w, x[1] += v.y * w, x[2] += v.z * w, x[3] += v.w * w;
    } else {
      const float2 v = *reinterpret_cast<const float2*>(from);
      x[0] += v.x * w, x[1] += v.y * w;
    }
  }
  if (p.sink) total += exp2f((p.sink_values ? p.sink_values[head] * 1.4426950408889634f : 0.0f) - best);
  const float* gate = p.gate ? p.gate + static_cast<size_t>(token) * p.gate_stride + (p.gate_per_head ? head : head * D + lane * kOwn) : nullptr;
#pragma unroll
  for (int c = 0; c < kOwn; ++c) {
    x[c] /= total;
    if (gate) x[c] *= 1.0f / (1.0f + expf(-gate[p.gate_per_head ? 0 : c]));
  }
  T* to = static_cast<T*>(p.out) + row * D + lane * kOwn;
  if constexpr (kOwn == 4) {
    store_four_as<T>(to, x[0], x[1], x[2], x[3]);
  } else if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(x[0], x[1]);
  } else {
    *reinterpret_cast<float2*>(to) = make_float2(x[0], x[1]);
  }
}

template <int D, typename T>
int launch_join(const JoinParams& p, cudaStream_t stream) {
  const long long blocks = (static_cast<long long>(p.num_tokens) * p.num_heads + 7) / 8;
  if (blocks > 0x7fffffffLL) return VIPERA_BAD_SHAPE;
  return vipera_launch(attention_q4_join_rows_kernel<D, T>, dim3(static_cast<unsigned>(blocks)), 256, 0, stream, p);
}

}  // namespace
