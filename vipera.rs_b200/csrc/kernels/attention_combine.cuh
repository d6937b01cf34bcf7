// The second kernel of split-key attention: partial results of an entry's splits become its output rows.  For
// the kernels over pages of bfloat16 (attention_mma.cu); those over pages of 4 bits take the keys a query sees from here.
//
// partial layout: [entry][head][place]: max (log2 units), sum, and D unnormalised outputs.
#pragma once

#include "common.cuh"

namespace {

// The first key a query at `position` sees.  window > 0: the last `window` keys; window < 0: a
// mask of chunks of -window positions counted from position 0 (the query sees the earlier keys
// of its own chunk); 0: every earlier key.
__device__ __forceinline__ int first_visible_key(int position, int window) {
  if (window > 0) return max(0, position - window + 1);
  if (window < 0) return position / (-window) * (-window);
  return 0;
}

// grid: (tokens, heads); one block of D threads combines the splits of one row.
// WIDE: the output is 32-bit (behind the VIRT instance, whose rows are mixed in 32-bit afterwards).
template <int D, bool KEPT = false, bool WIDE = false>
__global__ void attention_combine_kernel(const float* __restrict__ partial_ml, const float* __restrict__ partial_out,
                                         int slices, __nv_bfloat16* __restrict__ out, int num_heads,
                                         const int* __restrict__ positions, int window, int chunk,
                                         const int* __restrict__ entry_starts, int keep_first, int sink,
                                         const float* __restrict__ sink_values = nullptr,
                                         const float* __restrict__ gate = nullptr, long long gate_stride = 0,
                                         int gate_per_head = 0) {
  // KEPT instances also know a learned sink (`sink_values` [heads]: exp(sink_h) joins head h's sum
  // instead of one) and an output gate (`gate`: the row of the entry's token, at gate + token *
  // gate_stride, holds [heads * D] 32-bit pre-activations whose sigmoid multiplies the output; with
  // gate_per_head [heads] of them, one for all values of a head).
  // `slices` counts the window's splits; with kept first keys (keep_first > 0) each row has one
  // more place, the last, for the kept keys the window has left behind.  sink != 0: a key of score
  // 0 without a value joins the softmax, which adds exp2(-max) to the sum.
  __shared__ float maxima[130];
  __shared__ float sums[130];
  pdl_launch_dependents();
  // the step's description (written by the host before the step) is read before the wait
  const size_t row = static_cast<size_t>(blockIdx.x) * num_heads + blockIdx.y;
  size_t out_row = row;
  size_t out_token = blockIdx.x;
  if (entry_starts) {   // a step with portions: only entries of one token, written at their token's row
    const int token = entry_starts[blockIdx.x];
    if (entry_starts[blockIdx.x + 1] - token != 1) return;
    out_row = static_cast<size_t>(token) * num_heads + blockIdx.y;
    out_token = static_cast<size_t>(token);
  }
  const int places = slices + ((KEPT && keep_first > 0) ? 1 : 0);
  const float* ml = partial_ml + 2 * row * places;
  const float* values = partial_out + row * places * D + threadIdx.x;
  // only the splits that hold visible keys were written by the decode kernel
  const int position = positions[blockIdx.x];
  pdl_wait();
  const int first_visible = first_visible_key(position, window);
  const int first = (first_visible / 32 * 32) / chunk;
  const int window_last = min(slices - 1, position / chunk);
  // the kept keys' split holds keys when the window has left some of them behind; it is folded in
  // as the split after the window's last one (its partials are fetched from the row's last place)
  const bool kept = KEPT && keep_first > 0 && min(keep_first, first_visible) > 0;
  const int last = window_last + (kept ? 1 : 0);
  auto place_of = [&](int s) { return (kept && s == last) ? slices : s; };
  // Everything is asked for at once: this thread's column of every split's partial output (up to
  // kHeld of them stay in registers) beside all (max, sum) pairs, so that the combine costs one
  // trip to memory and not one per few splits; then the weights of the splits (at most 128 splits).
  constexpr int kHeld = 32;
  const int count = last - first + 1;
  float held[kHeld];
  if (count <= kHeld) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = i < count ? values[static_cast<size_t>(place_of(first + i)) * D] : 0.0f;
  }
  float mine = -INFINITY;
  for (int s = first + threadIdx.x; s <= last; s += D) {
    maxima[s] = ml[2 * place_of(s)];
    sums[s] = ml[2 * place_of(s) + 1];
  }
  __syncthreads();
  for (int s = first; s <= last; ++s) mine = fmaxf(mine, maxima[s]);
  float total = 0.0f, value = 0.0f;
  if (count <= kHeld) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      if (i < count) {
        const float m = maxima[first + i];
        const float w = m == -INFINITY ? 0.0f : exp2f(m - mine);  // a split that saw no key
        total += sums[first + i] * w;
        value += held[i] * w;
      }
    }
  } else {
#pragma unroll 8
    for (int s = first; s <= last; ++s) {
      const float m = maxima[s];
      const float w = m == -INFINITY ? 0.0f : exp2f(m - mine);
      total += sums[s] * w;
      value += values[static_cast<size_t>(place_of(s)) * D] * w;
    }
  }
  if (KEPT && sink) total += sink_values ? exp2f(sink_values[blockIdx.y] * 1.4426950408889634f - mine) : exp2f(-mine);   // the maxima are in units of log2
  float result = value / total;
  if (KEPT && gate) result *= 1.0f / (1.0f + expf(-gate[out_token * gate_stride + (gate_per_head ? static_cast<size_t>(blockIdx.y) : static_cast<size_t>(blockIdx.y) * D + threadIdx.x)]));
  if (WIDE) reinterpret_cast<float*>(out)[out_row * D + threadIdx.x] = result;
  else out[out_row * D + threadIdx.x] = __float2bfloat16_rn(result);
}

}  // namespace
