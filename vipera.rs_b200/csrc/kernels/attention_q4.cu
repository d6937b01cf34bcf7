// Attention of single tokens over pages of 4 bits (formats: q4.cuh), split over the keys, on mma.sync m16n8k16.
//
// A block is (entry, KV head and up to 8 NT of its query heads, split of the keys); its four warps fold 32 keys at a time each with a
// running (max, sum, output) and merge at the end; attention_combine_kernel joins the splits.
//
// Both products put the packed operand on the side of 16 (keys for the scores, channels for the values) and the query
// heads on the side of 8: a group of 8 heads or fewer costs half of the products that the other way round would
// waste on empty rows.  Codes become bfloat16 by a mask and an OR (0x4300 | u is 128 + u) and an exact subtraction of 136;
// the scales stay outside of them:
//   scores   the 32 channels of a group are one accumulator's two products, which the key's scale multiplies in 32
//            bits: s[key, head] = sum_g scale[key, g] (c[key, g, :] . q[head, g, :]), exact but for the 32-bit sums;
//   values   the weights take the scales, w[key, head, g] = p[key, head] scale[key, g], rounded to bfloat16 a second time (2^-9 of
//            the weight, as p itself): 2 products of pairs a group in the place of 16 on the codes.
// A score's accumulators have the keys on their rows, the second product wants them on its inner axis: movmatrix turns the
// weights' 8 x 8 blocks in registers, so nothing passes through shared memory until the end.
#include "attention_combine.cuh"
#include "attention_mma.cuh"
#include "q4.cuh"

namespace {

struct DecodeParams {
  const __nv_bfloat16* q;         // [rows, heads, d]
  __nv_bfloat16* out;
  const uint8_t *k_codes, *v_codes;
  const __nv_bfloat16 *k_scales, *v_scales;
  const int* positions;           // [entries]
  const int* block_table;
  const int* entry_starts;        // null: token i is entry i
  const float* sink_values;
  const float* gate;
  float* partial_ml;
  float* partial_out;
  long long gate_stride;
  int gate_per_head;
  int table_width, page_size, page_shift, num_pages, num_entries, num_heads, num_kv_heads, head_dim;
  float scale;
  int window, keep_first, sink, chunk, num_splits;
};

constexpr int kWarps = 4;
constexpr int kWarpKeys = 32;   // keys a warp folds at a time: two tiles of 16

__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// The codes at bits 4 j and 16 + 4 j of a word as two bfloat16.
__device__ __forceinline__ uint32_t codes_of(uint32_t word, int j) {
  return sub_bf16x2(((word >> (4 * j)) & 0x000f000fu) | 0x43004300u, 0x43084308u);
}
__device__ __forceinline__ uint32_t turn_8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float low_of(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float high_of(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

template <int WORDS>
__device__ __forceinline__ void load_words(uint32_t (&to)[WORDS], const void* from) {
  if constexpr (WORDS == 4) {
    const uint4 v = *static_cast<const uint4*>(from);
    to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
  } else if constexpr (WORDS == 2) {
    const uint2 v = *static_cast<const uint2*>(from);
    to[0] = v.x; to[1] = v.y;
  } else {
    to[0] = *static_cast<const uint32_t*>(from);
  }
}

// What a warp holds of 16 keys.  Lane 4 g + t: the keys' codes and scales of keys g and g + 8 (word t of every group), the
// values' of keys 2 t, 2 t + 1, 2 t + 8 and 2 t + 9 (unit g of every group).
template <int D>
struct Tile {
  static constexpr int G = D / 32;
  uint32_t k[2][G];            // [key g, g + 8][group]
  uint32_t k_scale[2][G / 2];  // pairs of groups
  uint32_t v[4][G / 2];        // [key][pair of groups]: a unit of 16 bits a group
  uint32_t v_scale[2][G];      // [pair of keys][first key's groups, second key's]
  int key0;                    // its first key; -1: nothing to see

  __device__ __forceinline__ void load(const DecodeParams& p, const int* table, int kv_head, int key, int first, int last, int lane) {
    key0 = -1;
    if (key > last || key + 15 < first) return;
    const int index = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
    if (index >= p.table_width) return;
    const int page = table[index];
    if (page < 0 || page >= p.num_pages) return;
    key0 = key;
    const size_t row = (static_cast<size_t>(page) * p.num_kv_heads + kv_head) * p.page_size + (key - index * p.page_size);
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const size_t at = row + g + 8 * r;
      load_words<G>(k[r], p.k_codes + at * (D / 2) + t * 4 * G);
      load_words<G / 2>(k_scale[r], p.k_scales + at * G);
      load_words<G>(v_scale[r], p.v_scales + (row + 2 * t + 8 * r) * G);
#pragma unroll
      for (int i = 0; i < 2; ++i) load_words<G / 2>(v[2 * r + i], p.v_codes + (row + 2 * t + 8 * r + i) * (D / 2) + g * 2 * G);
    }
  }
};

template <int D, int NT>
__global__ void __launch_bounds__(32 * kWarps) attention_q4_decode_kernel(DecodeParams p) {
  constexpr int G = D / 32;
  constexpr int kRow = D + 4;             // floats of a head's partial in shared memory
  extern __shared__ __align__(16) float merge[];   // [warp][8 NT heads][kRow]
  pdl_wait();
  // only now: the kernel behind reads the positions before its own wait, and they may come from the kernel ahead
  pdl_launch_dependents();
  const int group = p.num_heads / p.num_kv_heads, head_tiles = (group + 8 * NT - 1) / (8 * NT);
  const int entry = blockIdx.x, split = blockIdx.z;
  const int kv_head = blockIdx.y / head_tiles, head0 = (blockIdx.y - kv_head * head_tiles) * 8 * NT;
  int token = entry;
  if (p.entry_starts) {
    token = p.entry_starts[entry];
    if (p.entry_starts[entry + 1] - token != 1) return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int position = p.positions[entry];
  const int* table = p.block_table + static_cast<size_t>(entry) * p.table_width;
  const int window_first = first_visible_key(position, p.window);
  const bool kept_split = split == p.num_splits;   // the kept first keys that the window has left behind
  const int places = p.num_splits + (p.keep_first > 0 ? 1 : 0);
  const int first = kept_split ? 0 : window_first;
  const int last = kept_split ? min(p.keep_first, window_first) - 1 : position;
  const int begin = kept_split ? 0 : max(split * p.chunk, first / 32 * 32);
  const int end = kept_split ? last + 1 : min((split + 1) * p.chunk, position + 1);
  if (begin >= end) return;   // a split without visible keys: the combine kernel skips it too

  uint32_t q[NT][G][4];       // lane (g, t): channels 32 group + 8 t .. + 7 of head 8 nt + g
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int h = head0 + nt * 8 + g;
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      q[nt][gr][0] = q[nt][gr][1] = q[nt][gr][2] = q[nt][gr][3] = 0;
      if (h < group)
        load_words<4>(q[nt][gr], p.q + (static_cast<size_t>(token) * p.num_heads + kv_head * group + h) * D + 32 * gr + 8 * t);
    }
  }
  float o[NT][2 * G][4];      // channels 32 gr + 4 g + 2 h and the next (rows g, g + 8), heads 2 t and 2 t + 1
  float most[NT][2], sum[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    most[nt][0] = most[nt][1] = -INFINITY;
    sum[nt][0] = sum[nt][1] = 0.0f;
#pragma unroll
    for (int m = 0; m < 2 * G; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nt][m][i] = 0.0f;
  }
  const float scale_log2 = p.scale * kLog2e;

  for (int key0 = begin + warp * kWarpKeys; key0 < end; key0 += kWarps * kWarpKeys) {
    Tile<D> tile[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) tile[i].load(p, table, kv_head, key0 + 16 * i, first, last, lane);
    float s[2][NT][4];        // keys g (0, 1) and g + 8 (2, 3), heads 2 t and 2 t + 1; in units of log2
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[i][nt][c] = tile[i].key0 < 0 ? -INFINITY : 0.0f;
      if (tile[i].key0 < 0) continue;
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
        uint32_t a[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          a[half][0] = codes_of(tile[i].k[0][gr], 2 * half);
          a[half][1] = codes_of(tile[i].k[1][gr], 2 * half);
          a[half][2] = codes_of(tile[i].k[0][gr], 2 * half + 1);
          a[half][3] = codes_of(tile[i].k[1][gr], 2 * half + 1);
        }
        const uint32_t pair0 = tile[i].k_scale[0][gr / 2], pair1 = tile[i].k_scale[1][gr / 2];
        const float scale0 = gr & 1 ? high_of(pair0) : low_of(pair0), scale1 = gr & 1 ? high_of(pair1) : low_of(pair1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          mma_16816(acc, a[0], q[nt][gr][0], q[nt][gr][1]);
          mma_16816(acc, a[1], q[nt][gr][2], q[nt][gr][3]);
          s[i][nt][0] = fmaf(scale0, acc[0], s[i][nt][0]);
          s[i][nt][1] = fmaf(scale0, acc[1], s[i][nt][1]);
          s[i][nt][2] = fmaf(scale1, acc[2], s[i][nt][2]);
          s[i][nt][3] = fmaf(scale1, acc[3], s[i][nt][3]);
        }
      }
      const bool whole = tile[i].key0 >= first && tile[i].key0 + 15 <= last;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[i][nt][c] *= scale_log2;
      if (!whole) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int key = tile[i].key0 + g + 8 * r;
          if (key < first || key > last) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[i][nt][2 * r] = s[i][nt][2 * r + 1] = -INFINITY;
          }
          // a hidden key's weight is 0, and its scale must not make that NaN
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int value_key = tile[i].key0 + 2 * t + 8 * r + n;
            if (value_key < first || value_key > last) {
#pragma unroll
              for (int w = 0; w < G / 2; ++w) tile[i].v_scale[r][n * (G / 2) + w] = 0;
            }
          }
        }
      }
    }
    // the running maximum of each head, over the eight lanes that hold its keys
    float now[NT][2], safe[NT][2];
    bool grown = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float m = fmaxf(fmaxf(s[0][nt][c], s[0][nt][2 + c]), fmaxf(s[1][nt][c], s[1][nt][2 + c]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        now[nt][c] = m = fmaxf(m, most[nt][c]);
        safe[nt][c] = m == -INFINITY ? 0.0f : m;
        grown = grown || m > most[nt][c];
      }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float shrink = exp2f(most[nt][c] - safe[nt][c]);
          sum[nt][c] *= shrink;
#pragma unroll
          for (int m = 0; m < 2 * G; ++m) {
            o[nt][m][c] *= shrink;
            o[nt][m][2 + c] *= shrink;
          }
          most[nt][c] = now[nt][c];
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (tile[i].key0 < 0) continue;
      uint32_t w[NT][2];      // weights of head g: keys 2 t, 2 t + 1 and 2 t + 8, 2 t + 9
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float weight[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          weight[c] = exp2f(s[i][nt][c] - safe[nt][c & 1]);
          sum[nt][c & 1] += weight[c];
        }
        w[nt][0] = turn_8x8(pack_bf16(weight[0], weight[1]));
        w[nt][1] = turn_8x8(pack_bf16(weight[2], weight[3]));
      }
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
        uint32_t pairs[2], scales[2];   // of the keys 2 t, 2 t + 1 and of 2 t + 8, 2 t + 9
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t pick = gr & 1 ? 0x7632u : 0x5410u;
          pairs[r] = __byte_perm(tile[i].v[2 * r][gr / 2], tile[i].v[2 * r + 1][gr / 2], pick);
          scales[r] = __byte_perm(tile[i].v_scale[r][gr / 2], tile[i].v_scale[r][G / 2 + gr / 2], pick);
        }
        uint32_t b[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          b[nt][0] = mul_bf16x2(w[nt][0], scales[0]);
          b[nt][1] = mul_bf16x2(w[nt][1], scales[1]);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t a[4];
          a[0] = codes_of(pairs[0], 2 * half);
          a[1] = codes_of(pairs[0], 2 * half + 1);
          a[2] = codes_of(pairs[1], 2 * half);
          a[3] = codes_of(pairs[1], 2 * half + 1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816(o[nt][2 * gr + half], a, b[nt][0], b[nt][1]);
        }
      }
    }
  }

  // each warp leaves its partial in shared memory
  float* mine = merge + warp * (8 * NT * kRow);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float total = sum[nt][c];
      total += __shfl_xor_sync(0xffffffffu, total, 4);
      total += __shfl_xor_sync(0xffffffffu, total, 8);
      total += __shfl_xor_sync(0xffffffffu, total, 16);
      float* row = mine + (nt * 8 + 2 * t + c) * kRow;
      if (g == 0) {
        row[D] = most[nt][c];
        row[D + 1] = total;
      }
#pragma unroll
      for (int gr = 0; gr < G; ++gr)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          *reinterpret_cast<float2*>(row + 32 * gr + 4 * g + 2 * half) = make_float2(o[nt][2 * gr + half][c], o[nt][2 * gr + half][2 + c]);
    }
  }
  __syncthreads();
  // and the block merges them: a few threads a head
  constexpr int kThreadsOfHead = 32 * kWarps / (8 * NT), kColumns = D / kThreadsOfHead;
  const int head = threadIdx.x / kThreadsOfHead, part = threadIdx.x % kThreadsOfHead;
  if (head0 + head >= group) return;
  float m[kWarps], best = -INFINITY, total = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    m[w] = merge[(w * 8 * NT + head) * kRow + D];
    best = fmaxf(best, m[w]);
  }
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    // a warp that saw no key has sum 0; one whose scores are all NaN has no maximum either, and a sum that is NaN
    m[w] = best == -INFINITY ? 1.0f : exp2f(m[w] - best);
    total += merge[(w * 8 * NT + head) * kRow + D + 1] * m[w];
  }
  const size_t at = (static_cast<size_t>(entry) * p.num_heads + kv_head * group + head0 + head) * places + split;
  if (part == 0) {
    p.partial_ml[2 * at] = best == -INFINITY && total != total ? 0.0f : best;   // the combine kernel passes over -inf
    p.partial_ml[2 * at + 1] = total;
  }
#pragma unroll
  for (int c = 0; c < kColumns; c += 4) {
    const int column = part * kColumns + c;
    float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(merge + (w * 8 * NT + head) * kRow + column);
      value.x += m[w] * v.x;
      value.y += m[w] * v.y;
      value.z += m[w] * v.z;
      value.w += m[w] * v.w;
    }
    *reinterpret_cast<float4*>(p.partial_out + at * D + column) = value;
  }
}

template <int D, int NT>
int launch(const DecodeParams& p, cudaStream_t s) {
  constexpr int kSmem = kWarps * 8 * NT * (D + 4) * 4;
  static_assert(kSmem <= 48 * 1024, "shared memory that needs no opt-in");
  const int group = p.num_heads / p.num_kv_heads, head_tiles = (group + 8 * NT - 1) / (8 * NT);
  const dim3 grid(p.num_entries, p.num_kv_heads * head_tiles, p.num_splits + (p.keep_first > 0 ? 1 : 0));
  int status = vipera_launch(attention_q4_decode_kernel<D, NT>, grid, 32 * kWarps, kSmem, s, p);
  if (status != VIPERA_OK) return status;
  const bool ending = p.keep_first > 0 || p.sink || p.gate;
  return vipera_launch(ending ? attention_combine_kernel<D, true> : attention_combine_kernel<D>, dim3(p.num_entries, p.num_heads),
                       D, 0, s, p.partial_ml, p.partial_out, p.num_splits, p.out, p.num_heads, p.positions, p.window, p.chunk,
                       p.entry_starts, p.keep_first, p.sink, p.sink_values, p.gate, p.gate_stride, p.gate_per_head);
}

bool on_16_bytes(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

VIPERA_API int vipera_attention_q4_params_size() { return static_cast<int>(sizeof(DecodeParams)); }

// Attention of the entries that bring one token (all of them where entry_starts is null).  `scratch` holds the splits'
// partials, (2 + d) floats per (entry, head, place); p->partial_ml and p->partial_out are set here.
VIPERA_API int vipera_attention_q4_decode(const DecodeParams* given, float* scratch, size_t scratch_floats, void* stream) {
  DecodeParams p = *given;
  if (p.num_entries <= 0) return VIPERA_OK;
  if (p.num_heads <= 0 || p.num_kv_heads <= 0 || p.num_heads % p.num_kv_heads || p.keep_first < 0 || p.page_size <= 0 ||
      p.page_size % 16 || p.num_heads > 65535 || p.num_splits <= 0 || p.num_splits > 128 || p.chunk <= 0 ||
      p.chunk % (kWarps * kWarpKeys) || (p.head_dim != 64 && p.head_dim != 128))
    return VIPERA_BAD_SHAPE;
  if (p.window <= 0) p.keep_first = 0;
  if (p.sink_values) p.sink = 1;
  const size_t rows = static_cast<size_t>(p.num_entries) * p.num_heads * (p.num_splits + (p.keep_first > 0 ? 1 : 0));
  const size_t pairs = (2 * rows + 3) / 4 * 4;
  if (!scratch || scratch_floats < pairs + rows * p.head_dim || !on_16_bytes(scratch) || !on_16_bytes(p.q) || !on_16_bytes(p.k_codes) ||
      !on_16_bytes(p.v_codes) || !on_16_bytes(p.k_scales) || !on_16_bytes(p.v_scales))
    return VIPERA_BAD_ARGUMENT;
  p.partial_ml = scratch;
  p.partial_out = scratch + pairs;
  p.page_shift = -1;
  if ((p.page_size & (p.page_size - 1)) == 0)
    for (p.page_shift = 0; (1 << p.page_shift) < p.page_size;) ++p.page_shift;
  const bool wide = p.num_heads / p.num_kv_heads > 8;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p.head_dim == 128) return wide ? launch<128, 2>(p, s) : launch<128, 1>(p, s);
  return wide ? launch<64, 2>(p, s) : launch<64, 1>(p, s);
}
