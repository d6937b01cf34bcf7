// Attention of a step's tokens over pages of 4 bits, any number of tokens a request, split over the keys; part of attention_q4.cu.
//
// A block is (8 NT of the (token, query head) rows of one request and KV head, split of the keys); its four warps fold 16 keys at a
// time each.  Rows lie on the side of 8 of both products, as in the kernel of single tokens, each with a range of visible keys of its
// own.  What differs is exactness: codes become bfloat16 numbers exactly (128 + u less 136), and a 32-bit number (a query's channel, a
// weight times the value's scale) is the exact sum of three bfloat16 ones, each a product of its own, so that 32-bit steps are as exact
// as their sums; bfloat16 steps round a weight once.  The query's parts lie in shared memory.
//
// What bounds it: issuing, and for short steps the latency of one walk.  Rows times keys go by at 1.7e5 a microsecond with heads of
// 128 in bfloat16, so that the tensor cores' kernel (attention_q4_tc.cu) wins beyond a size (ops.attention_q4_takes_rows has the rule and
// both sides' times).  384 rows of 32 bits over 96 to 2,113 keys: 22 us with the joining launch, from a cold cache.
#pragma once

namespace {

struct RowsParams {
  const void* q;                  // [tokens, heads, d]
  const uint8_t *k_codes, *v_codes;
  const __nv_bfloat16 *k_scales, *v_scales;
  const int* entry_starts;
  const int* entry_pos0;
  const int* block_table;
  float* partial_ml;
  float* partial_out;
  int table_width, page_size, num_pages, num_entries, num_tokens, num_heads, num_kv_heads;
  float scale;
  int window, keep_first, chunk, num_splits;
};

__device__ __forceinline__ uint32_t exact_codes(uint32_t word, int j) {
  const uint32_t a = ((word >> (4 * j)) & 0x000f000fu) | 0x43004300u, b = 0x43084308u;
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Two numbers as the sum of PARTS pairs of bfloat16 ones.
template <int PARTS>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&to)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    to[i] = pack_bf16(x, y);
    if (i + 1 < PARTS) {
      x -= low_of(to[i]);
      y -= high_of(to[i]);
    }
  }
}

// T: float (three parts a number) or bfloat16 (one).
template <int D, typename T, int NT>
__global__ void __launch_bounds__(32 * kWarps) attention_q4_rows_kernel(RowsParams p) {
  constexpr int G = D / 32, PARTS = sizeof(T) == 4 ? 3 : 1, kRow = D + 4, kRows = 8 * NT;
  extern __shared__ __align__(16) uint8_t shared_rows[];
  uint4* parts = reinterpret_cast<uint4*>(shared_rows);                               // [NT][G][PARTS][lane]
  float* merge = reinterpret_cast<float*>(shared_rows + NT * G * PARTS * 512);        // [warp][row][kRow]
  pdl_wait();
  pdl_launch_dependents();
  const int group = p.num_heads / p.num_kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // which entry's tile of rows this is: a lane an entry
  int entry = -1, tile = 0, token0 = 0, count = 0;
  for (int base = 0, before = 0; base < p.num_entries; base += 32) {
    const int e = base + lane;
    const int start = e < p.num_entries ? p.entry_starts[e] : 0, n = e < p.num_entries ? p.entry_starts[e + 1] - start : 0;
    const int tiles = (max(n, 0) * group + kRows - 1) / kRows;
    int upto = tiles;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, offset);
      if (lane >= offset) upto += v;
    }
    const int mine = static_cast<int>(blockIdx.x) - before - (upto - tiles);
    const uint32_t found = __ballot_sync(0xffffffffu, mine >= 0 && mine < tiles);
    if (found) {
      const int source = __ffs(found) - 1;
      entry = base + source;
      tile = __shfl_sync(0xffffffffu, mine, source);
      token0 = __shfl_sync(0xffffffffu, start, source);
      count = __shfl_sync(0xffffffffu, n, source);
      break;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (entry < 0) return;
  const int kv_head = blockIdx.y, split = blockIdx.z;
  const int row0 = tile * kRows, rows = min(kRows, count * group - row0);
  const int pos0 = p.entry_pos0[entry];
  const int* table = p.block_table + static_cast<size_t>(entry) * p.table_width;
  // the rows' ranges lie between those of the first and of the last
  const int last_low = pos0 + row0 / group, last_high = pos0 + (row0 + rows - 1) / group;
  const int first_low = first_visible_key(last_low, p.window), first_high = first_visible_key(last_high, p.window);
  const bool kept_split = split == p.num_splits;
  const int places = p.num_splits + (p.keep_first > 0 ? 1 : 0);
  const int begin = kept_split ? 0 : max(split * p.chunk, first_low / 32 * 32);
  const int end = kept_split ? min(p.keep_first, first_high) : min((split + 1) * p.chunk, last_high + 1);
  if (begin >= end && !kept_split) return;    // no row's keys are here: the joining kernel does not look (it does for kept keys)

  for (int i = threadIdx.x; i < NT * G * 32; i += blockDim.x) {     // (row tile, group, lane): eight channels
    const int l = i & 31, gr = i / 32 % G, nt = i / 32 / G, r = row0 + nt * 8 + (l >> 2);
    float x[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) x[c] = 0.0f;
    if (nt * 8 + (l >> 2) < rows) {
      const int token = token0 + r / group, head = kv_head * group + r % group;
      const T* from = static_cast<const T*>(p.q) + (static_cast<size_t>(token) * p.num_heads + head) * D + 32 * gr + 8 * (l & 3);
#pragma unroll
      for (int c = 0; c < 8; ++c) x[c] = to_float<T>(from[c]);
    }
    uint32_t pair[4][PARTS];
#pragma unroll
    for (int c = 0; c < 4; ++c) split_pair<PARTS>(x[2 * c], x[2 * c + 1], pair[c]);
#pragma unroll
    for (int k = 0; k < PARTS; ++k) parts[((nt * G + gr) * PARTS + k) * 32 + l] = make_uint4(pair[0][k], pair[1][k], pair[2][k], pair[3][k]);
  }
  __syncthreads();

  // what this lane's rows (columns 2 t and 2 t + 1 of every tile) see here: keys from first to last, of the kept ones' split those in
  // front of the row's window
  int first[NT][2], last[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = nt * 8 + 2 * t + c, position = pos0 + (row0 + r) / group;
      first[nt][c] = first_visible_key(position, p.window);
      last[nt][c] = r < rows ? position : -1;
      if (kept_split) {
        last[nt][c] = min(last[nt][c], min(p.keep_first, first[nt][c]) - 1);
        first[nt][c] = 0;
      }
    }

  float o[NT][2 * G][4], most[NT][2], base[NT][2], sum[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    most[nt][0] = most[nt][1] = -INFINITY;
    base[nt][0] = base[nt][1] = sum[nt][0] = sum[nt][1] = 0.0f;
#pragma unroll
    for (int m = 0; m < 2 * G; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nt][m][i] = 0.0f;
  }
  const float scale_log2 = p.scale * kLog2e;

  for (int key0 = begin + warp * 16; key0 < end; key0 += kWarps * 16) {
    const int index = key0 / p.page_size;
    const int page = index < p.table_width ? table[index] : -1;
    if (page < 0 || page >= p.num_pages) continue;
    const size_t row = (static_cast<size_t>(page) * p.num_kv_heads + kv_head) * p.page_size + (key0 - index * p.page_size);
    // keys g and g + 8 (accumulator rows), and the values' keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
    uint32_t k[2][G], k_scale[2][G / 2], v[4][G / 2], v_scale[2][G / 2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      load_words<G>(k[r], p.k_codes + (row + g + 8 * r) * (D / 2) + t * 4 * G);
      load_words<G / 2>(k_scale[r], p.k_scales + (row + g + 8 * r) * G);
      load_words<G / 2>(v_scale[r], p.v_scales + (row + g + 8 * r) * G);
#pragma unroll
      for (int i = 0; i < 2; ++i) load_words<G / 2>(v[2 * r + i], p.v_codes + (row + 2 * t + 8 * r + i) * (D / 2) + g * 2 * G);
    }
    float s[NT][4];        // keys g (0, 1) and g + 8 (2, 3), rows 2 t and 2 t + 1; in units of log2
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[nt][c] = 0.0f;
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      uint32_t a[2][4];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        a[half][0] = exact_codes(k[0][gr], 2 * half);
        a[half][1] = exact_codes(k[1][gr], 2 * half);
        a[half][2] = exact_codes(k[0][gr], 2 * half + 1);
        a[half][3] = exact_codes(k[1][gr], 2 * half + 1);
      }
      const float scale0 = gr & 1 ? high_of(k_scale[0][gr / 2]) : low_of(k_scale[0][gr / 2]);
      const float scale1 = gr & 1 ? high_of(k_scale[1][gr / 2]) : low_of(k_scale[1][gr / 2]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int part = PARTS - 1; part >= 0; --part) {   // the smallest first
          const uint4 q = parts[((nt * G + gr) * PARTS + part) * 32 + lane];
          mma_bf16(acc, a[0], q.x, q.y);
          mma_bf16(acc, a[1], q.z, q.w);
        }
        s[nt][0] = fmaf(scale0, acc[0], s[nt][0]);
        s[nt][1] = fmaf(scale0, acc[1], s[nt][1]);
        s[nt][2] = fmaf(scale1, acc[2], s[nt][2]);
        s[nt][3] = fmaf(scale1, acc[3], s[nt][3]);
      }
    }
    const bool whole = key0 >= first_high && key0 + 15 <= last_low && rows == kRows && !kept_split;
    bool grown = false;
    float high[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[nt][c] *= scale_log2;
        if (!whole) {
          const int key = key0 + g + 8 * (c >> 1);
          const bool seen = key >= first[nt][c & 1] && key <= last[nt][c & 1];
          if (!seen) s[nt][c] = -INFINITY;
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        high[nt][c] = fmaxf(s[nt][c], s[nt][2 + c]);
        grown = grown || high[nt][c] > most[nt][c];
      }
    }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float m = fmaxf(high[nt][c], most[nt][c]);
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          base[nt][c] = m == -INFINITY ? 0.0f : m;
          const float shrink = exp2_near(most[nt][c] - base[nt][c]);
          most[nt][c] = m;
          sum[nt][c] *= shrink;
#pragma unroll
          for (int n = 0; n < 2 * G; ++n) {
            o[nt][n][c] *= shrink;
            o[nt][n][2 + c] *= shrink;
          }
        }
    }
    float weight[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        weight[nt][c] = exp2_near(s[nt][c] - base[nt][c & 1]);
        sum[nt][c & 1] += weight[nt][c];
      }
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      const uint32_t pick = gr & 1 ? 0x7632u : 0x5410u;
      const float scale0 = gr & 1 ? high_of(v_scale[0][gr / 2]) : low_of(v_scale[0][gr / 2]);
      const float scale1 = gr & 1 ? high_of(v_scale[1][gr / 2]) : low_of(v_scale[1][gr / 2]);
      uint32_t a[2][4];
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t pairs = __byte_perm(v[2 * r][gr / 2], v[2 * r + 1][gr / 2], pick);
          a[half][2 * r] = exact_codes(pairs, 2 * half);
          a[half][2 * r + 1] = exact_codes(pairs, 2 * half + 1);
        }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint32_t b[2][PARTS];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float scale = r ? scale1 : scale0;
          // a hidden key's weight is 0, and its scale must not make that NaN
          float x = weight[nt][2 * r] * scale, y = weight[nt][2 * r + 1] * scale;
          if (!whole) {
            if (s[nt][2 * r] == -INFINITY) x = 0.0f;
            if (s[nt][2 * r + 1] == -INFINITY) y = 0.0f;
          }
          split_pair<PARTS>(x, y, b[r]);
        }
#pragma unroll
        for (int part = PARTS - 1; part >= 0; --part) {
          const uint32_t b0 = turn_8x8(b[0][part]), b1 = turn_8x8(b[1][part]);
          mma_bf16(o[nt][2 * gr], a[0], b0, b1);
          mma_bf16(o[nt][2 * gr + 1], a[1], b0, b1);
        }
      }
    }
  }

  float* mine = merge + warp * (kRows * kRow);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float total = sum[nt][c];
      total += __shfl_xor_sync(0xffffffffu, total, 4);
      total += __shfl_xor_sync(0xffffffffu, total, 8);
      total += __shfl_xor_sync(0xffffffffu, total, 16);
      float* to = mine + (nt * 8 + 2 * t + c) * kRow;
      if (g == 0) {
        to[D] = most[nt][c];
        to[D + 1] = total;
      }
#pragma unroll
      for (int gr = 0; gr < G; ++gr)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          *reinterpret_cast<float2*>(to + 32 * gr + 4 * g + 2 * half) = make_float2(o[nt][2 * gr + half][c], o[nt][2 * gr + half][2 + c]);
    }
  __syncthreads();
  constexpr int kThreadsOfRow = 32 * kWarps / kRows;
  const int r = threadIdx.x / kThreadsOfRow;
  if (r < rows) {
    const int token = token0 + (row0 + r) / group, head = kv_head * group + (row0 + r) % group;
    const size_t at = (static_cast<size_t>(token) * p.num_heads + head) * places + split;
    merge_warps<D, kRows>(merge, r, threadIdx.x % kThreadsOfRow, p.partial_ml + 2 * at, p.partial_out + at * D);
  }
}

template <int D, typename T, int NT>
int launch_rows(const RowsParams& p, cudaStream_t s) {
  constexpr int G = D / 32, PARTS = sizeof(T) == 4 ? 3 : 1;
  constexpr int kSmem = NT * G * PARTS * 512 + kWarps * 8 * NT * (D + 4) * 4;
  static_assert(kSmem <= 48 * 1024, "shared memory that needs no opt-in");
  const int group = p.num_heads / p.num_kv_heads;
  // at most this many tiles of rows: blocks beyond the last one leave
  const long long tiles = (static_cast<long long>(p.num_tokens) * group + 8 * NT - 1) / (8 * NT) + p.num_entries;
  if (tiles > 0x7fffffffLL || p.num_kv_heads > 65535) return VIPERA_BAD_SHAPE;
  const dim3 grid(static_cast<unsigned>(tiles), p.num_kv_heads, p.num_splits + (p.keep_first > 0 ? 1 : 0));
  return vipera_launch(attention_q4_rows_kernel<D, T, NT>, grid, 32 * kWarps, kSmem, s, p);
}

}  // namespace
