// Attention of single tokens over pages of 4 bits (formats: q4.cuh), split over the keys, on mma.sync m16n8k16.
//
// A block is (entry, KV head and up to 8 NT of its query heads, share of the visible keys); its four warps fold 32 keys at a time each
// with a running (max, sum, output) and merge at the end.  Where (entry, KV head) pairs are few, a cluster shares the keys of one and joins
// its parts through distributed shared memory: one launch, and nothing passes through memory.  Where they are many, the keys
// of all pairs are dealt to the blocks in even runs, and a second kernel joins the pairs that several runs share.
//
// Both products put the packed operand on the side of 16 (keys for the scores, channels for the values) and the query
// heads on the side of 8: a group of 8 heads or fewer costs half of the products that the other way round would
// waste on empty rows.  Offsets and scales of the codes stay outside of the products, and what is left of unpacking is what
// bounds the kernel beside the memory, so it is kept short:
//   scores   in half precision a nibble u at the bottom of 16 bits is the number u 2^-24, one at bits 4 to 7 is 16 u 2^-24 (the
//            smallest numbers are equally spaced), so a mask makes two codes an operand and one shift serves four.  The query's
//            channels, whose largest is brought to 2^14 .. 2^15, keep all their bits in half precision down to 2^-25 of the
//            largest, those that meet 16 u as a 16th.  The 32 channels of a group are one accumulator's two products, which
//            begins at -8 times the sum of the query's channels and which the key's scale multiplies in 32 bits:
//            s[key, head] = sum_g scale[key, g] (c[key, g, :] . q[head, g, :]).  The products' sums are as exact as if the codes
//            were 2^10: off by 2^-22 of that.
//   values   codes become bfloat16 by a shift, a mask and an OR (0x4300 | u is 128 + u, 136 above the code); the weights take the
//            scales in 32 bits, w[key, head, g] = p[key, head] scale[key, g], and are rounded to bfloat16 once; a product with
//            ones sums a group's, and 136 times that sum goes off at the end.
// A score's accumulators have the keys on their rows, the second product wants them on its inner axis: movmatrix turns the
// weights' 8 x 8 blocks in registers, so nothing passes through shared memory until the end.
//
// What bounds it.  48 requests of 8,192 keys, 40 heads of 128 on 8: 455 MB, read once, in 116 to 121 us with the joining kernel, 3.8 TB/s
// (58 % of the measured copy).  It is bound by issuing: 16 keys of a head are 290 instructions of a warp (156 of them integer and logic, 20
// products), issue slots are 59 % busy and the integer pipe 56 %, and fetching, unpacking, scaling and weighing each shorten the time by
// less than their share when taken out.  More blocks an SM (four of 128 registers), more or fewer stages and rows read
// straight into registers change nothing; 8-bit operands (e4m3, where a nibble is a number as it stands) cost conversions on this
// device, 443 instructions; shifts as high halves of products are 9 % slower; codes less their offset before the products 411.
#include "attention_q4_join.cuh"
#include "attention_mma.cuh"
#include "q4.cuh"

#include <cuda_fp16.h>

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
  long long gate_stride;
  int gate_per_head;
  int table_width, page_size, page_shift, num_pages, num_entries, num_heads, num_kv_heads, head_dim;
  float scale;
  int window, keep_first, sink, shares;
  // 1: positions, tables and earlier steps' rows are complete before the kernel ahead of this one begins.  2: that kernel, of the same step's
  // portions, lets this one begin once all that went before itself is complete, which `beside` says (attention_q4_join.cuh), and shares nothing
  // with it: this one waits for it at its end (portions of 512, 200 and 37 tokens beside 16 single ones behind 2,048: 57 us for 74).
  // What is read in front of a wait, and what another kernel has written behind it, is read from L2.
  int settled;
  int* beside;
  uint32_t magic;                 // set by the launcher
};

constexpr int kWarps = 4;
constexpr int kWarpKeys = 32;   // keys a warp folds at a time: two tiles of 16
constexpr int kStages = 3;      // such pairs of tiles on their way to shared memory for each warp

// The codes at bits 4 j and 16 + 4 j of a word as two bfloat16, 128 + u each.  `magic` is 0x43004300 from a parameter: a constant
// would be an instruction's immediate beside the mask's, and two do not fit into one.
__device__ __forceinline__ uint32_t codes_of(uint32_t word, int j, uint32_t magic) { return ((word >> (4 * j)) & 0x000f000fu) | magic; }
constexpr float kOffset = 136.0f;   // what such a number is above its code
constexpr uint32_t kOnes = 0x3f803f80u;

__device__ __forceinline__ uint32_t turn_8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float exp2_near(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float low_of(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float high_of(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }
// d = a . b + c, and d += a . b, of half-precision operands
__device__ __forceinline__ void mma_half_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float4& c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y), "f"(c.z), "f"(c.w));
}
__device__ __forceinline__ void mma_half(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// a float, and four of them, at `local` (a shared-memory address of this block) in the block of rank `rank`
__device__ __forceinline__ float cluster_load(uint32_t local, uint32_t rank) {
  uint32_t remote;
  float value;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(value) : "r"(remote) : "memory");
  return value;
}
__device__ __forceinline__ float4 cluster_load_4(uint32_t local, uint32_t rank) {
  uint32_t remote;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
  return v;
}
__device__ __forceinline__ void cp_async_all(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

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

// The warps' partials of one row ([warp][ROWS][D + 4] floats: outputs, maximum, sum) become the block's: 32 kWarps / ROWS threads a row,
// `part` one of them.
template <int D, int ROWS>
__device__ __forceinline__ void merge_warps(const float* merge, int row, int part, float* ml, float* out) {
  constexpr int kRow = D + 4, kColumns = D * ROWS / (32 * kWarps);
  float m[kWarps], best = -INFINITY, total = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    m[w] = merge[(w * ROWS + row) * kRow + D];
    best = fmaxf(best, m[w]);
  }
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    // a warp that saw no key has sum 0; one whose scores are all NaN has no maximum either, and a sum that is NaN
    m[w] = best == -INFINITY ? 1.0f : exp2f(m[w] - best);
    total += merge[(w * ROWS + row) * kRow + D + 1] * m[w];
  }
  if (part == 0) {
    ml[0] = best == -INFINITY && total != total ? 0.0f : best;   // the joining kernel passes over -inf
    ml[1] = total;
  }
#pragma unroll
  for (int c = 0; c < kColumns; c += 4) {
    const int column = part * kColumns + c;
    float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(merge + (w * ROWS + row) * kRow + column);
      value.x += m[w] * v.x;
      value.y += m[w] * v.y;
      value.z += m[w] * v.z;
      value.w += m[w] * v.w;
    }
    *reinterpret_cast<float4*>(out + column) = value;
  }
}

// Two tiles of 16 keys in a warp's part of shared memory.  Row r of a tile's score accumulators is key 4 (r & 1) + (r & 7) / 2 + 8 (r / 8):
// the keys whose weights a lane's operand of the second product holds, slots 2 t, 2 t + 1, 2 t + 8 and 2 t + 9, are then keys 4 i + t, i
// = 0 .. 3, whose rows four lanes read without a conflict; the keys' own rows lie in the order of the accumulators.
template <int D>
struct Stage {
  static constexpr int G = D / 32, kRowBytes = D / 2;
  uint8_t k[2][16 * kRowBytes];
  uint8_t v[2][16 * kRowBytes];
  uint8_t k_scale[2][16 * G * 2];
  uint8_t v_scale[2][16 * G * 2];
};

// The visible keys of a query in tiles of 16: those of the kept first keys that the window has left behind, then those of the window.
struct Visible {
  int position, first, kept, kept_tiles, first_tile, tiles;
  __device__ __forceinline__ Visible(const DecodeParams& p, int at) {
    position = at;
    first = first_visible_key(position, p.window);
    kept = p.window > 0 ? min(p.keep_first, first) : 0;
    kept_tiles = (kept + 15) >> 4;
    first_tile = first >> 4;
    tiles = kept_tiles + max((position >> 4) - first_tile + 1, 0);
  }
  __device__ __forceinline__ int key_of(int tile) const { return 16 * (tile < kept_tiles ? tile : tile - kept_tiles + first_tile); }
  __device__ __forceinline__ bool hides(int tile, int key) const {
    return tile < kept_tiles ? key >= kept : key < first || key > position;
  }
};

// What a block has in shared memory: the queries, the warps' stages, and, at the end of a walk in the place of the stages, the warps' partials
// [warp][8 NT heads][D + 4] and behind them what they join to, `joined` [8 NT heads][D + 4]: outputs, maximum, sum.
template <int D, int NT>
struct Shared {
  static constexpr int kRow = D + 4, kQueryBytes = NT * (D / 32) * (512 + 64);
  static constexpr int kStageBytes = kWarps * kStages * static_cast<int>(sizeof(Stage<D>)), kBytes = kQueryBytes + kStageBytes;
  static_assert((kWarps + 1) * 8 * NT * kRow * 4 <= kStageBytes, "the partials fit in the stages");
  uint8_t* at;
  __device__ __forceinline__ uint4* queries() const { return reinterpret_cast<uint4*>(at); }                                // [NT][G][lane]
  __device__ __forceinline__ float4* offsets() const { return reinterpret_cast<float4*>(at + NT * (D / 32) * 512); }        // [NT][G][t]
  __device__ __forceinline__ Stage<D>* stages() const { return reinterpret_cast<Stage<D>*>(at + kQueryBytes); }
  __device__ __forceinline__ float* merge() const { return reinterpret_cast<float*>(at + kQueryBytes); }
  __device__ __forceinline__ float* joined() const { return merge() + kWarps * 8 * NT * kRow; }
};

// The block's walk over tiles tile_begin (a multiple of 8) to tiles_end - 1 of what the query heads head0 .. of a KV head see; it leaves the
// heads' outputs, maxima and sums in `joined`, to be read behind a barrier.
template <int D, int NT>
__device__ __forceinline__ void walk(const DecodeParams& p, const Shared<D, NT> shared, const Visible seen, int entry, int token, int kv_head,
                                     int head0, int tile_begin, int tiles_end, bool waited = true) {
  constexpr int G = D / 32, kRowBytes = D / 2, kChunks = kRowBytes / 16;
  constexpr int kRow = D + 4;
  uint4* queries = shared.queries();
  float4* offsets = shared.offsets();
  const int group = p.num_heads / p.num_kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int* table = p.block_table + static_cast<size_t>(entry) * p.table_width;

  // --- the way of the rows into shared memory: 16 bytes a lane, kStages - 1 pairs of tiles ahead ---
  Stage<D>* stages = shared.stages() + warp * kStages;
  const int warp_tile = tile_begin + 2 * warp;     // step j has tiles warp_tile + 8 j and the next
  const int steps = warp_tile < tiles_end ? (tiles_end - warp_tile + 7) >> 3 : 0;
  // the page of the tile that is this lane's among 32 of the warp's; a tile that is not the block's, and one whose page is not held, has
  // none and is filled with zeros
  const auto page_of = [&](int index) {
    const int tile = warp_tile + (index >> 1) * 8 + (index & 1);
    if (tile >= tiles_end) return -1;
    const int key = seen.key_of(tile), place = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
    const int page = place < p.table_width ? __ldcg(table + place) : -1;
    return page < p.num_pages ? page : -1;
  };
  int pages_now = page_of(lane), pages_next = steps > 16 ? page_of(32 + lane) : -1;
  const uint32_t page_rows = static_cast<uint32_t>(p.num_kv_heads) * p.page_size;   // rows of a page
  const uint8_t* k_head = p.k_codes + static_cast<size_t>(kv_head) * p.page_size * kRowBytes + lane * 16;
  const uint8_t* v_head = p.v_codes + static_cast<size_t>(kv_head) * p.page_size * kRowBytes + lane * 16;
  // a lane's piece of the scales: tile, keys' or values', place
  constexpr int kScaleChunks = 16 * G * 2 / 16;
  const int scale_tile = lane / (2 * kScaleChunks), scale_values = lane / kScaleChunks & 1, scale_chunk = lane % kScaleChunks;
  const uint8_t* scale_head = reinterpret_cast<const uint8_t*>(scale_values ? p.v_scales : p.k_scales) +
                              static_cast<size_t>(kv_head) * p.page_size * G * 2 + scale_chunk * 16;
  const uint32_t stages_at = smem_addr(stages);
  uint32_t k_to, v_to, scale_to;   // where a lane's piece goes within a stage (pieces of 8 keys, or of 16 where a row has two)
  {
    const int key = lane / kChunks, chunk = lane % kChunks;   // key of the first 8 (16)
    const int row = 2 * (key & 3) + ((key >> 2) & 1) + 8 * (key >> 3);
    k_to = stages_at + offsetof(Stage<D>, k) + row * kRowBytes + chunk * 16;
    v_to = stages_at + offsetof(Stage<D>, v) + key * kRowBytes + (kChunks == 4 ? chunk ^ (key & 2) : chunk) * 16;
    scale_to = stages_at + (scale_values ? offsetof(Stage<D>, v_scale) : offsetof(Stage<D>, k_scale)) +
               scale_tile * (16 * G * 2) + scale_chunk * 16;
  }
  const bool one_tile_a_page = p.page_size == 16;
  constexpr uint32_t kStageBytes = sizeof(Stage<D>);
  const auto fetch = [&](int j) {
    if (j < steps) {
      const uint32_t stage = (j % kStages) * kStageBytes;
      const int pages = (j & 16) ? pages_next : pages_now;
      const int page[2] = {__shfl_sync(0xffffffffu, pages, (2 * j) & 31), __shfl_sync(0xffffffffu, pages, (2 * j + 1) & 31)};
      uint32_t place[2] = {0, 0};
      if (!one_tile_a_page) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = seen.key_of(warp_tile + 8 * j + i);
          place[i] = p.page_shift >= 0 ? key & (p.page_size - 1) : key % p.page_size;
        }
      }
      constexpr int kPieces = 16 * kChunks / 32;    // of 32 lanes a tile
      const bool all = (page[0] | page[1]) >= 0;    // every tile but the first and the last of a walk
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint64_t from = static_cast<uint64_t>(static_cast<uint32_t>(all ? page[i] : max(page[i], 0))) * (page_rows * kRowBytes) +
                              place[i] * kRowBytes;
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
          if (all) {
            cp_async_all(k_to + stage + i * 16 * kRowBytes + c * 512, k_head + from + c * 512);
            cp_async_all(v_to + stage + i * 16 * kRowBytes + c * 512, v_head + from + c * 512);
          } else {
            cp_async_16(k_to + stage + i * 16 * kRowBytes + c * 512, k_head + from + c * 512, page[i] >= 0);
            cp_async_16(v_to + stage + i * 16 * kRowBytes + c * 512, v_head + from + c * 512, page[i] >= 0);
          }
        }
      }
      if (lane < 4 * kScaleChunks) {
        const int mine = scale_tile ? page[1] : page[0];
        cp_async_16(scale_to + stage, scale_head + static_cast<uint64_t>(static_cast<uint32_t>(max(mine, 0))) * (page_rows * G * 2) +
                                          (scale_tile ? place[1] : place[0]) * (G * 2), mine >= 0);
      }
    }
    cp_async_commit();
  };

  // Rows of earlier steps may come before the kernel ahead has ended; the query's own row, and the queries, only then.  The kernel behind
  // may start from there on and not before: the decode step of one request is 1.32 ms so and 1.46 where it may start at once (its
  // blocks then take the places that this kernel's clusters wait for).
  if (!waited && tiles_end == seen.tiles) {
    pdl_wait();
    pdl_launch_dependents();
  }
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) fetch(j);
  if (!waited && tiles_end != seen.tiles) {
    pdl_wait();
    pdl_launch_dependents();
  }

  // --- the queries in half precision: lane (g, t) has channels 32 group + 8 t .. + 7 of head 8 nt + g ---
  // in shared memory, a piece of 16 bytes a lane: neighbouring channels, the second and fourth pair a 16th; and, for heads 2 t and 2 t + 1,
  // -8 times the sum of a group's channels, as what accumulators begin with
  float q_factor[NT][2];      // what a product has to be multiplied by, of heads 2 t and 2 t + 1; in units of log2
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int h = head0 + nt * 8 + g;
    uint32_t q[G][4];
    float largest = 0.0f;
    bool fine = true;
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      q[gr][0] = q[gr][1] = q[gr][2] = q[gr][3] = 0;
      if (h < group) {
        const uint4 v = __ldcg(reinterpret_cast<const uint4*>(
            p.q + (static_cast<size_t>(token) * p.num_heads + kv_head * group + h) * D + 32 * gr + 8 * t));
        q[gr][0] = v.x, q[gr][1] = v.y, q[gr][2] = v.z, q[gr][3] = v.w;
      }
    }
#pragma unroll
    for (int gr = 0; gr < G; ++gr)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        largest = fmaxf(largest, fmaxf(fabsf(low_of(q[gr][w])), fabsf(high_of(q[gr][w]))));
        fine = fine && fabsf(low_of(q[gr][w])) < INFINITY && fabsf(high_of(q[gr][w])) < INFINITY;
      }
#pragma unroll
    for (int offset = 1; offset <= 2; offset <<= 1) {
      largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, offset));
      fine = __shfl_xor_sync(0xffffffffu, static_cast<int>(fine), offset) && fine;
    }
    // the largest to 2^14 .. 2^15 (a number that is not finite: everything NaN)
    const int exponent = static_cast<int>(__float_as_uint(largest) >> 23) - 127;
    const int up = min(max(14 - exponent, -113), 110);
    const float lift = fine ? __uint_as_float(static_cast<uint32_t>(127 + up) << 23) : __int_as_float(0x7fffffff);
    const float factor = ldexpf(p.scale * kLog2e, 24 - up);   // a code is u 2^-24 (both powers at once: one alone may leave the type)
    q_factor[nt][0] = __shfl_sync(0xffffffffu, factor, 8 * t);
    q_factor[nt][1] = __shfl_sync(0xffffffffu, factor, 8 * t + 4);
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      if (gr % kWarps != warp) continue;      // every warp a group
      float total = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float lo = low_of(q[gr][w]) * lift, hi = high_of(q[gr][w]) * lift;
        total += lo + hi;
        q[gr][w] = w & 1 ? pack_half(lo * 0.0625f, hi * 0.0625f) : pack_half(lo, hi);
      }
      total += __shfl_xor_sync(0xffffffffu, total, 1);
      total += __shfl_xor_sync(0xffffffffu, total, 2);
      const float x = -8.0f * 0x1p-24f * __shfl_sync(0xffffffffu, total, 8 * t), y = -8.0f * 0x1p-24f * __shfl_sync(0xffffffffu, total, 8 * t + 4);
      queries[(nt * G + gr) * 32 + lane] = make_uint4(q[gr][0], q[gr][1], q[gr][2], q[gr][3]);
      if (g == 0) offsets[(nt * G + gr) * 4 + t] = make_float4(x, y, x, y);
    }
  }
  __syncthreads();
  const uint32_t magic = p.magic;
  float o[NT][2 * G][4];      // channels 32 gr + 4 g + 2 h and the next (rows g, g + 8), heads 2 t and 2 t + 1, of codes + 136
  float w_sum[NT][G][4];      // sums of a group's scaled weights, alike in every row (a group's alone: ones in some rows and zeros in others would
                              // carry a weight that is NaN into the other groups' sums)
  float most[NT][2], base[NT][2], sum[NT][2];   // base: most, or 0 where nothing has been seen
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    most[nt][0] = most[nt][1] = -INFINITY;
    base[nt][0] = base[nt][1] = 0.0f;
    sum[nt][0] = sum[nt][1] = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int m = 0; m < 2 * G; ++m) o[nt][m][i] = 0.0f;
#pragma unroll
      for (int gr = 0; gr < G; ++gr) w_sum[nt][gr][i] = 0.0f;
    }
  }
  const uint32_t ones[4] = {kOnes, kOnes, kOnes, kOnes};
  const int row_key = 4 * (g & 1) + (g >> 1);                       // the key of accumulator row g
  const uint32_t v_from = t * kRowBytes + (kChunks == 4 ? ((g >> 1) ^ (t & 2)) * 16 + (g & 1) * 8 : g * (2 * G));

  for (int j = 0; j < steps; ++j) {
    if (j > 0 && (j & 15) == 0) {   // the next 32 tiles' pages; those behind are on their way
      if (j & 16) pages_now = page_of(2 * j + 32 + lane);
      else pages_next = page_of(2 * j + 32 + lane);
    }
    fetch(j + kStages - 1);
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const Stage<D>& from = stages[j % kStages];
    const int tile0 = warp_tile + 8 * j;
    float s[2][NT][4];        // rows g (0, 1) and g + 8 (2, 3), heads 2 t and 2 t + 1; in units of log2
    uint32_t k[2][2][G], k_scale[2][2][G / 2];       // [tile][row g, g + 8]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        load_words<G>(k[i][r], from.k[i] + (g + 8 * r) * kRowBytes + t * 4 * G);
        load_words<G / 2>(k_scale[i][r], from.k_scale[i] + (row_key + 8 * r) * (G * 2));
      }
#pragma unroll
    for (int gr = 0; gr < G; ++gr)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint4 q = queries[(nt * G + gr) * 32 + lane];
        const float4 offset = offsets[(nt * G + gr) * 4 + t];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t k0 = k[i][0][gr], k1 = k[i][1][gr], l0 = k0 >> 8, l1 = k1 >> 8;
          const uint32_t a[4] = {k0 & 0x000f000fu, k1 & 0x000f000fu, k0 & 0x00f000f0u, k1 & 0x00f000f0u};
          const uint32_t b[4] = {l0 & 0x000f000fu, l1 & 0x000f000fu, l0 & 0x00f000f0u, l1 & 0x00f000f0u};
          const float scale0 = gr & 1 ? high_of(k_scale[i][0][gr / 2]) : low_of(k_scale[i][0][gr / 2]);
          const float scale1 = gr & 1 ? high_of(k_scale[i][1][gr / 2]) : low_of(k_scale[i][1][gr / 2]);
          float acc[4];
          mma_half_from(acc, a, q.x, q.y, offset);
          mma_half(acc, b, q.z, q.w);
          s[i][nt][0] = gr ? fmaf(scale0, acc[0], s[i][nt][0]) : scale0 * acc[0];
          s[i][nt][1] = gr ? fmaf(scale0, acc[1], s[i][nt][1]) : scale0 * acc[1];
          s[i][nt][2] = gr ? fmaf(scale1, acc[2], s[i][nt][2]) : scale1 * acc[2];
          s[i][nt][3] = gr ? fmaf(scale1, acc[3], s[i][nt][3]) : scale1 * acc[3];
        }
      }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[i][nt][c] *= q_factor[nt][c & 1];
    // every step but those with a border: all 32 keys are seen
    const int key0 = seen.key_of(tile0);
    const bool whole = tile0 >= seen.kept_tiles && key0 >= seen.first && key0 + kWarpKeys - 1 <= seen.position && tile0 + 1 < tiles_end;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (tile0 + i >= tiles_end || seen.hides(tile0 + i, seen.key_of(tile0 + i) + 8 * r + row_key)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[i][nt][2 * r] = s[i][nt][2 * r + 1] = -INFINITY;
          }
        }
    }
    // Only a step that raises some head's maximum needs a word among the eight lanes that hold a head's keys.  The maximum follows at once
    // (a threshold of 2^8 would save one such step in three): the weight of the key that a head looks at most is then 1, and is
    // not rounded, which halves the error where few keys count.
    float high[NT][2];
    bool grown = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        high[nt][c] = fmaxf(fmaxf(s[0][nt][c], s[0][nt][2 + c]), fmaxf(s[1][nt][c], s[1][nt][2 + c]));
        grown = grown || high[nt][c] > most[nt][c];
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
#pragma unroll
          for (int gr = 0; gr < G; ++gr) {
            w_sum[nt][gr][c] *= shrink;
            w_sum[nt][gr][2 + c] *= shrink;
          }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t v[4][G / 2], scale[2][G / 2];     // of keys 4 n + t: a unit of 16 bits a group; the scales of rows g and g + 8
#pragma unroll
      for (int n = 0; n < 4; ++n) load_words<G / 2>(v[n], from.v[i] + v_from + 4 * n * kRowBytes);
#pragma unroll
      for (int r = 0; r < 2; ++r) load_words<G / 2>(scale[r], from.v_scale[i] + (row_key + 8 * r) * (G * 2));
      if (!whole) {   // a hidden key's weight is 0, and its scale must not make that NaN
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (tile0 + i >= tiles_end || seen.hides(tile0 + i, seen.key_of(tile0 + i) + 8 * r + row_key)) {
#pragma unroll
            for (int w = 0; w < G / 2; ++w) scale[r][w] = 0;
          }
        }
      }
      float weight[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          weight[nt][c] = exp2_near(s[i][nt][c] - base[nt][c & 1]);
          sum[nt][c & 1] += weight[nt][c];
        }
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
        const uint32_t pick = gr & 1 ? 0x7632u : 0x5410u;
        uint32_t pairs[2], b[NT][2];      // b: scaled weights of head g, of keys t, 4 + t and of 8 + t, 12 + t
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          pairs[r] = __byte_perm(v[2 * r][gr / 2], v[2 * r + 1][gr / 2], pick);
          const float x = gr & 1 ? high_of(scale[r][gr / 2]) : low_of(scale[r][gr / 2]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) b[nt][r] = turn_8x8(pack_bf16(weight[nt][2 * r] * x, weight[nt][2 * r + 1] * x));
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t a[4];
          a[0] = codes_of(pairs[0], 2 * half, magic);
          a[1] = codes_of(pairs[0], 2 * half + 1, magic);
          a[2] = codes_of(pairs[1], 2 * half, magic);
          a[3] = codes_of(pairs[1], 2 * half + 1, magic);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_bf16(o[nt][2 * gr + half], a, b[nt][0], b[nt][1]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_bf16(w_sum[nt][gr], ones, b[nt][0], b[nt][1]);
      }
    }
    __syncwarp();   // the stage is free
  }
  cp_async_wait<0>();
  __syncthreads();  // the stages become the warps' partials
  float* merge = shared.merge();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int m = 0; m < 2 * G; ++m)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[nt][m][c] = fmaf(-kOffset, w_sum[nt][m / 2][c & 1], o[nt][m][c]);

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
  // the block merges them, a few threads a head
  float* joined = shared.joined();
  constexpr int kThreadsOfHead = 32 * kWarps / (8 * NT);
  const int head = threadIdx.x / kThreadsOfHead;
  merge_warps<D, 8 * NT>(merge, head, threadIdx.x % kThreadsOfHead, joined + head * kRow + D, joined + head * kRow);
}

// Four channels of a head's output: the ending's sink and gate, and the store.
template <int D>
__device__ __forceinline__ void finish(const DecodeParams& p, int token, int head, int column, float best, float total, const float4& value) {
  if (p.sink) total += exp2f((p.sink_values ? p.sink_values[head] * kLog2e : 0.0f) - best);
  float out[4] = {value.x / total, value.y / total, value.z / total, value.w / total};
  if (p.gate) {
    const float* gate = p.gate + static_cast<size_t>(token) * p.gate_stride + (p.gate_per_head ? head : head * D + column);
#pragma unroll
    for (int c = 0; c < 4; ++c) out[c] *= 1.0f / (1.0f + expf(-__ldcg(gate + (p.gate_per_head ? 0 : c))));
  }
  store_four_as<__nv_bfloat16>(p.out + (static_cast<size_t>(token) * p.num_heads + head) * D + column, out[0], out[1], out[2], out[3]);
}

// One more part joins a row's four channels: its weights were taken against another maximum.
struct Join {
  float best = -INFINITY, total = 0.0f;
  float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  __device__ __forceinline__ void add(float m, float l, const float4& v) {
    const float w = m == -INFINITY ? 0.0f : exp2f(m - best);    // -inf: a part without visible keys
    total += l * w;
    value.x += v.x * w;
    value.y += v.y * w;
    value.z += v.z * w;
    value.w += v.w * w;
  }
};

// The start and the end of a block beside the step's portions (DecodeParams::settled == 2).
__device__ __forceinline__ void begin_beside(const DecodeParams& p) {
  __shared__ int word;
  if (threadIdx.x == 0) word = acquire_word(p.beside);
  __syncthreads();
  if (word != 1) pdl_wait();
}
__device__ __forceinline__ void end_beside(const DecodeParams& p, bool first_block) {
  pdl_wait();
  if (first_block && threadIdx.x == 0) release_word(p.beside, 0);
}

// Few (entry, KV head) pairs: the blocks of a cluster share the keys of one, each a part as large, and join their parts.
// One entry of 2,048 keys, 12 heads of 128 on 2, sixteen blocks a pair: 7.8 us, the latency of a start (2), one walk and two cluster barriers.
template <int D, int NT>
__global__ void __launch_bounds__(32 * kWarps, NT == 1 ? 3 : 2) attention_q4_cluster_kernel(DecodeParams p) {
  constexpr int kRow = D + 4;
  extern __shared__ __align__(128) uint8_t shared_at[];
  const Shared<D, NT> shared{shared_at};
  if (p.settled == 0) {
    pdl_wait();
    pdl_launch_dependents();
  }
  if (p.settled == 2) begin_beside(p);
  const bool first_block = (blockIdx.x | blockIdx.y | blockIdx.z) == 0;
  const int group = p.num_heads / p.num_kv_heads, head_tiles = (group + 8 * NT - 1) / (8 * NT);
  const int entry = blockIdx.x, share = blockIdx.z;
  const int kv_head = blockIdx.y / head_tiles, head0 = (blockIdx.y - kv_head * head_tiles) * 8 * NT;
  int token = entry;
  if (p.entry_starts) {
    token = __ldcg(p.entry_starts + entry);
    if (__ldcg(p.entry_starts + entry + 1) - token != 1) {   // the whole cluster's; a grid without an entry must not end before the kernels ahead
      if (p.settled == 2 && first_block) end_beside(p, true);
      else if (p.settled && entry == 0) pdl_wait();
      return;
    }
  }
  const Visible seen(p, __ldcg(p.positions + entry));
  const int each = (seen.tiles + 8 * p.shares - 1) / (8 * p.shares) * 8;      // of a block: whole steps of its warps
  walk<D, NT>(p, shared, seen, entry, token, kv_head, head0, min(share * each, seen.tiles), min((share + 1) * each, seen.tiles), p.settled != 1);
  cluster_sync_all();
  const int heads_here = min(8 * NT, group - head0);
  const uint32_t joined_at = smem_addr(shared.joined());
  for (int i = share * static_cast<int>(blockDim.x) + threadIdx.x; i < heads_here * (D / 4); i += p.shares * blockDim.x) {
    const int h = i / (D / 4), column = (i - h * (D / 4)) * 4;
    Join join;
    for (int c = 0; c < p.shares; ++c) join.best = fmaxf(join.best, cluster_load(joined_at + (h * kRow + D) * 4, c));
#pragma unroll 4
    for (int c = 0; c < p.shares; ++c)
      join.add(cluster_load(joined_at + (h * kRow + D) * 4, c), cluster_load(joined_at + (h * kRow + D + 1) * 4, c),
               cluster_load_4(joined_at + (h * kRow + column) * 4, c));
    finish<D>(p, token, kv_head * group + head0 + h, column, join.best, join.total, join.value);
  }
  cluster_sync_all();   // nobody's shared memory goes while others read it
  if (p.settled == 2) {
    end_beside(p, first_block);
    pdl_launch_dependents();
  }
}

// Many pairs: the keys of all of them, in units of 8 tiles one pair behind the other, are dealt to the launch's blocks in even runs, so
// that no block waits for another's longer history.  A walk costs as much as kBegin units before its first one (its queries, its first
// rows' way, joining its warps), so a pair counts that many in front of its own, or a run of short pairs would outlast the others (the
// batch of 64 with histories of 0 to 4,095 keys: 39 us with most blocks idle for half of it).  A pair that lies in one block's run is
// finished there; of one that several share, each leaves its part in memory (`parts`: two places a block, the first for a pair
// that began in an earlier block) and a second kernel joins them.
constexpr int kBegin = 3;
__device__ __forceinline__ int units_for(const DecodeParams& p, int position) {
  const int tiles = Visible(p, position).tiles;
  return tiles > 0 ? ((tiles + 7) >> 3) + kBegin : 0;
}
__device__ __forceinline__ int units_of(const DecodeParams& p, int entry) {
  if (entry >= p.num_entries || (p.entry_starts && __ldcg(p.entry_starts + entry + 1) - __ldcg(p.entry_starts + entry) != 1)) return 0;
  return units_for(p, __ldcg(p.positions + entry));
}
constexpr int kRunEntries = 1024;   // entries whose lengths a block holds

template <int D, int NT>
__global__ void __launch_bounds__(32 * kWarps, NT == 1 ? 3 : 2) attention_q4_runs_kernel(DecodeParams p, float* __restrict__ parts) {
  constexpr int kRow = D + 4;
  extern __shared__ __align__(128) uint8_t shared_at[];
  const Shared<D, NT> shared{shared_at};
  __shared__ int positions[kRunEntries], ends[kRunEntries];    // ends: units up to and with an entry
  __shared__ int warp_units[kWarps];
  if (p.settled != 2) {
    pdl_wait();
    pdl_launch_dependents();
  } else {
    begin_beside(p);
  }
  const bool last = p.settled == 2 && blockIdx.x == 0;      // a grid that found nothing to do must not end before the kernels ahead
  const int group = p.num_heads / p.num_kv_heads, head_tiles = (group + 8 * NT - 1) / (8 * NT), pairs = p.num_kv_heads * head_tiles;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int whole = 0;
  for (int e0 = 0; e0 < p.num_entries; e0 += 32 * kWarps) {
    const int e = e0 + threadIdx.x;
    int position = -1;
    if (e < p.num_entries && !(p.entry_starts && __ldcg(p.entry_starts + e + 1) - __ldcg(p.entry_starts + e) != 1))
      position = __ldcg(p.positions + e);
    int upto = position >= 0 ? units_for(p, position) : 0;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, offset);
      if (lane >= offset) upto += v;
    }
    if (lane == 31) warp_units[warp] = upto;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) upto += warp_units[w];
      total += warp_units[w];
    }
    if (e < p.num_entries) {
      positions[e] = position;
      ends[e] = whole + upto;
    }
    whole += total;
    __syncthreads();
  }
  const long long all = static_cast<long long>(whole) * pairs;
  const long long runs = min(static_cast<long long>(gridDim.x), all);     // each with a unit at least
  if (blockIdx.x >= runs) {
    if (last) end_beside(p, true);
    return;
  }
  long long at = all * blockIdx.x / runs;
  const long long stop = all * (blockIdx.x + 1) / runs;
  int entry = 0;                                   // in which the run begins: the first that ends behind it
  for (int high = p.num_entries - 1; entry < high;) {
    const int middle = (entry + high) >> 1;
    if (static_cast<long long>(ends[middle]) * pairs > at) high = middle;
    else entry = middle + 1;
  }
  const auto units_at = [&](int e) { return ends[e] - (e > 0 ? ends[e - 1] : 0); };
  int units = units_at(entry);
  if (units == 0) {
    if (last) end_beside(p, true);
    return;
  }
  const int into = static_cast<int>(at - static_cast<long long>(ends[entry] - units) * pairs);
  int pair = into / units, unit = into - pair * units;
  while (at < stop && entry < p.num_entries) {
    const int token = p.entry_starts ? __ldcg(p.entry_starts + entry) : entry;
    const int kv_head = pair / head_tiles, head0 = (pair - kv_head * head_tiles) * 8 * NT;
    const int run = static_cast<int>(min(static_cast<long long>(units - unit), stop - at));
    // the run's own keys: units kBegin and behind
    const int own = max(unit - kBegin, 0), own_end = unit + run - kBegin;
    const bool whole_pair = own == 0 && own_end == units - kBegin;
    if (own_end > 0) {
      const Visible seen(p, positions[entry]);
      walk<D, NT>(p, shared, seen, entry, token, kv_head, head0, 8 * own, min(8 * own_end, seen.tiles));
      __syncthreads();
      const int heads_here = min(8 * NT, group - head0);
      const float* joined = shared.joined();
      if (whole_pair) {
        for (int i = threadIdx.x; i < heads_here * (D / 4); i += blockDim.x) {
          const int h = i / (D / 4), column = (i - h * (D / 4)) * 4;
          finish<D>(p, token, kv_head * group + head0 + h, column, joined[h * kRow + D], joined[h * kRow + D + 1],
                    *reinterpret_cast<const float4*>(joined + h * kRow + column));
        }
      } else {
        float* part = parts + (2 * static_cast<size_t>(blockIdx.x) + (own > 0 ? 0 : 1)) * (8 * NT * kRow);
        for (int i = threadIdx.x; i < heads_here * (kRow / 4); i += blockDim.x)
          reinterpret_cast<float4*>(part)[i] = reinterpret_cast<const float4*>(joined)[i];
      }
      __syncthreads();   // the next walk's queries and stages lie where this one's are
    }
    at += run;
    unit = 0;
    if (at < stop && ++pair == pairs) {
      pair = 0;
      do ++entry;
      while (entry < p.num_entries && (units = units_at(entry)) == 0);
    }
  }
  if (p.settled == 2) {
    end_beside(p, blockIdx.x == 0);
    pdl_launch_dependents();
  }
}

// Two blocks an (entry, pair): they join the parts of a pair that several runs share.  4 us for 48 entries of 8 pairs, two trips to memory (the
// lengths, the parts) behind a launch.
template <int D, int NT>
__global__ void __launch_bounds__(128) attention_q4_join_kernel(DecodeParams p, const float* __restrict__ parts, int blocks) {
  constexpr int kRow = D + 4;
  __shared__ int sums[2][4];
  pdl_wait();
  pdl_launch_dependents();
  const int group = p.num_heads / p.num_kv_heads, head_tiles = (group + 8 * NT - 1) / (8 * NT), pairs = p.num_kv_heads * head_tiles;
  const int entry = blockIdx.x, pair = blockIdx.y;
  int ahead = 0, whole = 0;
#pragma unroll 4
  for (int e = threadIdx.x; e < p.num_entries; e += 128) {
    const int units = units_of(p, e);
    whole += units;
    if (e < entry) ahead += units;
  }
  const int units = units_of(p, entry);
  ahead = __reduce_add_sync(0xffffffffu, ahead);
  whole = __reduce_add_sync(0xffffffffu, whole);
  if ((threadIdx.x & 31) == 0) {
    sums[0][threadIdx.x >> 5] = ahead;
    sums[1][threadIdx.x >> 5] = whole;
  }
  __syncthreads();
  if (units == 0) return;
  ahead = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3];
  whole = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
  const long long all = static_cast<long long>(whole) * pairs, start = static_cast<long long>(ahead) * pairs + static_cast<long long>(pair) * units;
  const long long last = start + units - 1, runs = min(static_cast<long long>(blocks), all);
  // the run that holds a unit x: the last one that begins at x or in front of it; the pair's keys begin behind its first kBegin
  const int first_run = static_cast<int>(((start + kBegin + 1) * runs - 1) / all), last_run = static_cast<int>(((last + 1) * runs - 1) / all);
  if (first_run == last_run) return;      // finished there
  const int kv_head = pair / head_tiles, head0 = (pair - kv_head * head_tiles) * 8 * NT, heads_here = min(8 * NT, group - head0);
  const int token = p.entry_starts ? p.entry_starts[entry] : entry;
  const auto part_of = [&](int r) { return parts + (2 * static_cast<size_t>(r) + (r == first_run ? 1 : 0)) * (8 * NT * kRow); };
  for (int i = blockIdx.z * 128 + threadIdx.x; i < heads_here * (D / 4); i += 256) {
    const int h = i / (D / 4), column = (i - h * (D / 4)) * 4;
    Join join;
    constexpr int kAtOnce = 8;        // parts that are asked for together; the maximum follows them
    for (int r = first_run; r <= last_run; r += kAtOnce) {
      float m[kAtOnce], l[kAtOnce];
      float4 v[kAtOnce];
#pragma unroll
      for (int c = 0; c < kAtOnce; ++c) {
        const float* part = part_of(min(r + c, last_run)) + h * kRow;
        m[c] = r + c <= last_run ? part[D] : -INFINITY;
        l[c] = part[D + 1];
        v[c] = *reinterpret_cast<const float4*>(part + column);
      }
      float best = join.best;
#pragma unroll
      for (int c = 0; c < kAtOnce; ++c) best = fmaxf(best, m[c]);
      const Join before = join;
      join = Join();
      join.best = best;
      join.add(before.best, before.total, before.value);
#pragma unroll
      for (int c = 0; c < kAtOnce; ++c) join.add(m[c], l[c], v[c]);
    }
    finish<D>(p, token, kv_head * group + head0 + h, column, join.best, join.total, join.value);
  }
}

// Shared memory beyond 48 KB and clusters of 16 blocks are asked for once on every device (a bit each in `asked`).
template <typename Kernel>
int ask_once(uint64_t* asked, Kernel kernel, int shared_bytes, bool clusters) {
  int device = 0;
  cudaError_t error = cudaGetDevice(&device);
  if (error == cudaSuccess && device < 64 && (*asked >> device & 1u)) return VIPERA_OK;
  if (error == cudaSuccess) error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared_bytes);
  if (error == cudaSuccess && clusters) error = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (error != cudaSuccess) return static_cast<int>(error);
  if (device < 64) *asked |= 1ull << device;
  return VIPERA_OK;
}

template <int D, int NT>
int launch(const DecodeParams& p, float* parts, int runs, cudaStream_t s) {
  constexpr int kSmem = Shared<D, NT>::kBytes;
  const int group = p.num_heads / p.num_kv_heads, head_tiles = (group + 8 * NT - 1) / (8 * NT);
  if (p.num_kv_heads * head_tiles > 65535) return VIPERA_BAD_SHAPE;
  if (p.shares == 0) {
    const auto kernel = attention_q4_runs_kernel<D, NT>;
    static uint64_t asked = 0;
    const int ready = ask_once(&asked, kernel, kSmem, false);
    if (ready != VIPERA_OK) return ready;
    const int status = vipera_launch(kernel, dim3(runs), 32 * kWarps, kSmem, s, p, parts);
    if (status != VIPERA_OK) return status;
    return vipera_launch(attention_q4_join_kernel<D, NT>, dim3(p.num_entries, p.num_kv_heads * head_tiles, 2), 128, 0, s, p, parts, runs);
  }
  const auto kernel = attention_q4_cluster_kernel<D, NT>;
  static uint64_t asked = 0;
  const int ready = ask_once(&asked, kernel, kSmem, true);
  if (ready != VIPERA_OK) return ready;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(p.num_entries, p.num_kv_heads * head_tiles, p.shares);
  config.blockDim = dim3(32 * kWarps);
  config.dynamicSmemBytes = kSmem;
  config.stream = s;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = vipera_pdl_enabled() ? 1 : 0;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = 1;
  attributes[1].val.clusterDim.y = 1;
  attributes[1].val.clusterDim.z = static_cast<unsigned>(p.shares);
  config.attrs = attributes;
  config.numAttrs = 2;
  const cudaError_t error = cudaLaunchKernelEx(&config, kernel, p);
  return error == cudaSuccess ? VIPERA_OK : static_cast<int>(error);
}

}  // namespace

#include "attention_q4_rows.cuh"

namespace {

bool on_16_bytes(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

VIPERA_API int vipera_attention_q4_params_size() { return static_cast<int>(sizeof(DecodeParams)); }

// Floats of scratch for `runs` runs: two parts each, of the query heads that a block has.
VIPERA_API size_t vipera_attention_q4_parts(int runs, int num_heads, int num_kv_heads, int head_dim) {
  return static_cast<size_t>(runs) * 2 * (num_heads / num_kv_heads > 8 ? 16 : 8) * (head_dim + 4);
}

// Attention of the entries that bring one token (all of them where entry_starts is null).  p->shares: the blocks, a power of two up to
// 16, that share an entry's keys; 0: all entries' keys go to `runs` blocks in even runs, and `parts` holds their parts.
VIPERA_API int vipera_attention_q4_decode(const DecodeParams* given, float* parts, size_t parts_floats, int runs, void* stream) {
  DecodeParams p = *given;
  if (p.num_entries <= 0) return VIPERA_OK;
  if (p.num_heads <= 0 || p.num_kv_heads <= 0 || p.num_heads % p.num_kv_heads || p.keep_first < 0 || p.page_size <= 0 ||
      p.page_size % 16 || p.num_heads > 65535 || p.shares < 0 || p.shares > 16 || (p.shares & (p.shares - 1)) ||
      (p.head_dim != 64 && p.head_dim != 128))
    return VIPERA_BAD_SHAPE;
  if (p.shares == 0 && (runs <= 0 || p.num_entries > kRunEntries || !parts || !on_16_bytes(parts) ||
                        parts_floats < vipera_attention_q4_parts(runs, p.num_heads, p.num_kv_heads, p.head_dim)))
    return VIPERA_BAD_ARGUMENT;
  if (p.settled < 0 || p.settled > 2 || (p.settled == 2 && !p.beside)) return VIPERA_BAD_ARGUMENT;
  if (p.sink_values) p.sink = 1;
  if (!on_16_bytes(p.q) || !on_16_bytes(p.k_codes) || !on_16_bytes(p.v_codes) || !on_16_bytes(p.k_scales) || !on_16_bytes(p.v_scales) ||
      (reinterpret_cast<uintptr_t>(p.out) & 7))
    return VIPERA_BAD_ARGUMENT;
  p.magic = 0x43004300u;
  p.page_shift = -1;
  if ((p.page_size & (p.page_size - 1)) == 0)
    for (p.page_shift = 0; (1 << p.page_shift) < p.page_size;) ++p.page_shift;
  const bool wide = p.num_heads / p.num_kv_heads > 8;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (p.head_dim == 128) return wide ? launch<128, 2>(p, parts, runs, s) : launch<128, 1>(p, parts, runs, s);
  return wide ? launch<64, 2>(p, parts, runs, s) : launch<64, 1>(p, parts, runs, s);
}

VIPERA_API int vipera_attention_q4_rows_params_size() { return static_cast<int>(sizeof(RowsParams)); }

// Attention of every token of a step, q of `dtype` and out too: partials per (token, head, place) in `scratch`, then the endings that
// the joining kernel knows (`positions` [tokens]; sink, sink_values and gate as for the kernel of single tokens).
VIPERA_API int vipera_attention_q4_rows(const RowsParams* given, void* out, int dtype, int head_dim, const int* positions, int sink,
                                        const float* sink_values, const float* gate, long long gate_stride, int gate_per_head,
                                        float* scratch, size_t scratch_floats, void* stream) {
  RowsParams p = *given;
  if (p.num_entries <= 0 || p.num_tokens <= 0) return VIPERA_OK;
  if (p.num_heads <= 0 || p.num_kv_heads <= 0 || p.num_heads % p.num_kv_heads || p.keep_first < 0 || p.page_size <= 0 ||
      p.page_size % 16 || p.num_heads > 65535 || p.num_splits <= 0 || p.num_splits > 128 || p.chunk <= 0 || p.chunk % 64 ||
      (head_dim != 64 && head_dim != 128))
    return VIPERA_BAD_SHAPE;
  if (dtype != VIPERA_F32 && dtype != VIPERA_BF16) return VIPERA_BAD_DTYPE;
  if (p.window <= 0) p.keep_first = 0;
  if (sink_values) sink = 1;
  const size_t rows = static_cast<size_t>(p.num_tokens) * p.num_heads * (p.num_splits + (p.keep_first > 0 ? 1 : 0));
  const size_t pairs = (2 * rows + 3) / 4 * 4;
  // the joining kernel's lanes store a 32nd of a row at once
  const uintptr_t piece = static_cast<uintptr_t>(head_dim / 32) * (dtype == VIPERA_F32 ? 4 : 2);
  if (reinterpret_cast<uintptr_t>(out) & (piece - 1)) return VIPERA_BAD_ARGUMENT;
  if (!scratch || scratch_floats < pairs + rows * head_dim || !on_16_bytes(scratch) || !on_16_bytes(p.k_codes) ||
      !on_16_bytes(p.v_codes) || !on_16_bytes(p.k_scales) || !on_16_bytes(p.v_scales))
    return VIPERA_BAD_ARGUMENT;
  p.partial_ml = scratch;
  p.partial_out = scratch + pairs;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int status = VIPERA_BAD_DTYPE;
  const bool wide = dtype == VIPERA_F32;
  if (wide) status = head_dim == 128 ? launch_rows<128, float, 1>(p, s) : launch_rows<64, float, 2>(p, s);
  else if (dtype == VIPERA_BF16) status = head_dim == 128 ? launch_rows<128, __nv_bfloat16, 2>(p, s) : launch_rows<64, __nv_bfloat16, 2>(p, s);
  if (status != VIPERA_OK) return status;
  const JoinParams join{p.partial_ml, p.partial_out, out, positions, p.entry_starts + p.num_entries, sink_values, gate, gate_stride, gate_per_head,
                        sink, p.num_tokens, p.num_heads, p.window, p.keep_first, p.chunk, p.num_splits};
  if (wide) return head_dim == 128 ? launch_join<128, float>(join, s) : launch_join<64, float>(join, s);
  return head_dim == 128 ? launch_join<128, __nv_bfloat16>(join, s) : launch_join<64, __nv_bfloat16>(join, s);
}
