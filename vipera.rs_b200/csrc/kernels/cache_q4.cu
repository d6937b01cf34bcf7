// A cache in 4 bits: the maps of a step, the write of a step's keys and values, and rows read back.
// Formats: q4.cuh.  Attention over such pages: attention_q4.cu.
#include "q4.cuh"

namespace {

// ---------------------------------------------------------------------------------------
// The maps of a step, from its requests' lengths
// ---------------------------------------------------------------------------------------
struct MapsParams {
  const int* entry_starts;   // [entries + 1] cumulative token counts
  const int* entry_pos0;     // [entries] position of each entry's first token
  const int* page_starts;    // [entries + 1] where each entry's pages begin in `pages`; null: block_table is read, not written
  const int* pages;
  int* block_table;          // [entries, table_width], -1 where no page is held
  int* positions;            // [tokens] or null, as the next two
  int* token_entry;
  int* slots;                // page * page_size + place in the page; -1 without a page
  int num_entries, num_tokens, num_pages, table_width, page_size;
};

// Block (x, e): its share of entry e's table row and of its tokens.  What bounds it is the latency of two trips to
// memory (lengths, then pages) behind the launch, not bytes, so an entry's lengths are asked for at once and nothing
// is searched: a token's entry is the block's.  It does not let the kernel behind it start early: kernels of a step read positions and
// tables before their own wait, and must find them written.
// 64 entries of one token, tables of 33 pages: 3.7 us; 101 entries with 8,192 tokens, tables of 2,001 pages: 4.4 us.
__global__ void __launch_bounds__(256) step_maps_kernel(MapsParams p) {
  pdl_wait();
  const int e = blockIdx.y;
  const int begin = max(p.entry_starts[e], 0), end = min(p.entry_starts[e + 1], p.num_tokens);
  const int pos0 = p.entry_pos0[e];
  int first_page = 0, held = 0;
  if (p.page_starts) {
    first_page = max(p.page_starts[e], 0);
    held = min(p.page_starts[e + 1], p.num_pages) - first_page;
  }
  const int at = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
  int* row = p.block_table + static_cast<size_t>(e) * p.table_width;
  if (p.page_starts)
    for (int w = at; w < p.table_width; w += step) row[w] = w < held ? p.pages[first_page + w] : -1;
  for (int t = begin + at; t < end; t += step) {
    const int position = pos0 + t - begin;
    if (p.positions) p.positions[t] = position;
    if (p.token_entry) p.token_entry[t] = e;
    if (p.slots) {
      int page = -1, place = 0;
      if (position >= 0) {
        const int index = position / p.page_size;
        place = position - index * p.page_size;
        if (p.page_starts) page = index < held ? p.pages[first_page + index] : -1;
        else page = index < p.table_width ? row[index] : -1;
      }
      p.slots[t] = page < 0 ? -1 : page * p.page_size + place;
    }
  }
  __threadfence();
}

// ---------------------------------------------------------------------------------------
// Rotation, queries to their type, keys and values to 4 bits
// ---------------------------------------------------------------------------------------
enum RopeStyle { ROPE_NONE = 0, ROPE_NEOX = 1, ROPE_INTERLEAVED = 2 };

struct StoreParams {
  const float* qkv;          // [tokens, row_stride]: q heads, k heads, v heads of d values each
  long long row_stride;
  void* q_out;               // [tokens, heads * d]
  uint8_t *k_codes, *v_codes;
  __nv_bfloat16 *k_scales, *v_scales;
  const int* positions;
  const float *cos_table, *sin_table;   // [positions, rot_dims / 2]
  const int* slots;          // null: nothing is written but q
  long long num_slots;       // slots of the pool: a slot outside is not written
  int table_rows;            // rows of the tables: the last serves positions beyond
  int num_tokens, num_heads, num_kv_heads, head_dim, rot_dims, style, page_size;
};

// Where a token's rows of a KV head go.
struct Row {
  bool write;
  size_t row;
};
__device__ __forceinline__ Row row_of(const StoreParams& p, int slot, int kv_head) {
  const bool write = slot >= 0 && slot < p.num_slots;
  const int page = write ? slot / p.page_size : 0, place = write ? slot - page * p.page_size : 0;
  return Row{write, (static_cast<size_t>(page) * p.num_kv_heads + kv_head) * p.page_size + place};
}

// An octet of a head on its way: queries to their type, keys and values to codes.  Four neighbouring lanes hold a group of 32 channels and
// find its ends together; every lane of the warp takes part.
template <typename T>
__device__ __forceinline__ void put_octet(const StoreParams& p, const float (&x)[8], int t, int h, int octet, bool live, const Row& to) {
  const bool is_q = h < p.num_heads, is_v = h >= p.num_heads + p.num_kv_heads;
  if (live && is_q) {
    T* q = static_cast<T*>(p.q_out) + (static_cast<size_t>(t) * p.num_heads + h) * p.head_dim + octet * 8;
    store_four_as<T>(q, x[0], x[1], x[2], x[3]);
    store_four_as<T>(q + 4, x[4], x[5], x[6], x[7]);
  }
  if (!__any_sync(0xffffffffu, live && !is_q && to.write)) return;
  float high = x[0], low = x[0];
  bool fine = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    high = fmaxf(high, x[i]);
    low = fminf(low, x[i]);
    fine = fine && fabsf(x[i]) <= 3.402823466e38f;
  }
#pragma unroll
  for (int offset = 1; offset <= 2; offset <<= 1) {
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, offset));
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, offset));
    fine = __shfl_xor_sync(0xffffffffu, static_cast<int>(fine), offset) && fine;
  }
  if (!live || is_q || !to.write) return;
  const float scale = fine ? q4::round5((high >= -low ? high : low) * -0.125f) : __int_as_float(0x7fffffff);
  uint32_t code[8];
  q4::codes_of(x, scale, code);
  const int groups = p.head_dim / q4::kGroup, g = octet >> 2, quarter = octet & 3;
  if (quarter == 0) (is_v ? p.v_scales : p.k_scales)[to.row * groups + g] = __float2bfloat16_rn(scale);
  if (is_v) {
    uint16_t* units = reinterpret_cast<uint16_t*>(p.v_codes) + to.row * (p.head_dim / 4);
    units[(2 * quarter) * groups + g] = static_cast<uint16_t>(code[0] | code[1] << 4 | code[2] << 8 | code[3] << 12);
    units[(2 * quarter + 1) * groups + g] = static_cast<uint16_t>(code[4] | code[5] << 4 | code[6] << 8 | code[7] << 12);
  } else {
    reinterpret_cast<uint32_t*>(p.k_codes)[to.row * (p.head_dim >> 3) + quarter * groups + g] =
        code[0] | code[2] << 4 | code[4] << 8 | code[6] << 12 | (code[1] | code[3] << 4 | code[5] << 8 | code[7] << 12) << 16;
  }
}

__device__ __forceinline__ void load_octet(float (&x)[8], const float* from) {
  *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(from);
  *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(from + 4);
}

// A thread has an octet of a head of a token.  Every product and sum of the rotation is rounded by itself (no fused multiply-add), so that a
// key next to a border between two codes falls the same way wherever the rotation is computed in 32 bits.  VEC: rows start on 16 bytes
// and the rotation's halves are whole octets.
// 2,048 tokens of 28 + 2 x 4 heads of 128: 17 us, bound by instructions (38 MB read, 16 MB written); an octet of both halves a thread, which
// reads the row and the tables once, takes 19 us, and two or four heads a thread 20 to 21 (fewer threads, longer chains).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) rope_cache_q4_kernel(StoreParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int octets = p.head_dim >> 3;
  const int all_heads = p.num_heads + 2 * p.num_kv_heads;
  const uint32_t item = blockIdx.x * blockDim.x + threadIdx.x, per_token = all_heads * octets;     // the launcher keeps them below 2^31
  const bool live = item < static_cast<uint32_t>(p.num_tokens) * per_token;
  const int t = live ? static_cast<int>(item / per_token) : 0;
  const int rest = live ? static_cast<int>(item - static_cast<uint32_t>(t) * per_token) : 0;
  const int h = rest / octets, octet = rest - h * octets, c0 = octet * 8;
  const bool is_q = h < p.num_heads, is_v = h >= p.num_heads + p.num_kv_heads;
  const float* head = p.qkv + static_cast<size_t>(t) * p.row_stride + static_cast<size_t>(h) * p.head_dim;
  const int position = live ? p.positions[t] : 0;
  const int slot = live && !is_q && p.slots ? p.slots[t] : -1;
  const int half = p.rot_dims >> 1;
  const size_t table_row = static_cast<size_t>(max(min(position, p.table_rows - 1), 0)) * half;
  float x[8];
  if (VEC) {
    load_octet(x, head + c0);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = head[c0 + i];
  }
  if (!is_v && p.style != ROPE_NONE && c0 < p.rot_dims) {
    if (p.style == ROPE_INTERLEAVED) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        if (c0 + i < p.rot_dims) {
          const float c = p.cos_table[table_row + (c0 + i) / 2], s = p.sin_table[table_row + (c0 + i) / 2];
          const float a = x[i], b = x[i + 1];
          x[i] = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
          x[i + 1] = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
        }
      }
    } else if (VEC) {   // half is a multiple of 8: the octet lies in one half
      const bool low = c0 < half;
      const int i0 = low ? c0 : c0 - half, other = low ? c0 + half : c0 - half;
      float y[8], c[8], s[8];
      load_octet(y, head + other);
      load_octet(c, p.cos_table + table_row + i0);
      load_octet(s, p.sin_table + table_row + i0);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = low ? __fsub_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], s[i]))
                   : __fadd_rn(__fmul_rn(y[i], s[i]), __fmul_rn(x[i], c[i]));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = c0 + i;
        if (at < p.rot_dims) {
          const bool low = at < half;
          const int pair = low ? at : at - half;
          const float y = head[low ? at + half : at - half];
          const float c = p.cos_table[table_row + pair], s = p.sin_table[table_row + pair];
          x[i] = low ? __fsub_rn(__fmul_rn(x[i], c), __fmul_rn(y, s)) : __fadd_rn(__fmul_rn(y, s), __fmul_rn(x[i], c));
        }
      }
    }
  }
  put_octet<T>(p, x, t, h, octet, live, row_of(p, slot, max(h - p.num_heads - (is_v ? p.num_kv_heads : 0), 0)));
}

// ---------------------------------------------------------------------------------------
// Rows read back
// ---------------------------------------------------------------------------------------
struct ExpandParams {
  const uint8_t *k_codes, *v_codes;
  const __nv_bfloat16 *k_scales, *v_scales;
  void *k_room, *v_room;     // [pages, page size, KV heads, d], the cache's page numbers
  const int* entry_starts;
  const int* entry_pos0;
  const int* block_table;
  int table_width, page_size, num_entries, num_pages, num_kv_heads, head_dim, window, keep_first, skip_single;
};

constexpr int kSlab = 1024;   // entries a block looks over at a time

// The rows that an entry's tokens see are those of positions [first, last] and, with a window, [0, kept).
struct Seen {
  int first, last, kept;
};
__device__ __forceinline__ Seen seen_by(const ExpandParams& p, int e) {
  const int count = p.entry_starts[e + 1] - p.entry_starts[e], pos0 = p.entry_pos0[e];
  Seen s{0, -1, 0};
  if (count <= 0 || pos0 < 0 || (p.skip_single && count == 1)) return s;
  s.first = p.window > 0 ? max(0, pos0 - p.window + 1) : 0;
  s.last = min(pos0 + count - 1, p.table_width * p.page_size - 1);
  s.kept = p.window > 0 ? min(p.keep_first, s.first) : 0;
  return s;
}

// Eight channels of a row as numbers.
__device__ __forceinline__ void key_octet(float (&x)[8], uint32_t w, float scale) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = static_cast<float>(static_cast<int>((w >> (4 * j)) & 15u) - 8) * scale;
    x[2 * j + 1] = static_cast<float>(static_cast<int>((w >> (16 + 4 * j)) & 15u) - 8) * scale;
  }
}
__device__ __forceinline__ void value_octet(float (&x)[8], uint32_t lo, uint32_t hi, float scale) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[j] = static_cast<float>(static_cast<int>((lo >> (4 * j)) & 15u) - 8) * scale;
    x[4 + j] = static_cast<float>(static_cast<int>((hi >> (4 * j)) & 15u) - 8) * scale;
  }
}

// A unit of work is one page of one entry.  Every block counts the units of all entries for itself (two trips to memory and a scan),
// then takes every gridDim-th: the load is even however the lengths differ, and the launch needs no count from the host, so that
// a captured one serves any lengths.  A thread has an octet of the keys and the same of the values, kAhead rows of them at once.
// 2,048 tokens of 4 KV heads of 128 (1.2 MB read, 4.2 MB written): 8 us, of which the bytes are one: a chain of five trips to memory (lengths,
// lengths of the unit's entry, table, codes, the write) bounds it.
constexpr int kAhead = 4;
template <typename T>
__global__ void __launch_bounds__(256) expand_q4_kernel(ExpandParams p) {
  __shared__ int ends[kSlab];      // pages up to and with this entry
  __shared__ int warp_totals[8];
  pdl_launch_dependents();
  pdl_wait();
  const int octets = p.head_dim >> 3, groups = p.head_dim / q4::kGroup;
  const int per_unit = p.page_size * p.num_kv_heads * octets;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int slab = 0; slab < p.num_entries; slab += kSlab) {
    const int entries = min(kSlab, p.num_entries - slab);
    int mine[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = threadIdx.x * 4 + i;
      mine[i] = 0;
      if (e < entries) {
        const Seen s = seen_by(p, slab + e);
        if (s.last >= s.first) {
          const int low = s.first / p.page_size;
          mine[i] = s.last / p.page_size - low + 1 + (s.kept > 0 ? min((s.kept - 1) / p.page_size + 1, low) : 0);
        }
      }
      sum += mine[i];
    }
    int before = sum;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, offset);
      if (lane >= offset) before += v;
    }
    __syncthreads();
    if (lane == 31) warp_totals[warp] = before;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if (w < warp) before += warp_totals[w];
      total += warp_totals[w];
    }
    before -= sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      before += mine[i];
      ends[threadIdx.x * 4 + i] = before;
    }
    __syncthreads();
    for (int index = blockIdx.x; index < total; index += gridDim.x) {
      int low = 0, high = entries - 1;      // the first entry whose end is above index
      while (low < high) {
        const int middle = (low + high) >> 1;
        if (ends[middle] > index) high = middle;
        else low = middle + 1;
      }
      const int e = slab + low;
      const Seen s = seen_by(p, e);
      const int first_page = s.first / p.page_size;
      const int kept_pages = s.kept > 0 ? min((s.kept - 1) / p.page_size + 1, first_page) : 0;
      const int within = index - (low > 0 ? ends[low - 1] : 0);
      const int at = within < kept_pages ? within : first_page + within - kept_pages;
      const int page = p.block_table[static_cast<size_t>(e) * p.table_width + at];
      if (page < 0 || page >= p.num_pages) continue;
      const size_t page_row = static_cast<size_t>(page) * p.num_kv_heads * p.page_size;
      for (int i0 = threadIdx.x; i0 < per_unit; i0 += kAhead * blockDim.x) {
        uint32_t k[kAhead], v_lo[kAhead], v_hi[kAhead];
        float k_scale[kAhead], v_scale[kAhead];
        size_t to[kAhead];
        bool seen[kAhead];
#pragma unroll
        for (int c = 0; c < kAhead; ++c) {     // rows of a KV head lie together in the page: (KV head, place, octet)
          const int i = i0 + c * blockDim.x;
          const int row_in = i / octets, octet = i - row_in * octets, kv_head = row_in / p.page_size, place = row_in - kv_head * p.page_size;
          const int position = at * p.page_size + place, g = octet >> 2, quarter = octet & 3;
          seen[c] = i < per_unit && ((position >= s.first && position <= s.last) || position < s.kept);
          if (!seen[c]) continue;
          const size_t row = page_row + row_in;
          k[c] = reinterpret_cast<const uint32_t*>(p.k_codes)[row * octets + quarter * groups + g];
          const uint16_t* units = reinterpret_cast<const uint16_t*>(p.v_codes) + row * (p.head_dim / 4);
          v_lo[c] = units[(2 * quarter) * groups + g];
          v_hi[c] = units[(2 * quarter + 1) * groups + g];
          k_scale[c] = __bfloat162float(p.k_scales[row * groups + g]);
          v_scale[c] = __bfloat162float(p.v_scales[row * groups + g]);
          to[c] = ((static_cast<size_t>(page) * p.page_size + place) * p.num_kv_heads + kv_head) * p.head_dim + octet * 8;
        }
#pragma unroll
        for (int c = 0; c < kAhead; ++c) {
          if (!seen[c]) continue;
          float x[8];
          key_octet(x, k[c], k_scale[c]);
          store_four_as<T>(static_cast<T*>(p.k_room) + to[c], x[0], x[1], x[2], x[3]);
          store_four_as<T>(static_cast<T*>(p.k_room) + to[c] + 4, x[4], x[5], x[6], x[7]);
          value_octet(x, v_lo[c], v_hi[c], v_scale[c]);
          store_four_as<T>(static_cast<T*>(p.v_room) + to[c], x[0], x[1], x[2], x[3]);
          store_four_as<T>(static_cast<T*>(p.v_room) + to[c] + 4, x[4], x[5], x[6], x[7]);
        }
      }
    }
    __syncthreads();
  }
}

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace

VIPERA_API int vipera_step_maps_params_size() { return static_cast<int>(sizeof(MapsParams)); }
VIPERA_API int vipera_rope_cache_q4_params_size() { return static_cast<int>(sizeof(StoreParams)); }
VIPERA_API int vipera_expand_q4_params_size() { return static_cast<int>(sizeof(ExpandParams)); }

VIPERA_API int vipera_step_maps(const MapsParams* p, void* stream) {
  if (p->num_entries <= 0) return VIPERA_OK;
  if (p->page_size <= 0 || p->table_width < 0 || p->num_entries > 65535 || p->num_tokens < 0) return VIPERA_BAD_SHAPE;
  const int longest = p->page_starts && p->table_width > p->num_tokens ? p->table_width : p->num_tokens;
  const int blocks = longest <= 256 ? 1 : longest >= 8192 ? 8 : (longest + 1023) / 1024;
  return vipera_launch(step_maps_kernel, dim3(blocks, p->num_entries), 256, 0, static_cast<cudaStream_t>(stream), *p);
}

VIPERA_API int vipera_rope_cache_q4(const StoreParams* p, int dtype, void* stream) {
  if (p->num_tokens <= 0) return VIPERA_OK;
  if (p->head_dim <= 0 || p->head_dim % q4::kGroup || p->head_dim > 256 || p->num_heads <= 0 || p->num_kv_heads <= 0 ||
      p->page_size <= 0 || p->rot_dims < 0 || p->rot_dims > p->head_dim || p->rot_dims % 2 ||
      (p->style != ROPE_NONE && p->rot_dims > 0 && p->table_rows <= 0))
    return VIPERA_BAD_SHAPE;
  // rows are written in pieces of up to 16 bytes
  if (!aligned(p->q_out, 16) || !aligned(p->k_codes, 16) || !aligned(p->v_codes, 16)) return VIPERA_BAD_ARGUMENT;
  const int half = p->rot_dims / 2;
  const bool vec = aligned(p->qkv, 16) && p->row_stride % 4 == 0 &&
                   (p->style != ROPE_NEOX || half == 0 || (half % 8 == 0 && aligned(p->cos_table, 16) && aligned(p->sin_table, 16)));
  const long long items = static_cast<long long>(p->num_tokens) * (p->num_heads + 2 * p->num_kv_heads) * (p->head_dim / 8);
  const long long blocks = (items + 255) / 256;
  if (blocks > 0x7fffffLL) return VIPERA_BAD_SHAPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(blocks));
  if (dtype == VIPERA_BF16)
    return vec ? vipera_launch(rope_cache_q4_kernel<__nv_bfloat16, true>, grid, 256, 0, s, *p)
               : vipera_launch(rope_cache_q4_kernel<__nv_bfloat16, false>, grid, 256, 0, s, *p);
  if (dtype == VIPERA_F32)
    return vec ? vipera_launch(rope_cache_q4_kernel<float, true>, grid, 256, 0, s, *p)
               : vipera_launch(rope_cache_q4_kernel<float, false>, grid, 256, 0, s, *p);
  return VIPERA_BAD_DTYPE;
}

VIPERA_API int vipera_expand_q4(const ExpandParams* p, int dtype, int blocks, void* stream) {
  if (p->num_entries <= 0) return VIPERA_OK;
  if (p->head_dim <= 0 || p->head_dim % q4::kGroup || p->head_dim > 256 || p->num_kv_heads <= 0 || p->page_size <= 0 ||
      p->table_width <= 0 || blocks <= 0 || static_cast<long long>(p->table_width) * p->page_size > 0x7fffffffLL)
    return VIPERA_BAD_SHAPE;
  if (!aligned(p->k_room, 16) || !aligned(p->v_room, 16) || !aligned(p->k_codes, 16) || !aligned(p->v_codes, 16)) return VIPERA_BAD_ARGUMENT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == VIPERA_BF16) return vipera_launch(expand_q4_kernel<__nv_bfloat16>, dim3(blocks), 256, 0, s, *p);
  if (dtype == VIPERA_F32) return vipera_launch(expand_q4_kernel<float>, dim3(blocks), 256, 0, s, *p);
  return VIPERA_BAD_DTYPE;
}
