// Attention of a step's portions over pages of 4 bits (formats: q4.cuh) on the fifth-generation tensor cores, bfloat16 steps, heads of
// 64 and 128: the rows are unpacked on their way to shared memory, never to memory.
//
// A block is 256 of the (token, query head) rows of one request and KV head, two tiles of 128, and a split of the keys; both tiles use
// every 128 keys and values that the block unpacks.  (A tile of 128 tokens of one head would unpack a history group times as often, and
// a portion of a few tokens would leave its rows empty: 18 tokens of 7 heads fill one tile.)  A chain of work goes with each: softmax warps,
// scores and output in tensor memory, an issuing warp.  Scores are computed 64 keys at a time into two places in turn, so that a chain's
// products run while it computes the weights of the 64 before.  Where a block has one tile of rows, both chains work at it, each at every
// second 64 keys, and join their outputs at the end.
//
//   unpacking  four warps, a thread a key: the next 128 rows' codes are asked for while these become bfloat16 numbers, exactly: u of a
//              code moved to the top of the fraction under 0x4180 is 16 + u, and (16 + u) s - 24 s = (u - 8) s in one rounding,
//              which rounds nothing.  Shared rows are 128 bytes with the 16-byte pieces swizzled; a value's
//              channels lie in the order in which its word holds them (a channel of group g beside the same one of group g + 1),
//              which orders the output's columns and is undone when they leave.
//   scores     S = Q K^T, tcgen05.mma 128 x 64 x d.
//   softmax    a thread a row: the largest of 64 scores, then weights and their sum, in 32 bits.  The maximum follows when it has
//              grown by 2^8, so that the outputs are rarely rescaled.  Weights go back to tensor memory as bfloat16, over the
//              scores, and are the left operand from there: shared memory, whose rate bounds products of two shared
//              operands of 128 rows, then feeds this product's right one alone.
//   output     O += P V, 128 x d x 64 in tensor memory.  S, S, O and O of 128 columns are all of it.
//
// A block whose rows are all there is (one split) writes them; else maxima, sums and outputs go to `partial_ml` and `partial_out`, and a second
// kernel joins them (kept first keys are a split of their own, as in attention_q4_rows.cuh).  Rows that hold no visible key of the block
// are zeros and are never read.  A value's group that is not finite is held as zeros, and its key is noted for the softmax, which makes the
// outputs NaN of the rows that see it and of no other.  Every wait is bounded: one that runs out leaves an error in the
// status word, and every role runs to its end.
//
// What bounds it.  2,048 tokens of 28 heads of 128 on 4: 49 us, 57 from a cold cache, 617 and 525 TFLOP/s (of 1,661 measured; expanding and the
// flash kernel take 69 and 73).  A block takes 5 us to its first scores and 2.5 to its ending, and 4,200 clocks for 128 keys of its 256
// rows: the exponentials alone are 2,048 (16 a clock), the tensor cores are busy for 2,700 (products of 64 columns cost as much as of 128),
// and both chains' softmax warps and the unpacking ones share the issue slots, of which they take 2,700.  Without the rows' loads 51 us (of
// 55, an earlier form), without the exponentials 55, without both 47.  Scores of 128 keys at once, weights and products one behind the
// other, took 6,000 clocks, with the products of both tiles from one warp in turn 4,700; rows asked for a whole tile ahead 4 % longer
// (registers), eight unpacking warps 7 % longer there and 10 % shorter where blocks have one tile.  A lone block's 128 keys of 128 rows
// take 2 us: the unpacking warps' loads and work.
#include "attention_q4_join.cuh"
#include "q4.cuh"
#include "tcgen05.cuh"

enum { ATTENTION_Q4_WAIT_EXPIRED = 3 };

namespace {

struct PortionParams {
  const __nv_bfloat16* q;         // [tokens, heads, d]
  __nv_bfloat16* out;
  const uint8_t *k_codes, *v_codes;
  const __nv_bfloat16 *k_scales, *v_scales;
  const int* entry_starts;
  const int* entry_pos0;
  const int* block_table;
  const float* sink_values;
  const float* gate;
  long long gate_stride;
  float* partial_ml;              // null: the block's split is the only one
  float* partial_out;
  int* status;
  int* beside;                    // for single tokens that run beside (attention_q4_join.cuh); null: none do
  int gate_per_head, sink;
  int table_width, page_size, num_pages, num_entries, num_tokens, num_heads, num_kv_heads, head_dim;
  float scale;
  int window, keep_first, chunk, num_splits, skip_single;
  int block_rows;                 // rows of a block: 256, or 128 (a tile alone)
};

constexpr int kTileRows = 128, kKeys = 128;
constexpr int kSoftmaxWarps = 8, kUnpackWarp = kSoftmaxWarps, kUnpackThreads = 128, kIssueWarp = kUnpackWarp + 4, kThreads = 32 * (kIssueWarp + 2);
constexpr int kHalfBytes = 128 * 128;                       // 128 rows of 64 values
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMaxSlack = 8.0f;                           // in powers of two
constexpr uint32_t kTmemCols = 512;                         // S of both tiles, O of both tiles

struct Job {
  int entry, row0, rows, token0, pos0;   // of the entry's (token, head) rows: the block's first and how many; its first token and position
};

struct Shared {
  uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2][2], p_full[2][2], pv_done[2][2];      // the last three by chain and buffer
  uint4 bad_any[4];                // of the last four tiles of keys: those with a group of values that is not finite
  uint32_t bad[4][4][4];           // [tile & 3][group][32 keys]
  float4 told[2][kTileRows];       // a pair's chains: maximum, sum and noted groups of every row
  uint32_t tmem;
  int abort_flag;
  Job job;
};

// (Without the pauses of the shared form: a role that waits here is asked for next, and its warps are few.)
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status) {
  for (uint32_t spin = 0; spin < tcgen05::kWaitLimit; ++spin) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(shared_address(bar)), "r"(parity) : "memory");
    if (done) return;
    if ((spin & 1023u) == 1023u && *abort_flag) return;
  }
  *abort_flag = 1;
  atomicExch(status, ATTENTION_Q4_WAIT_EXPIRED);
}

// D (tensor memory) += A . B, A in tensor memory (two bfloat16 of a row side by side in 32 bits), B in shared memory
__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, leader;\n elect.sync _|leader, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @leader tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

__device__ __forceinline__ void tensor_load_32(uint32_t from, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(from));
}
__device__ __forceinline__ void tensor_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tensor_store_32(uint32_t to, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(to), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tensor_load_16(uint32_t from, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(from));
}
__device__ __forceinline__ void tensor_store_16(uint32_t to, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(to), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                 "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tensor_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 2^x by the hardware's approximation, near enough for weights that are rounded to bfloat16; 2^-inf = 0.
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two numbers side by side: an instruction for both.
__device__ __forceinline__ unsigned long long both(float x) {
  const unsigned long long bits = __float_as_uint(x);
  return bits << 32 | bits;
}
__device__ __forceinline__ void scaled_pair(float& a, float& b, uint32_t x, uint32_t y, unsigned long long scale, unsigned long long shift) {
  asm("{\n .reg .b64 v;\n mov.b64 v, {%2, %3};\n fma.rn.f32x2 v, v, %4, %5;\n mov.b64 {%0, %1}, v;\n}\n"
      : "=f"(a), "=f"(b) : "r"(x), "r"(y), "l"(scale), "l"(shift));
}
__device__ __forceinline__ void add_pair(unsigned long long& sum, float a, float b) {
  asm("{\n .reg .b64 v;\n mov.b64 v, {%1, %2};\n add.rn.f32x2 %0, %0, v;\n}\n" : "+l"(sum) : "f"(a), "f"(b));
}

// Where 16 bytes of a row lie: halves of 64 values, 128-byte rows, pieces swizzled by the row.
__device__ __forceinline__ uint32_t piece_at(int row, int piece) {
  return static_cast<uint32_t>((piece >> 3) * kHalfBytes + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}
// Such rows as an operand whose inner axis runs along them (keys for the scores), and down them (values for the output).
__device__ __forceinline__ uint64_t operand(uint32_t address, uint32_t leading) {
  return static_cast<uint64_t>((address & 0x3FFFFu) >> 4) | static_cast<uint64_t>(leading) << 16 | static_cast<uint64_t>(1024 >> 4) << 32 |
         static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
__device__ __forceinline__ uint64_t operand_along(uint32_t address) { return operand(address, 1); }
__device__ __forceinline__ uint64_t operand_down(uint32_t address) { return operand(address, kHalfBytes >> 4); }

__device__ __forceinline__ __nv_bfloat162 pair_of(uint32_t bits) { return *reinterpret_cast<const __nv_bfloat162*>(&bits); }
__device__ __forceinline__ uint32_t bits_of(__nv_bfloat162 pair) { return *reinterpret_cast<const uint32_t*>(&pair); }

// Eight codes of a word (bits 4 j and 16 + 4 j) as numbers, one scale for the low ones and one for the high ones.
__device__ __forceinline__ uint4 numbers_of(uint32_t w, uint32_t scale, uint32_t offset) {
  uint32_t r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t moved = j == 0 ? w << 3 : w >> (4 * j - 3);
    const __nv_bfloat162 x = pair_of((moved & 0x00780078u) | 0x41804180u);
    r[j] = bits_of(__hfma2(x, pair_of(scale), pair_of(offset)));
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ uint32_t offset_of(uint32_t scale) { return bits_of(__hmul2(pair_of(scale), pair_of(0xC1C0C1C0u))); }   // -24 s
__device__ __forceinline__ bool not_finite(uint32_t half) { return (half & 0x7F80u) == 0x7F80u; }
// Scales near the type's largest number, whose product with 24 is none, go in as a 2^8th, and their numbers are made larger where they lie.
__device__ __forceinline__ uint32_t large(uint32_t pair) {     // bit 0: the low scale, bit 16: the high one is 2^117 and more
  const uint32_t low = pair & 0x7F80u, high = pair >> 16 & 0x7F80u;
  return (low >= 0x7A00u && low != 0x7F80u ? 1u : 0u) | (high >= 0x7A00u && high != 0x7F80u ? 0x10000u : 0u);
}

template <int D>
struct Row {
  uint4 codes[D / 32];
};
template <int D>
struct Scales {
  uint32_t pair[D / 64];     // of groups 2 i and 2 i + 1
};

template <int D>
__device__ __forceinline__ void put_keys(uint8_t* tile, int row, const Row<D>& from, const Scales<D>& scales) {
  constexpr int G = D / 32;
  uint32_t scale[G], offset[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    scale[g] = __byte_perm(scales.pair[g / 2], 0, g & 1 ? 0x3232 : 0x1010);
    offset[g] = offset_of(scale[g]);
  }
  const uint32_t* words = reinterpret_cast<const uint32_t*>(from.codes);
#pragma unroll
  for (int w = 0; w < 4 * G; ++w) {      // word t G + g: channels 32 g + 8 t and on
    const int t = w / G, g = w % G;
    *reinterpret_cast<uint4*>(tile + piece_at(row, 4 * g + t)) = numbers_of(words[w], scale[g], offset[g]);
  }
}
template <int D>
__device__ __forceinline__ void put_values(uint8_t* tile, int row, const Row<D>& from, const Scales<D>& scales) {
  constexpr int P = D / 64;
  uint32_t offset[P];
#pragma unroll
  for (int i = 0; i < P; ++i) offset[i] = offset_of(scales.pair[i]);
  const uint32_t* words = reinterpret_cast<const uint32_t*>(from.codes);
#pragma unroll
  for (int w = 0; w < D / 8; ++w)        // word r P + i: channels 4 r and on of groups 2 i (low) and 2 i + 1 (high)
    *reinterpret_cast<uint4*>(tile + piece_at(row, w)) = numbers_of(words[w], scales.pair[w % P], offset[w % P]);
}
// 2^8 times the pieces of the groups whose scales went in smaller: `which` a pair's large() for each two groups.
template <int D, bool KEYS>
__device__ __forceinline__ void enlarge(uint8_t* tile, int row, const uint32_t (&which)[D / 64]) {
#pragma unroll 1
  for (int piece = 0; piece < D / 8; ++piece) {
    const int at = KEYS ? piece >> 3 : piece % (D / 64);
    const uint32_t pair = D == 128 && at ? which[D / 64 - 1] : which[0], one = pair >> (piece >> 2 & 1 ? 16 : 0) & 1;
    const uint32_t low = KEYS ? one : pair & 1, high = KEYS ? one : pair >> 16;
    const __nv_bfloat162 factor = pair_of((low ? 0x4380u : 0x3F80u) | (high ? 0x43800000u : 0x3F800000u));
    uint4* where = reinterpret_cast<uint4*>(tile + piece_at(row, piece));
    const uint4 x = *where;
    *where = make_uint4(bits_of(__hmul2(pair_of(x.x), factor)), bits_of(__hmul2(pair_of(x.y), factor)),
                        bits_of(__hmul2(pair_of(x.z), factor)), bits_of(__hmul2(pair_of(x.w), factor)));
  }
}

// The block's rows: blocks are numbered from the back, so that the longest histories of a prompt start first.
__device__ __forceinline__ Job find_job(const PortionParams& p, int index, int group, int lane) {
  Job job{-1, 0, 0, 0, 0};
  for (int base = 0; base < p.num_entries; base += 32) {
    const int e = base + lane;
    int start = 0, count = 0, pos0 = 0;
    if (e < p.num_entries) {
      start = __ldcg(p.entry_starts + e);       // (in front of the wait: from L2, whatever this multiprocessor has read before)
      count = max(__ldcg(p.entry_starts + e + 1) - start, 0);
      pos0 = __ldcg(p.entry_pos0 + e);
    }
    if (p.skip_single && count == 1) count = 0;
    const int tiles = (count * group + p.block_rows - 1) / p.block_rows;
    int upto = tiles;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, offset);
      if (lane >= offset) upto += v;
    }
    const int mine = index - (upto - tiles);
    const uint32_t found = __ballot_sync(0xffffffffu, mine >= 0 && mine < tiles);
    if (found) {
      const int owner = __ffs(found) - 1;
      job.entry = base + owner;
      job.row0 = __shfl_sync(0xffffffffu, mine, owner) * p.block_rows;
      job.rows = min(p.block_rows, __shfl_sync(0xffffffffu, count, owner) * group - job.row0);
      job.token0 = __shfl_sync(0xffffffffu, start, owner);
      job.pos0 = __shfl_sync(0xffffffffu, pos0, owner);
      return job;
    }
    index -= __shfl_sync(0xffffffffu, upto, 31);
  }
  return job;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) attention_q4_portions_kernel(const PortionParams p) {
  constexpr int kTile = kTileRows * D * 2, kPieces = D / 8, G = D / 32;
  extern __shared__ uint8_t room[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(room) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t *q_tiles = smem, *k_tiles = smem + 2 * kTile, *v_tiles = smem + 4 * kTile;
  Shared* sh = reinterpret_cast<Shared*>(smem + 6 * kTile);
  volatile int* abort_flag = &sh->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = p.num_heads / p.num_kv_heads, kv_head = blockIdx.x, split = blockIdx.z;
  if (warp == 0) {      // the step's description may be read before the kernels ahead are done
    const Job found = find_job(p, static_cast<int>(gridDim.y) - 1 - static_cast<int>(blockIdx.y), group, lane);
    if (lane == 0) sh->job = found;
  }
  if (threadIdx.x == 32) {
    for (int i = 0; i < 2; ++i) {
      tcgen05::bar_init(&sh->q_full[i], kTileRows);
      tcgen05::bar_init(&sh->k_full[i], kUnpackThreads);
      tcgen05::bar_init(&sh->v_full[i], kUnpackThreads);
      tcgen05::bar_init(&sh->k_empty[i], 2);
      tcgen05::bar_init(&sh->v_empty[i], 2);
      for (int half = 0; half < 2; ++half) {
        tcgen05::bar_init(&sh->s_full[i][half], 1);
        tcgen05::bar_init(&sh->p_full[i][half], kTileRows);
        tcgen05::bar_init(&sh->pv_done[i][half], 1);
      }
    }
    sh->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_address(&sh->tmem)), "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tcgen05::fence_before();
  __syncthreads();
  tcgen05::fence_after();
  const uint32_t tmem = sh->tmem;
  const Job job = sh->job;
  // visible keys of the block's rows in this split: those from `begin` up to `end`
  const bool kept_split = split == p.num_splits;
  const int low_position = job.pos0 + job.row0 / group, high_position = job.pos0 + (job.row0 + job.rows - 1) / group;
  const int begin = kept_split ? 0 : max(split * p.chunk, first_visible_key(low_position, p.window));
  const int end = kept_split ? min(p.keep_first, first_visible_key(high_position, p.window))
                             : min(p.num_splits > 1 ? (split + 1) * p.chunk : 0x7fffffff, high_position + 1);
  const bool first_block = (blockIdx.x | blockIdx.y | blockIdx.z) == 0;
  if (job.entry < 0 || begin >= end) {  // no rows, or none of them sees a key here and none will be looked for
    // (a grid that found nothing to do must not end before the kernels ahead of it: one block stays for them)
    if (first_block) {
      pdl_wait();
      if (p.beside && threadIdx.x == 0) release_word(p.beside, 1);
    }
    if (warp == kIssueWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    return;
  }
  const int first_tile = begin / kKeys, num_tiles = (end + kKeys - 1) / kKeys - first_tile;
  const int steps = (end - first_tile * kKeys + 63) / 64;       // of 64 keys
  // One tile of rows only: both chains (softmax warps, scores, output, issuing warp) work at it, on every first and every second 64 keys.
  const bool pair = job.rows <= kTileRows;
  const auto steps_of = [&](int chain) { return !pair ? steps : (steps + 1 - chain) / 2; };

  if (warp < kSoftmaxWarps) {
    // ---------------- a thread a row ----------------
    const int chain = warp >> 2, tile = pair ? 0 : chain, row = threadIdx.x & (kTileRows - 1), r = tile * kTileRows + row, own_steps = steps_of(chain);
    {
      const int used = min(r, job.rows - 1);        // rows behind the last compute what nobody reads
      const int token = job.token0 + (job.row0 + used) / group, head = kv_head * group + (job.row0 + used) % group;
      const int position = job.pos0 + (job.row0 + used) / group;
      uint8_t* q_tile = q_tiles + tile * kTile;
      pdl_wait();
      // The kernel behind may start from here on: not before every block has its tensor memory (one that took it would wait for this one's end),
      // and with what went before this kernel complete, so that the step's single tokens, which share nothing with the portions, need
      // not wait for them (DecodeParams::settled in attention_q4.cu).  One thread says so, in front of its block's leave to start.
      if (!first_block || !p.beside) {
        pdl_launch_dependents();
      } else if (threadIdx.x == 0) {
        release_word(p.beside, 1);
        pdl_launch_dependents();
      }
      // a warp's 32 rows, neighbouring lanes side by side in one row, all asked for before the first is stored
      const long long row_at = (static_cast<long long>(token) * p.num_heads + head) * D;
      const int warp_row = (warp & 3) * 32, piece_of = lane % kPieces, row_of = lane / kPieces;
      if (tile == chain) {
        uint4 asked[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
          asked[i] = *reinterpret_cast<const uint4*>(p.q + __shfl_sync(0xffffffffu, row_at, i * (32 / kPieces) + row_of) + 8 * piece_of);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) *reinterpret_cast<uint4*>(q_tile + piece_at(warp_row + i * (32 / kPieces) + row_of, piece_of)) = asked[i];
        tcgen05::fence_async();
        tcgen05::bar_arrive(&sh->q_full[tile]);
      }
      // what the row sees here, and what every row of the tile sees
      const int tile_last = min(tile * kTileRows + kTileRows, job.rows) - 1;
      const int tile_low_position = job.pos0 + (job.row0 + tile * kTileRows) / group, tile_high_position = job.pos0 + (job.row0 + tile_last) / group;
      int row_first = first_visible_key(position, p.window), row_last = position;
      int all_first = first_visible_key(tile_high_position, p.window), all_last = tile_low_position;
      if (kept_split) {
        row_last = min(p.keep_first, row_first) - 1;
        all_last = min(p.keep_first, first_visible_key(tile_low_position, p.window)) - 1;
        row_first = all_first = 0;
      }
      const float scale_log2 = p.scale * kLog2e;
      const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
      const uint32_t s_at = lanes + chain * 128, o_at = lanes + 256 + chain * 128;
      float row_max = -INFINITY, row_sum = 0.0f;
      uint32_t bad_groups = 0;
      for (int n = 0; n < own_steps; ++n) {
        const int i = pair ? 2 * n + chain : n, half = i & 1, key0 = first_tile * kKeys + 64 * i, buffer = n & 1;
        const uint32_t scores_at = s_at + 64 * buffer;
        const bool edge = key0 < all_first || key0 + 63 > all_last;
        wait(&sh->s_full[chain][buffer], (n >> 1) & 1, abort_flag, p.status);
        tcgen05::fence_after();
        uint32_t s[64];
        tensor_load_32(scores_at, s);
        tensor_load_32(scores_at + 32, s + 32);
        const uint2 bad = reinterpret_cast<const uint2*>(&sh->bad_any[(i >> 1) & 3])[half];
        if (bad.x | bad.y) {       // values that are not finite: do this row's keys include theirs?
#pragma unroll
          for (int w = 0; w < 2; ++w)
            for (uint32_t left = w ? bad.y : bad.x; left; left &= left - 1) {
              const int k = __ffs(left) - 1, key = key0 + 32 * w + k;
              if (key < row_first || key > row_last) continue;
              for (int g = 0; g < G; ++g) bad_groups |= (sh->bad[(i >> 1) & 3][g][2 * half + w] >> k & 1u) << g;
            }
        }
        tensor_load_wait();
        if (edge) {
#pragma unroll
          for (int k = 0; k < 64; ++k)
            if (key0 + k < row_first || key0 + k > row_last) s[k] = __float_as_uint(-INFINITY);
        }
        float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < 64; k += 2) m[(k >> 1) & 3] = fmaxf(m[(k >> 1) & 3], fmaxf(__uint_as_float(s[k]), __uint_as_float(s[k + 1])));
        const float step_max = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * scale_log2;
        float new_max = row_max;
        if (step_max > row_max + kMaxSlack || row_max == -INFINITY) new_max = fmaxf(row_max, step_max);
        const float shrink = new_max == row_max ? 1.0f : exp2_of(row_max - new_max);
        row_max = new_max;
        row_sum *= shrink;
        if (n > 0 && __any_sync(0xffffffffu, shrink != 1.0f)) {
          wait(&sh->pv_done[chain][buffer ^ 1], ((n - 1) >> 1) & 1, abort_flag, p.status);
          tcgen05::fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tensor_load_16(o_at + c, o);
            tensor_load_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * shrink);
            tensor_store_16(o_at + c, o);
          }
        }
        const float shift = row_max == -INFINITY ? 0.0f : row_max;
        const unsigned long long scale_pair = both(scale_log2), shift_pair = both(-shift);
        unsigned long long sum[2] = {0ull, 0ull};
        uint32_t weights[32];
#pragma unroll
        for (int k = 0; k < 64; k += 2) {
          float a, b;
          scaled_pair(a, b, s[k], s[k + 1], scale_pair, shift_pair);
          a = exp2_of(a);
          b = exp2_of(b);
          add_pair(sum[(k >> 1) & 1], a, b);
          weights[k >> 1] = bits_of(__floats2bfloat162_rn(a, b));
        }
        tensor_store_32(scores_at, weights);
        row_sum += sum_of_pair(sum[0]) + sum_of_pair(sum[1]);
        tensor_store_wait();
        tcgen05::fence_before();
        tcgen05::bar_arrive(&sh->p_full[chain][buffer]);
      }
      if (own_steps > 0) wait(&sh->pv_done[chain][(own_steps - 1) & 1], ((own_steps - 1) >> 1) & 1, abort_flag, p.status);
      tcgen05::fence_after();
      // A pair's chains join: each has the rows' other half of the keys, and writes half of the columns.
      float factor = own_steps > 0 ? 1.0f : 0.0f, other_factor = 0.0f;
      const bool other_too = pair && steps_of(chain ^ 1) > 0;
      const auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory"); };
      if (pair) {
        sh->told[chain][row] = make_float4(row_max, row_sum, __uint_as_float(bad_groups), 0.0f);
        tcgen05::fence_before();
        meet();
        tcgen05::fence_after();
        const float4 other = sh->told[chain ^ 1][row];
        const float best = fmaxf(row_max, other.x);
        factor = row_max == -INFINITY ? 0.0f : exp2_of(row_max - best);
        other_factor = other.x == -INFINITY ? 0.0f : exp2_of(other.x - best);
        row_sum = (own_steps > 0 ? row_sum * factor : 0.0f) + (other_too ? other.y * other_factor : 0.0f);
        row_max = best;
        bad_groups |= __float_as_uint(other.z);
      }
      const bool whole = p.partial_ml == nullptr;
      const size_t place = (static_cast<size_t>(token) * p.num_heads + head) * (p.num_splits + (p.keep_first > 0 ? 1 : 0)) + split;
      if (whole) {
        if (p.sink) row_sum += exp2f((p.sink_values ? p.sink_values[head] * kLog2e : 0.0f) - row_max);
        float inverse = 1.0f / row_sum;
        if (p.gate && p.gate_per_head) inverse *= 1.0f / (1.0f + __expf(-p.gate[static_cast<size_t>(token) * p.gate_stride + head]));
        factor *= inverse;
        other_factor *= inverse;
      } else if (r < job.rows && tile == chain && !*abort_flag) {
        // (the joining kernel passes over -inf, which stands for no visible key and not for keys whose scores are all NaN)
        *reinterpret_cast<float2*>(p.partial_ml + 2 * place) = make_float2(row_max == -INFINITY && row_sum != row_sum ? 0.0f : row_max, row_sum);
      }
      const float* gate = p.gate && !p.gate_per_head ? p.gate + static_cast<size_t>(token) * p.gate_stride + static_cast<size_t>(head) * D : nullptr;
      const uint32_t other_at = lanes + 256 + (chain ^ 1) * 128;
#pragma unroll 1
      for (int a = pair ? chain * (D / 64) : 0; a < (pair ? (chain + 1) * (D / 64) : D / 32); ++a) {
        uint32_t o[32];
        if (own_steps > 0) tensor_load_32(o_at + 32 * a, o);
        tensor_load_wait();
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = own_steps > 0 ? __float_as_uint(__uint_as_float(o[k]) * factor) : 0u;
        if (other_too) {
          uint32_t more[32];
          tensor_load_32(other_at + 32 * a, more);
          tensor_load_wait();
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(fmaf(__uint_as_float(more[k]), other_factor, __uint_as_float(o[k])));
        }
#pragma unroll
        for (int part = 0; part < 4; ++part) {     // eight neighbouring channels
          const int g = D == 128 ? part : part >> 1, piece = D == 128 ? 4 * part + a : 4 * (part >> 1) + 2 * a + (part & 1);
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int word = D == 128 ? 2 * (i / 4) + g / 2 : 2 * (part & 1) + i / 4;
            x[i] = __uint_as_float(o[8 * word + 2 * (i & 3) + (g & 1)]);
            if (bad_groups >> g & 1) x[i] = __int_as_float(0x7fffffff);
          }
          if (whole) {
            if (gate) {
#pragma unroll
              for (int i = 0; i < 8; ++i) x[i] *= 1.0f / (1.0f + __expf(-gate[8 * piece + i]));
            }
            uint32_t packed[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) packed[i] = bits_of(__floats2bfloat162_rn(x[2 * i], x[2 * i + 1]));
            // through the tile of queries, whose products are done: a warp's stores then cover whole rows
            *reinterpret_cast<uint4*>(q_tile + piece_at(row, piece)) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
          } else if (r < job.rows && !*abort_flag) {
            float4* to = reinterpret_cast<float4*>(p.partial_out + place * D + 8 * piece);
            to[0] = make_float4(x[0], x[1], x[2], x[3]);
            to[1] = make_float4(x[4], x[5], x[6], x[7]);
          }
        }
      }
      if (whole) {
        if (pair) meet();
        else __syncwarp();
        const bool failed = *abort_flag;
        uint4 done[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
          if (!pair || i / (kPieces / 2) == chain) done[i] = *reinterpret_cast<const uint4*>(q_tile + piece_at(warp_row + i * (32 / kPieces) + row_of, piece_of));
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int from = i * (32 / kPieces) + row_of;
          const long long at = __shfl_sync(0xffffffffu, row_at, from);
          if ((!pair || i / (kPieces / 2) == chain) && tile * kTileRows + warp_row + from < job.rows && !failed)
            *reinterpret_cast<uint4*>(p.out + at + 8 * piece_of) = done[i];
        }
      }
    }
    tcgen05::fence_before();
  } else if (warp < kUnpackWarp + kUnpackThreads / 32) {
    // ---------------- keys and values, a thread a row ----------------
    const int row = threadIdx.x - 32 * kUnpackWarp;
    const int* table = p.block_table + static_cast<size_t>(job.entry) * p.table_width;
    const int shift = (p.page_size & (p.page_size - 1)) == 0 ? 31 - __clz(p.page_size) : -1;
    auto page_of = [&](int j, bool waited = true) {
      const int key = (first_tile + j) * kKeys + row;
      if (j >= num_tiles || key < begin || key >= end) return -1;
      const int index = shift >= 0 ? key >> shift : key / p.page_size;
      const int page = index < p.table_width ? (waited ? table[index] : __ldcg(table + index)) : -1;
      return page < p.num_pages ? page : -1;
    };
    auto row_of = [&](int j, int page) {
      const int key = (first_tile + j) * kKeys + row;
      const int place = shift >= 0 ? key & (p.page_size - 1) : key % p.page_size;
      return (static_cast<size_t>(page) * p.num_kv_heads + kv_head) * p.page_size + place;
    };
    auto codes = [&](Row<D>& to, const uint8_t* pool, size_t at, bool held) {
      const uint4* from = reinterpret_cast<const uint4*>(pool + at * (D / 2));
#pragma unroll
      for (int i = 0; i < D / 32; ++i) to.codes[i] = held ? from[i] : make_uint4(0, 0, 0, 0);
    };
    auto scales = [&](Scales<D>& to, const __nv_bfloat16* pool, size_t at, bool held) {
      const uint32_t* from = reinterpret_cast<const uint32_t*>(pool + at * G);
#pragma unroll
      for (int i = 0; i < D / 64; ++i) to.pair[i] = held ? from[i] : 0u;
    };
    // a tile's keys are asked for when the last one's are unpacked, its values behind the last one's, its pages a tile before
    Row<D> keys, values;
    Scales<D> key_scales, value_scales, next_value_scales;
    int page = page_of(0, false);
    pdl_wait();
    size_t at = page >= 0 ? row_of(0, page) : 0;
    codes(keys, p.k_codes, at, page >= 0);
    scales(key_scales, p.k_scales, at, page >= 0);
    scales(value_scales, p.v_scales, at, page >= 0);
    codes(values, p.v_codes, at, page >= 0);
    page = page_of(1);
    for (int j = 0; j < num_tiles; ++j) {
      const int stage = j & 1;
      const uint32_t before = ((j >> 1) - 1) & 1;
      uint8_t *k_tile = k_tiles + stage * kTile, *v_tile = v_tiles + stage * kTile;
      uint32_t large_keys[D / 64], large_values[D / 64], any_large = 0;
      bool any_bad = false;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        any_bad = any_bad || not_finite(value_scales.pair[i]) || not_finite(value_scales.pair[i] >> 16);
        large_keys[i] = large(key_scales.pair[i]);
        large_values[i] = large(value_scales.pair[i]);
        any_large |= large_keys[i] | large_values[i];
      }
      if (j >= 2) wait(&sh->k_empty[stage], before, abort_flag, p.status);
      // the notes of tile j - 4 have been read: its softmax came before the scores of tile j - 2, and their keys are gone
      const uint32_t bad = __ballot_sync(0xffffffffu, any_bad);
      if (bad) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint32_t pair = value_scales.pair[g / 2];
          const bool mine = not_finite(g & 1 ? pair >> 16 : pair);
          const uint32_t keys_of = __ballot_sync(0xffffffffu, mine);
          if (lane == 0) sh->bad[j & 3][g][row >> 5] = keys_of;
          if (mine) value_scales.pair[g / 2] &= g & 1 ? 0x0000FFFFu : 0xFFFF0000u;
        }
      }
      if (lane == 0) reinterpret_cast<uint32_t*>(&sh->bad_any[j & 3])[row >> 5] = bad;
      if (any_large) {
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          key_scales.pair[i] -= large_keys[i] << 10;
          value_scales.pair[i] -= large_values[i] << 10;
        }
      }
      put_keys<D>(k_tile, row, keys, key_scales);
      if (any_large) enlarge<D, true>(k_tile, row, large_keys);
      tcgen05::fence_async();
      tcgen05::bar_arrive(&sh->k_full[stage]);
      at = page >= 0 ? row_of(j + 1, page) : 0;
      codes(keys, p.k_codes, at, page >= 0);
      scales(key_scales, p.k_scales, at, page >= 0);
      scales(next_value_scales, p.v_scales, at, page >= 0);
      if (j >= 2) wait(&sh->v_empty[stage], before, abort_flag, p.status);
      put_values<D>(v_tile, row, values, value_scales);
      if (any_large) enlarge<D, false>(v_tile, row, large_values);
      tcgen05::fence_async();
      tcgen05::bar_arrive(&sh->v_full[stage]);
      codes(values, p.v_codes, at, page >= 0);
      value_scales = next_value_scales;
      page = page_of(j + 2);
    }
  } else if (warp < kIssueWarp + 2) {
    // ---------------- products of one chain ----------------
    const int chain = warp - kIssueWarp, tile = pair ? 0 : chain, own_steps = steps_of(chain);
    constexpr uint32_t kTypes = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(kTileRows >> 4) << 24);
    constexpr uint32_t kScores = kTypes | (static_cast<uint32_t>(64 >> 3) << 17);
    constexpr uint32_t kOutput = kTypes | (static_cast<uint32_t>(D >> 3) << 17) | (1u << 16);      // the right operand's inner axis runs down its rows
    if (own_steps > 0) {
      const uint32_t q_at = shared_address(q_tiles + tile * kTile), s_at = tmem + chain * 128, o_at = tmem + 256 + chain * 128;
      wait(&sh->q_full[tile], 0, abort_flag, p.status);
      auto scores = [&](int n) {
        const int i = pair ? 2 * n + chain : n, j = i >> 1, half = i & 1, stage = j & 1, buffer = n & 1;
        const uint32_t k_at = shared_address(k_tiles + stage * kTile) + half * 64 * 128;
        if (pair || half == 0) wait(&sh->k_full[stage], (j >> 1) & 1, abort_flag, p.status);
        if (n >= 2) wait(&sh->pv_done[chain][buffer], ((n >> 1) - 1) & 1, abort_flag, p.status);     // the weights lie where these scores go
        tcgen05::fence_after();
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t offset = static_cast<uint32_t>((ks >> 2) * kHalfBytes + (ks & 3) * 32);
          tcgen05::mma_shared(s_at + 64 * buffer, operand_along(q_at + offset), operand_along(k_at + offset), kScores, ks > 0 ? 1u : 0u);
        }
        tcgen05::commit(&sh->s_full[chain][buffer]);
        if (pair || half == 1 || i == steps - 1) tcgen05::commit(&sh->k_empty[stage]);
      };
      scores(0);
      if (own_steps > 1) scores(1);
      for (int n = 0; n < own_steps; ++n) {
        const int i = pair ? 2 * n + chain : n, j = i >> 1, half = i & 1, stage = j & 1, buffer = n & 1;
        const uint32_t v_at = shared_address(v_tiles + stage * kTile) + half * 64 * 128;
        if (pair || half == 0) wait(&sh->v_full[stage], (j >> 1) & 1, abort_flag, p.status);
        wait(&sh->p_full[chain][buffer], (n >> 1) & 1, abort_flag, p.status);
        tcgen05::fence_after();
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          mma_tensor(o_at, s_at + 64 * buffer + ks * 8, operand_down(v_at + ks * 2048), kOutput, (n > 0 || ks > 0) ? 1u : 0u);
        tcgen05::commit(&sh->pv_done[chain][buffer]);
        if (pair || half == 1 || i == steps - 1) tcgen05::commit(&sh->v_empty[stage]);
        if (n + 2 < own_steps) scores(n + 2);
      }
    }
    tcgen05::fence_before();
  }
  __syncthreads();
  if (warp == kIssueWarp) {
    tcgen05::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

template <int D>
int launch(const PortionParams& p, cudaStream_t s) {
  // heads of 64 ask for as much as those of 128: a block holds all of its SM's tensor memory, so nothing else that wants some should join it
  constexpr int kSmem = 6 * kTileRows * 128 * 2 + 1024 + static_cast<int>(sizeof(Shared));
  static_assert(kSmem <= 227 * 1024, "a block's shared memory");
  static SharedMemoryOptIn opt_in;
  const int refused = opt_in.ask(reinterpret_cast<const void*>(attention_q4_portions_kernel<D>), kSmem);
  if (refused) return refused;
  const long long tiles = (static_cast<long long>(p.num_tokens) * (p.num_heads / p.num_kv_heads) + p.block_rows - 1) / p.block_rows + p.num_entries;
  const int places = p.num_splits + (p.keep_first > 0 ? 1 : 0);
  if (tiles > 65535) return VIPERA_BAD_SHAPE;
  return vipera_launch(attention_q4_portions_kernel<D>, dim3(p.num_kv_heads, static_cast<unsigned>(tiles), places), kThreads, kSmem, s, p);
}

bool on_16_bytes(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

VIPERA_API int vipera_attention_q4_portions_params_size() { return static_cast<int>(sizeof(PortionParams)); }

// Attention of every token of a step (with skip_single: of the entries that bring more than one).  p->num_splits > 1, or kept first keys:
// parts go to `scratch` and a second kernel joins them (`positions` [tokens]); tokens that were left out then get rows without meaning, for
// the kernel of single tokens to write behind it.
// `status` is 0 before the launch, and not 0 after it if a bounded wait ran out.
VIPERA_API int vipera_attention_q4_portions(const PortionParams* given, const int* positions, float* scratch, size_t scratch_floats, void* stream) {
  PortionParams p = *given;
  if (p.num_entries <= 0 || p.num_tokens <= 0) return VIPERA_OK;
  if (p.num_heads <= 0 || p.num_kv_heads <= 0 || p.num_heads % p.num_kv_heads || p.num_kv_heads > 65535 || p.num_heads > 65535 || p.keep_first < 0 ||
      p.page_size <= 0 || p.page_size % 16 || p.num_splits <= 0 || p.num_splits > 128 || p.chunk <= 0 || p.chunk % kKeys ||
      (p.head_dim != 64 && p.head_dim != 128) ||
      static_cast<long long>(p.num_tokens) * (p.num_heads / p.num_kv_heads) > 0x7fffffffLL - 2 * kTileRows || (p.block_rows != kTileRows && p.block_rows != 2 * kTileRows))
    return VIPERA_BAD_SHAPE;
  if (p.window <= 0) p.keep_first = 0;
  if (p.sink_values) p.sink = 1;
  if (!p.status || !on_16_bytes(p.q) || !on_16_bytes(p.out) || !on_16_bytes(p.k_codes) || !on_16_bytes(p.v_codes) || !on_16_bytes(p.k_scales) ||
      !on_16_bytes(p.v_scales))
    return VIPERA_BAD_ARGUMENT;
  const int places = p.num_splits + (p.keep_first > 0 ? 1 : 0);
  p.partial_ml = p.partial_out = nullptr;
  if (places > 1) {
    const size_t rows = static_cast<size_t>(p.num_tokens) * p.num_heads * places, pairs = (2 * rows + 3) / 4 * 4;
    if (!positions || !scratch || scratch_floats < pairs + rows * p.head_dim || !on_16_bytes(scratch)) return VIPERA_BAD_ARGUMENT;
    p.partial_ml = scratch;
    p.partial_out = scratch + pairs;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int status = p.head_dim == 128 ? launch<128>(p, s) : launch<64>(p, s);
  if (status != VIPERA_OK || places == 1) return status;
  const JoinParams join{p.partial_ml, p.partial_out, p.out, positions, p.entry_starts + p.num_entries, p.sink_values, p.gate, p.gate_stride,
                        p.gate_per_head, p.sink, p.num_tokens, p.num_heads, p.window, p.keep_first, p.chunk, p.num_splits};
  return p.head_dim == 128 ? launch_join<128, __nv_bfloat16>(join, s) : launch_join<64, __nv_bfloat16>(join, s);
}
