// rt_shared.h — launch-shape constants that the kernels and the host runtime
// must agree on.  Plain C++ (no HIP types): included by the device sources
// and by runtime.cpp, so a grid and the kernel it launches cannot disagree.
#pragma once
#include <stdint.h>

// Decode attention: query heads per workgroup at a head size.  Head sizes 64
// and 128 take 1: a group of 7 query heads spreads over 7 workgroups per KV
// head and split, each thread's score chain one head long (0.5B step: 690 →
// 667 µs, 7B step: 1889 → 1846 µs against 8 and 4 heads per workgroup);
// head size 256 takes 8.
constexpr uint32_t rt_attn_gm(uint32_t head_dim) { return head_dim == 256 ? 8u : 1u; }
// Head groups of 256 threads per workgroup: one (groups share the query heads
// of their workgroup, so one head leaves one group; head size 256 is bound to
// one by its registers).
constexpr uint32_t rt_attn_hg(uint32_t) { return 1u; }
// The persistent step's attention phase runs RT_STEP_THREADS / 256 = 2 head
// groups, so its workgroups take 2 query heads (step 772 → 753 µs against 8).
constexpr uint32_t rt_step_attn_gm(uint32_t) { return 2u; }
// Multi-query (verify / prefill) attention on the matrix cores: the most
// waves a workgroup of 16 query columns may have at a head size.
constexpr uint32_t rt_attn_mq_wmax(uint32_t head_dim) { return head_dim == 256 ? 4u : 8u; }
// Key ranges of one column group merged by its last workgroup (at most).
constexpr uint32_t RT_ATTN_MQ_NSP_MAX = 8;
// LDS bytes of such a workgroup of w waves: per wave 16 columns × head_dim
// outputs + 16 maxima + 16 sums.
constexpr uint32_t rt_attn_mq_lds(uint32_t head_dim, uint32_t w) { return w * (16u * head_dim + 32u) * 4u; }

// Device scratch of the no-allocation entry points: one fixed array in the
// code object (k_scratch.hip), laid out as [arrival counters | activation
// workspace | K-split partial sums].
constexpr uint64_t RT_SCRATCH_BYTES = 4ull << 20;
constexpr uint64_t RT_SCRATCH_COUNTER_BYTES = 56ull << 10;  // as the context's counter area
constexpr uint64_t RT_SCRATCH_WS_OFF = 64ull << 10;
constexpr uint64_t RT_SCRATCH_WS_BYTES = 1ull << 20;
constexpr uint64_t RT_SCRATCH_PART_OFF = RT_SCRATCH_WS_OFF + RT_SCRATCH_WS_BYTES;
constexpr uint64_t RT_SCRATCH_PART_BYTES = RT_SCRATCH_BYTES - RT_SCRATCH_PART_OFF;

// Persistent decode step (k_step.hip): phase record size and the most
// workgroups a step grid may have.
constexpr uint32_t RT_STEP_PHASE_BYTES = 400;
constexpr uint32_t RT_STEP_MAX_WGS = 1024;
// threads per workgroup of the persistent step (its attention phase runs
// RT_STEP_THREADS / 256 head groups)
#define RT_STEP_THREADS 512
constexpr uint32_t RT_STEP_SYNC_BYTES = 2048;  // StepSync (k_step.hip)
constexpr uint32_t RT_STEP_STATUS_OFF = 1280;  // its status word

// Attention over paged caches (k_paged.hip): the columns of a narrow block, the
// positions of a tile (page sizes are multiples of it), the waves of a workgroup.
constexpr uint32_t RT_PAGED_ROWS = 16;
constexpr uint32_t RT_PAGED_TILE = 16;
constexpr uint32_t RT_PAGED_WAVES = 4;
constexpr uint32_t RT_PAGED_WIDE_ROWS = 128;  // columns of a wide block, 32 a wave

// One batch over a paged cache, as rt_paged_batch describes it.
struct PagedBatch {
    void* k;                    // page p at p·page_stride elements (4 bits: bytes): [KVH][page size][head size]
    void* v;
    const uint32_t* table;      // [n_seqs][table_stride] page ids
    const uint32_t* row_start;  // [n_seqs + 1], or null: one row a sequence
    const uint32_t* kv_len;     // [n_seqs]
    uint64_t page_stride;
    uint32_t num_pages, ps_shift, table_stride, n_seqs, rows, KVH;
};
struct PagedAppendArgs {
    PagedBatch b;
    const float* q;  // [rows][H][head size]
    const float* k;  // [rows][KVH][head size]
    const float* v;
    float* q_out;
    double log2_theta;
    uint32_t H;
};
struct PagedGatherArgs {
    PagedBatch b;
    void* k_out;  // [rows][KVH][head size], or null
    void* v_out;
    uint32_t head_dim;
};
// Pages copied (k_paged.hip), at most: pages of a call; of a launch, as every workgroup looks through
// its list (4,000 pages of 1 KB in 48 pools: 1,024 a launch 258 µs, 2,048 323, 4,000 443; 512 271);
// bytes of a workgroup; pools of a launch (2 KB of its arguments).
constexpr uint32_t RT_COPY_MAX = 65535;
constexpr uint32_t RT_COPY_LIST = 1024;
constexpr uint32_t RT_COPY_SLICE = 16384;
constexpr uint32_t RT_COPY_POOLS = 256;
struct PagedCopyArgs {
    const uint32_t *src, *dst;
    uint64_t page_stride;  // bytes
    uint32_t page_bytes, slice_bytes, slices, num_pages, n;
    uint32_t n_pools, group;  // small pages: pools, and those of a workgroup
    void* pools[RT_COPY_POOLS];
};
struct PagedAttnArgs {
    PagedBatch b;
    const float* q;  // [rows][H][head size]
    float* out;
    const uint32_t* shared_table;  // positions below shared_len are read through it
    float* part;     // [jobs][KVH][rows of a slot][head size] unnormalised outputs
    float* ml;       // [jobs][KVH][rows of a slot][max, sum]
    // where chunks meet in a launch of their own (wide blocks, a shared prefix):
    // [rows][H][own, prefix][first job, chunks · rows of a slot + row in its block]
    uint32_t* info;
    uint32_t* counters;  // else: [jobs][KVH][2] arrivals at the block's and the group's first job, 0 between launches
    uint32_t H, shared_len;
    uint32_t jobs;    // jobs of a KV head (at most)
    uint32_t target;  // its chunks beyond one a block (at most; 0: blocks are not split)
    uint32_t slots;      // workgroups of a KV head that are resident together, ≤ jobs
    uint32_t min_chunk;  // tiles of a chunk (at least)
    uint32_t noted;      // chunks meet in a launch of their own (pages of 4 bits)
    float scale;
};

// Rules on logits (k_rules.hip).
constexpr uint32_t RT_RULES_SEG = 4096;     // tokens of a workgroup
constexpr uint32_t RT_RULES_THREADS = 512;  // its threads
struct RulesArgs {
    const void* x;  // [rows][row_stride]
    void* out;
    uint64_t row_stride;
    uint32_t n, rows, segs, inplace;
    float inv_more;  // 1 / (segs − 1)
    // lists: row r's is at start[r], len[r] long, cut to the n_* that are there
    const uint32_t *tokens, *token_start, *token_len, *prompt_len;
    uint64_t n_tokens, n_bias;
    const float *repetition, *frequency, *presence;
    const uint32_t *bias_ids, *bias_start, *bias_len;
    const float* bias;
    const uint32_t *mask, *mask_row;
    uint64_t mask_stride;
    uint32_t mask_rows;
};

// Token log probabilities (k_logprobs.hip).
constexpr uint32_t RT_LOGPROBS_TOP_MAX = 64;   // alternatives (at most): one a lane
constexpr uint32_t RT_LOGPROBS_SEG_MAX = 64;   // segments of a row (at most): one a lane where they meet
struct LogprobsArgs {
    const void* x;  // [rows][row_stride]
    const uint32_t* tokens;
    float* logprob;
    float* entropy;   // or null
    uint32_t* rank;   // or null
    uint32_t* top_ids;
    float* top_logprobs;
    uint64_t* part;      // segs > 1: [rows][segs][2]: max and Σe, Σe·(x − max) / ln 2 and rank
    uint64_t* keys;      //           [rows][segs][top]: the largest, in order
    uint32_t* counters;  //           [rows] arrivals, 0 between launches
    uint64_t row_stride;
    uint32_t n, top, segs, seg_len;
};
