// A paged key / value cache held in 4 bits: its layout, and what a step of several sequences works on.
//
// Blocks of 32 values along a head: minimum m and step d in half precision, a code of 4 bits a value, value = m + d * code; with the
// scales that is 5 bits a value. m = half(min), d = half(max(max - m, 0) / 15), code = (x - m) / d to the nearest whole number (ties to even) in 0..15,
// all of it as if in exact arithmetic. m and d stop at 65504; a block that holds an infinity or a NaN has d = 0 and m = NaN.
//
// A page holds page_tokens (a multiple of 16) positions of every key / value head: [page][kv head][tile of 16 positions], so one tile of
// one head is one contiguous piece of memory:
//   16 rows of key codes | 16 rows of value codes | 16 rows of key scales | 16 rows of value scales
// A row of codes has dim / 2 bytes, a row of scales the d of all blocks, then their m. The order within is the one in which the lanes of a
// warp hold the operands of m16n8k16 products, lane = 4 * g + t, so that a lane's share of a row is one load:
//   keys    row kv4_row(T) for position T of the tile; the 8 codes of dims 32 b + 8 t .. + 7 are word t * NB + b (NB = dim / 32; of 256
//           dims each half of the row by itself). Nibble i of a word is dim 8 t + i.
//   values  row T; the 4 codes of dims 32 b + 4 g .. + 3 are half-word g * NB + b
//   scales  of both in row kv4_row(T)
// kv4_row puts positions t, t + 4, t + 8, t + 12 where a lane's column pair of the second product's operand meets them.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace alice {

constexpr uint32_t KV4_BLOCK = 32, KV4_TILE = 16;
constexpr uint32_t KV4_PROMPT_ROWS = 128;      // of a job of csrc/kv4_prompt.cu

__host__ __device__ constexpr uint32_t kv4_tile_bytes(uint32_t dim) { return 20 * dim; }
__host__ __device__ constexpr uint32_t kv4_v_codes(uint32_t dim) { return 8 * dim; }
__host__ __device__ constexpr uint32_t kv4_k_scales(uint32_t dim) { return 16 * dim; }
__host__ __device__ constexpr uint32_t kv4_v_scales(uint32_t dim) { return 18 * dim; }
__host__ __device__ constexpr uint32_t kv4_row(uint32_t pos) { return (pos & 8u) | ((pos & 3u) << 1) | ((pos >> 2) & 1u); }
// place of a key word: 8 dims at 32 b + 8 t
__host__ __device__ constexpr uint32_t kv4_k_word(uint32_t nb, uint32_t b, uint32_t t) { return nb == 8 ? (b >> 2) * 16 + t * 4 + (b & 3) : t * nb + b; }

struct Kv4Shape {
    uint32_t pages, page_tokens, kv_heads, dim;
    __host__ __device__ uint32_t tiles() const { return page_tokens / KV4_TILE; }
    __host__ size_t bytes() const { return (size_t)pages * kv_heads * tiles() * kv4_tile_bytes(dim); }
};

// Written by alice_kv4_batch_set (or by a model's step, on the device) and read by the kernels when they run, so that a captured call
// works on what is there at its replay.
struct Kv4Head {
    uint32_t seqs, tokens, jobs, rows;   // rows: (token, query head) rows of a job
    uint32_t tiles;                      // of all jobs of one key / value head
    uint32_t end, top_page;              // positions of the longest sequence, highest page of a table
    uint32_t prompt_jobs;                // ahead of the others, of sequences with many rows
};

// A job: up to `rows` of Kv4Head consecutive (token, query head of the group) rows of a sequence, against the keys the last of them sees.
struct alignas(32) Kv4Job {
    uint32_t seq, row, rows;     // its first row, and how many it has
    uint32_t first, past;        // of the sequence: row of its first token in q, k, v; positions before it
    uint32_t tile0, tile1;       // of the tiles of all jobs of a key / value head
    uint32_t unused;
};
struct alignas(16) Kv4Token {
    uint32_t tile;               // of its page's first head, counted through the pool
    uint32_t row;                // in the tile
    uint32_t pos;                // position: row of the rotation table
    uint32_t unused;
};
struct Kv4Plan {
    const Kv4Head* head;
    const Kv4Token* token;       // [tokens]
    const Kv4Job* job;           // [prompt_jobs], [jobs]
    const uint32_t* job_tile;    // [jobs] tile0 of the latter by themselves
    const uint32_t* table;       // [seqs][table_ld] pages
    uint32_t table_ld;
};

struct Kv4Rope {
    const float* table;          // [row][dims / 2] (sin, cos), or null
    uint32_t dims;               // the first dims of a head are rotated
    uint32_t neox;               // 0: pairs (2 i, 2 i + 1), 1: pairs (i, i + dims / 2)
    uint32_t by_token;           // rows are those of the batch's tokens, not positions
    uint32_t rows;               // of the table
};

struct Kv4RowsArgs {             // append: k, v read; read: k, v written
    Kv4Plan plan;
    Kv4Shape shape;
    uint8_t* pool;
    float *k, *v;
    size_t k_ld, v_ld;           // floats from token to token
    uint32_t most_tokens;        // that k and v have room for
    uint32_t heads;              // key / value heads a warp takes (the launcher's)
    Kv4Rope rope;
    int* status;
};

struct Kv4AttnArgs {
    Kv4Plan plan;
    Kv4Shape shape;
    const uint8_t* pool;
    const float* q;
    float* out;
    size_t q_ld, out_ld;
    uint32_t most_tokens;
    uint32_t group;              // query heads a key / value head
    uint32_t rows, prompt_jobs;  // of what is launched: rows of a job, 0: only prompts; prompt jobs at most
    uint32_t end;                // positions of the longest sequence, as far as the host knows
    float scale;
    Kv4Rope rope;
    float* part;                 // scratch of the joins, kv4_part_floats
    unsigned int* tickets;       // [CTAs], zero between launches
    int* status;
};

// A captured call meets what the batch is at its replay: whether that stays within the buffers, tables and pages of the call.
__device__ __forceinline__ bool kv4_fits(const Kv4Head& h, uint32_t most_tokens, const Kv4Rope& rope, const Kv4Shape& shape, int* status, bool launched = true) {
    const bool ok = launched && h.tokens <= most_tokens && (!rope.table || (rope.by_token ? h.tokens : h.end) <= rope.rows) && (!h.tokens || h.top_page < shape.pages);
    if (!ok && threadIdx.x == 0) atomicCAS(status, 0, KERR_KV4_BATCH);
    return ok;
}

__device__ __forceinline__ bool kv4_fits(const Kv4Head& h, const Kv4AttnArgs& a) {
    return kv4_fits(h, a.most_tokens, a.rope, a.shape, a.status, (!h.jobs || h.rows == a.rows) && h.prompt_jobs <= a.prompt_jobs);
}

// Whether a sequence's (token, query head) rows are jobs of csrc/kv4_prompt.cu: from where its 128 rows a job, mostly empty, are faster than jobs of 16. Measured
// either way, us (32 x 8 heads of 128): 16 rows behind 4000 positions 21 against 19, 20 rows 21 / 30, 20 rows behind 100 11 / 17, 32 sequences of 20 rows behind 2000
// 94 / 104, of 64 rows 97 / 184; heads of 64: 32 sequences of 24 rows behind 2000 37 / 38, 64 of 32 rows behind 100 33 / 25, 16 of 64 rows behind 2000 40 / 109.
inline bool kv4_is_prompt(uint32_t rows, uint32_t dim) { return dim == 128 ? rows > 16 : dim == 64 && rows > 32; }
// Rows a job may have else, by the most rows a sequence has: 4, 8 or 16 (8 of 256 dims, whose operands would not fit the registers).
inline uint32_t kv4_job_rows(uint32_t most, uint32_t dim) { return most <= 4 ? 4 : most <= 8 || dim == 256 ? 8 : 16; }
// Writes `plan` for one sequence's n tokens from position *pos on (or pos0, where pos is null), its pages in order. A single CTA.
cudaError_t launch_kv4_plan(const Kv4Plan& plan, const Kv4Shape& shape, uint32_t group, uint32_t n, const int* pos, uint32_t pos0, cudaStream_t st, bool pdl);
size_t kv4_part_floats(uint32_t dim, int num_sms);
// `tokens`, `jobs`: how many the host knows of; the kernels take the numbers of plan.head and stride over them.
cudaError_t launch_kv4_append(const Kv4RowsArgs& a, uint32_t tokens, int num_sms, cudaStream_t st, bool pdl);
cudaError_t launch_kv4_read(const Kv4RowsArgs& a, uint32_t tokens, int num_sms, cudaStream_t st, bool pdl);
cudaError_t launch_kv4_attention(const Kv4AttnArgs& a, int num_sms, cudaStream_t st, bool pdl);
cudaError_t launch_kv4_prompt(const Kv4AttnArgs& a, cudaStream_t st, bool pdl);

}  // namespace alice
