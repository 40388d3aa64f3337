// Host side of a step over the 4-bit cache: its checks and the jobs it is cut into (csrc/kv4.cuh). No device needed.
#pragma once
#include <algorithm>
#include <vector>

#include "abi_internal.cuh"
#include "kv4.cuh"

namespace alice {

inline int kv4_check_shape(const char* who, uint32_t pages, uint32_t page_tokens, uint32_t kv_heads, uint32_t dim) {
    if (!pages || !kv_heads) return alice_fail(ALICE_E_SHAPE, "%s: zero pages or heads", who);
    if (dim != 64 && dim != 128 && dim != 256) return alice_fail(ALICE_E_SHAPE, "%s: heads of %u; 64, 128 and 256 are built", who, dim);
    if (!page_tokens || page_tokens % KV4_TILE || page_tokens > 4096) return alice_fail(ALICE_E_SHAPE, "%s: pages of %u positions; a multiple of 16 up to 4096 is wanted", who, page_tokens);
    if (kv_heads > 65535) return alice_fail(ALICE_E_SHAPE, "%s: %u key / value heads", who, kv_heads);
    if ((uint64_t)pages * page_tokens > 0xffffffffull || (uint64_t)pages * kv_heads * (page_tokens / KV4_TILE) > 0xffffffffull)      // places are 32 bits
        return alice_fail(ALICE_E_SHAPE, "%s: more than 2^32 positions, or pieces of 16 positions of a head", who);
    return ALICE_OK;
}

// Jobs of 8 or 16 rows, or one for each sequence where it has fewer.
inline uint32_t kv4_max_jobs(uint32_t seqs, uint32_t tokens, uint32_t group, uint32_t dim) {
    const uint32_t rows = dim == 256 ? 8 : 16;
    return seqs + (uint32_t)(((uint64_t)tokens * group + rows - 1) / rows);
}

inline int kv4_check_limits(const char* who, uint32_t kv_heads, uint32_t dim, uint32_t heads, uint32_t max_seqs, uint32_t max_tokens, uint32_t max_pages) {
    if (!heads || heads % kv_heads) return alice_fail(ALICE_E_SHAPE, "%s: %u query heads over %u key / value heads", who, heads, kv_heads);
    if (!max_seqs || !max_tokens || !max_pages) return alice_fail(ALICE_E_SHAPE, "%s: zero sequences, tokens or pages", who);
    if ((uint64_t)max_tokens * heads * dim > 0x80000000ull) return alice_fail(ALICE_E_SHAPE, "%s: %u tokens of %u x %u are too many for one step", who, max_tokens, heads, dim);
    if ((uint64_t)max_seqs * max_pages > 0x10000000ull || max_seqs > 0x1000000u) return alice_fail(ALICE_E_SHAPE, "%s: %u sequences of %u pages", who, max_seqs, max_pages);
    return ALICE_OK;
}

inline int kv4_check_batch(const char* who, uint32_t pages, uint32_t page_tokens, uint32_t max_seqs, uint32_t max_tokens, uint32_t max_pages, uint32_t seqs,
                           const uint32_t* past, const uint32_t* tokens, const uint32_t* tables, uint32_t table_ld) {
    if (!page_tokens) return alice_fail(ALICE_E_SHAPE, "%s: pages of no positions", who);
    if (seqs > max_seqs) return alice_fail(ALICE_E_SHAPE, "%s: %u sequences, the batch was made for %u", who, seqs, max_seqs);
    if (seqs && (!past || !tokens || !tables)) return alice_fail(ALICE_E_INVALID, "%s: null argument", who);
    uint64_t total = 0;
    std::vector<uint32_t> written;
    for (uint32_t s = 0; s < seqs; s++) {
        const uint64_t end = (uint64_t)past[s] + tokens[s];
        total += tokens[s];
        if (total > max_tokens) return alice_fail(ALICE_E_SHAPE, "%s: more than the %u tokens the batch was made for", who, max_tokens);
        if (!tokens[s]) continue;                      // nothing of it is read or written
        if (end > 0x7fffffffull) return alice_fail(ALICE_E_SHAPE, "%s: sequence %u would have %llu positions", who, s, (unsigned long long)end);
        const uint64_t need = (end + page_tokens - 1) / page_tokens;
        if (need > max_pages || need > table_ld)
            return alice_fail(ALICE_E_SHAPE, "%s: sequence %u needs %llu pages; its table has %u, the batch was made for %u", who, s, (unsigned long long)need, table_ld, max_pages);
        const uint32_t* t = tables + (size_t)s * table_ld;
        for (uint32_t p = 0; p < need; p++) {
            if (t[p] >= pages) return alice_fail(ALICE_E_INVALID, "%s: sequence %u, page %u is %u of %u", who, s, p, t[p], pages);
            if (p >= past[s] / page_tokens) written.push_back(t[p]);
        }
    }
    std::sort(written.begin(), written.end());
    const auto twice = std::adjacent_find(written.begin(), written.end());
    if (twice != written.end()) return alice_fail(ALICE_E_INVALID, "%s: page %u would be written in two places", who, *twice);
    return ALICE_OK;
}

struct Kv4HostPlan {
    Kv4Head head{};
    std::vector<uint32_t> job_tile, table;
    std::vector<Kv4Token> token;
    std::vector<Kv4Job> job;
};

// Of checked arguments. Rows of one job see up to `last` keys, those of its last token. false: more than 2^31 tiles.
inline bool kv4_make_plan(Kv4HostPlan& h, uint32_t dim, uint32_t kv_heads, uint32_t page_tokens, uint32_t group, uint32_t seqs, const uint32_t* past, const uint32_t* tokens, const uint32_t* tables,
                          uint32_t table_ld, uint32_t max_pages) {
    uint32_t most = 0, total = 0;
    uint64_t tiles = 0;
    std::vector<Kv4Job> prompts;
    for (uint32_t s = 0; s < seqs; s++)
        if (!kv4_is_prompt(tokens[s] * group, dim)) most = std::max(most, tokens[s] * group);
    const uint32_t rows = kv4_job_rows(most, dim);
    h.table.assign((size_t)seqs * max_pages, 0);
    for (uint32_t s = 0; s < seqs; s++) {
        const uint32_t first = total;
        total += tokens[s];
        if (!tokens[s]) continue;
        const uint32_t end = past[s] + tokens[s], need = (end + page_tokens - 1) / page_tokens;
        const uint32_t* t = tables + (size_t)s * table_ld;
        std::copy(t, t + need, h.table.begin() + (size_t)s * max_pages);
        for (uint32_t p = 0; p < need; p++) h.head.top_page = std::max(h.head.top_page, t[p]);
        h.head.end = std::max(h.head.end, end);
        for (uint32_t i = 0; i < tokens[s]; i++) {
            const uint32_t at = past[s] + i;
            h.token.push_back({t[at / page_tokens] * kv_heads * (page_tokens / KV4_TILE) + at % page_tokens / KV4_TILE, at % KV4_TILE, at, 0});
        }
        if (kv4_is_prompt(tokens[s] * group, dim)) {
            for (uint32_t r = 0; r < tokens[s] * group; r += KV4_PROMPT_ROWS) prompts.push_back({s, r, std::min(KV4_PROMPT_ROWS, tokens[s] * group - r), first, past[s], 0, 0, 0});
            continue;
        }
        for (uint32_t r = 0; r < tokens[s] * group; r += rows) {
            const uint32_t n = std::min(rows, tokens[s] * group - r), last = past[s] + (r + n - 1) / group + 1, tile0 = (uint32_t)tiles;
            tiles += (last + KV4_TILE - 1) / KV4_TILE;
            h.job.push_back({s, r, n, first, past[s], tile0, (uint32_t)tiles, 0});
            h.job_tile.push_back(tile0);
        }
    }
    // prompts are started in this order: those that see most first
    auto keys = [&](const Kv4Job& j) { return j.past + (j.row + j.rows - 1) / group; };
    std::stable_sort(prompts.begin(), prompts.end(), [&](const Kv4Job& x, const Kv4Job& y) { return keys(x) > keys(y); });
    h.head.prompt_jobs = (uint32_t)prompts.size();
    h.head.seqs = seqs; h.head.tokens = total; h.head.jobs = (uint32_t)h.job.size(); h.head.rows = rows; h.head.tiles = (uint32_t)tiles;
    h.job.insert(h.job.begin(), prompts.begin(), prompts.end());
    return tiles <= 0x7fffffffull;
}

}  // namespace alice
