// The paged key-value cache: what the engine keeps of it and the launchers of paged_cache.hip.
#pragma once
#include "common.h"

namespace mni {

// Device side.  Row (page, head, slot) of the pool holds head_dim values of one position, fp32 or int8 with a scale;
// table[sequence][i] is the page of positions i * page .. (i + 1) * page - 1; weight / pos (tracked caches) are kept
// per sequence, [sequence][head][row], because a page may be shared by sequences that weigh it differently.
constexpr int PAGED_TICKETS = 16384;
struct PagedPool {
    void *k, *v;
    float *kscale, *vscale;  // quantized only
    int32_t *table;
    float *weight;           // tracked only
    int32_t *pos;
    int32_t *tickets;        // [PAGED_TICKETS], zeros between launches: see attend_last
    int64_t max_pages, max_len;
    int heads, d, page, shift, quantized;
};
// Sequences of a launch, by value in its arguments: no upload, nothing to wait for.  Longer lists take several launches.
constexpr int PAGED_BATCH = 128;
struct PagedSeqs {
    int n;
    int32_t slot[PAGED_BATCH], len[PAGED_BATCH];
};
// Rows of k and v are read by stride (elements, the last extent contiguous).
struct PagedNew {
    const float *k, *v;
    int64_t k_seq, k_head, k_token, v_seq, v_head, v_token;
    int tokens;  // rows per (sequence, head) in the input; counts[i] of them are taken
};
// The sequences of an append and the pages that their new rows go to.  PagedAppend: one token each; page[i] is its new
// page, or -1 (the table has it).  PagedPrompt: several; pages from had[i] on are pages[first[i] ..] (had[i] = INT32_MAX:
// the table has them all).  The kernel enters the new ones into the table.
struct PagedAppend {
    static constexpr int MAX = PAGED_BATCH;
    int n;
    int32_t slot[MAX], len[MAX], count[MAX], seen[MAX];
    int32_t page[MAX];
};
constexpr int PAGED_PROMPT_PAGES = 704;
struct PagedPrompt {
    static constexpr int MAX = 32;
    int n;
    int32_t slot[MAX], len[MAX], count[MAX], seen[MAX], had[MAX], first[MAX];
    int32_t pages[PAGED_PROMPT_PAGES];
};
constexpr int PAGED_COPIES = 224;  // page copies of one launch
struct PagedCopies {
    int n;
    int64_t at[PAGED_COPIES];  // table entry that gets the new page
    int32_t from[PAGED_COPIES], to[PAGED_COPIES];
};

#ifdef __HIPCC__
__device__ __forceinline__ int64_t row_of(const PagedPool &p, int page, int head, int slot) {
    return ((int64_t)page * p.heads + head) * p.page + slot;
}
#endif

int k_paged_copy(const PagedPool &p, const PagedCopies &c);
int k_paged_append(const PagedPool &p, const PagedNew &in, const PagedAppend &a);
int k_paged_append(const PagedPool &p, const PagedNew &in, const PagedPrompt &a);
// q, out: [n, q_heads, d], contiguous
int k_paged_attend(const PagedPool &p, const PagedSeqs &s, const float *q, float *out, int q_heads, float scale, bool accumulate);
// w: [n, heads, width], contiguous
int k_paged_add_weights(const PagedPool &p, const PagedSeqs &s, const float *w, int64_t width);
// s.len: rows held; seen[i]: tokens seen
int k_paged_evict(const PagedPool &p, const PagedSeqs &s, const int32_t *seen, int budget, int recent);
// weights / positions: [n, heads, width]
int k_paged_track(const PagedPool &p, const PagedSeqs &s, float *weights, int32_t *positions, int64_t width);
int k_paged_read(const PagedPool &p, int32_t slot, int64_t len, float *k, float *v);
// table row and, when tracked, weights and positions of `len` rows
int k_paged_fork(const PagedPool &p, int32_t from, int32_t to, int64_t len);

}  // namespace mni
