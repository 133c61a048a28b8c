// paged.h -- what the paged-cache sources share: tile plans, the argument block of the
// attention kernels, status bits (not part of the ABI).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "wisp_b200.h"

namespace wb {

// Status bits of a paged call's workspace.
enum { PG_BAD_PAGE = 1, PG_BAD_LENGTH = 2, PG_TIMEOUT = 8 };

// One row tile: consecutive tokens whose rows (token, query head of the kv head) go through
// the same cached positions.  Positions come in tiles of kPagedTile from 0: the item's list is
// [sink0, sink0 + n_sink) and then n_tiles - n_sink tiles from `first` on.
struct PagedItem {
    int tok0, ntok;    // tokens
    int seq;           // row of the page table
    int kv_lo, kv_hi;  // positions outside [kv_lo, kv_hi) belong to another item or to none
    int pos0;          // position of tok0; the tokens' positions follow one another when
    int pmin, pmax;    // `mixed` is 0, else each token's is looked up; their range
    int sink0, n_sink, first, n_tiles;
    int mixed;
    int alone;  // prefix mode: the sequence is in no group
};

// What the join kernels read about a piece (written by the attention CTA of its first head).
struct PagedSplit {
    int tok0, n_rows;  // the item that begins in the piece and ends after it (n_rows 0: none)
    int last;          // its last piece
    int item;
    int item0, item1;  // the items that begin in the piece
};
// Prefix mode: where the parts of a token's rows are.
struct PagedWhere {
    int first, last;  // pieces (the same: a whole item)
    int row0;         // the token's first row in the tile
    int alone;        // its own part: no shared prefix comes before it
    int plan, item;
};

// A plan covers the row tiles of one kind.  On the line of their work an item is `lead` units
// (what it costs to begin one) and its KV tiles of `grain` units each (one unit where items of at
// most kPagedHalf rows cost half); cum[i] units lie before item i.  The line is cut into at most
// `lanes` equal pieces of at least `grain` units; a KV tile belongs to the piece that its first
// unit lies in.  One CTA takes a piece for one block of query heads.
struct PagedPlan {
    int* n_items;
    int* bad;       // [lanes * heads + 1] status bits of each CTA, then of the plan
    int* item_off;  // [segments + 1] items before each sequence (or group)
    int* cum;       // [max_items + 1]
    PagedItem* items;
    float* part_o;      // [lanes][heads][2][rows][hd]: pieces of items that lanes share
    float* part_ml;     // [lanes][heads][2][rows][2]: see PagedArgs.full_ml
    PagedSplit* split;  // [lanes]
    PagedWhere* where;  // prefix mode: [n_tokens]
    int* redo;          // [max_items][heads], set for items to be worked out without tiles
    int lead, grain;
    int tpt;            // tokens of a row tile
    int rows;           // rows of a row tile
    int used_rows;      // of them at most so many are used
    int gpb, hblocks;   // query heads of a block, blocks of a kv head
    int lanes, heads;   // heads = kv heads * hblocks
    int max_items;
    int per_seg;           // the most row tiles of a segment
    int inlined;           // item i is tile i % per_seg of segment i / per_seg (some are empty), and
                           // the attention CTAs find cum themselves
    int used;              // the call has this plan
};

constexpr int kPagedTile = 64;  // positions of a KV tile
// Rows up to which both of the tensor-core kernel's row tiles work on one item.
constexpr int kPagedHalf = 128;

// Row tiles that an attention CTA counts by itself.
constexpr int kPagedInline = 160;

enum { PLAN_FEW = 0, PLAN_PREFIX = 1, PLAN_MANY = 2, PLANS = 3 };

struct PagedArgs {
    const void* q;
    void* out;
    float* lse;
    const void* k;
    const void* v;
    const int* q_start;
    const int* kv_len;
    const int* table;
    const int* groups;      // prefix mode: [n_groups + 1] first sequence of each group
    const int* prefix_len;  // [n_groups]
    float* full_o;          // prefix mode: [own, shared][n_tokens * n_heads][hd], whole items
    float* full_ml;  // the same [2]: M and the sum of weights 2^(score - M), score in log2 units
    int* status;
    int* all_status;  // the caller's word, or NULL
    size_t q_stride, out_stride, page_stride;
    int n_seq, n_tokens, n_groups, table_stride, table_width, n_pages, page_size, page_shift;
    int nh, nkv, group, hd, window, sinks;
    float scale_log2;
    unsigned long long wait_ns;  // how long a wait in a kernel may take
    // the sequences' own part, of few or of many rows (one of the two), and the shared prefixes
    PagedPlan plan[PLANS];
};

}  // namespace wb
