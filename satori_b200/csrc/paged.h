// paged.h -- host-side state of a paged key/value cache and of a decode batch's plan.
//
// Plain C++: the page tables and the planner run without a GPU (a cache created without a context keeps
// its tables only), so their rules are tested on the CPU.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <vector>

#include "../../include/satori_cuda.h"

namespace satori {

size_t type_size(int type);      // bytes of a satori_type, 0 when unknown

// One sequence: its pages in order and the tokens they hold.  Only a sequence's last page can be partly
// filled, and that page always belongs to it alone: every page that several sequences share is full, so
// appending never writes a shared page.
struct PageSequence {
    bool live = false;
    int generation = 0;
    int length = 0;
    unsigned version = 0;        // counts the changes of `pages` / `length`: a batch plan notices them
    std::vector<int> pages;
};

// Page numbers, reference counts and sequences.  The lowest free page is always taken first.
class PageTables {
  public:
    PageTables(int pages, int page_tokens) : page_tokens_(page_tokens), refs_((size_t)pages, 0), free_(pages) {}

    int pages() const { return (int)refs_.size(); }
    int page_tokens() const { return page_tokens_; }
    int free_pages() const { return free_; }
    int top() const;                                   // 1 + the highest page in use
    PageSequence *find(int id);                        // nullptr: no such sequence
    bool room_for_sequences(int n) const;
    int add();                                         // id of a new empty sequence
    int take();                                        // the lowest free page (the caller checked free_pages())
    void share(int page) { ++refs_[page]; }
    int refs(int page) const { return refs_[page]; }
    void release(int page);
    void remove(int id);
    // Moves the live pages numbered L and above (L = pages in use) to the free numbers below L, both in
    // ascending order; appends (from, to) to `moves` and rewrites every table.
    void compact(std::vector<int> &moves);

  private:
    int page_tokens_;
    std::vector<int> refs_;
    int free_, hint_ = 0;                              // no page below hint_ is free
    std::vector<PageSequence> sequences_;
    std::vector<int> unused_;                          // slots of removed sequences
};

// ------------------------------------------------------------------------------------------------ plan
// A batch's step: `rows` query rows (the new tokens of its members, in order).  The pages that several
// members have in common form segments; each member's own pages are its private segment.  A segment's keys
// are read for all its rows together.  Rows times the query heads of a KV head give the segment's M index,
// cut into tiles of `tile_m`; a tile's keys are cut into blocks and ranges of blocks are dealt to the
// resident CTAs as items of about equal cost.
struct PlanShape {
    int page_tokens, kv_heads, group;                  // group: query heads per KV head
    int tile_m, block;                                 // M rows per tile, keys per block
    int ctas;                                          // CTAs that the items are dealt to
    int solo_m;                                        // tiles of at most this many rows cost solo_cost per block
    int solo_cost, pair_cost, item_cost;               // cost of a block (small / large tile) and of an item
    int least_cost = 0;                                // of a whole tile's item, however short
    int more_cost = 0;                                 // added to pair_cost in proportion to the rows beyond tile_m / 2
    int slots_per_item;                                // partial records an item writes
    int block_cost(int m) const
    {
        const int half = tile_m / 2;
        return m <= solo_m ? solo_cost : m <= half ? pair_cost : pair_cost + more_cost * (m - half) / half;
    }
    long long cost(int m, long long blocks) const      // of a tile as one item
    {
        const long long c = blocks * block_cost(m) + item_cost;
        return c < least_cost ? least_cost : c;
    }
};

struct PlanMember {
    const int *pages;                                  // its table
    int n_pages;
    int length;                                        // tokens, the new ones included
    int rows;                                          // new tokens
};

struct PlanHeader {
    int rows, segments, items, merges;
};
struct PlanRow {
    int row, position;                                 // a segment's row: its number in the step and its position
};
struct PlanSegment {
    int page_off, keys, start;                         // first entry of plan.pages, keys, position of key 0
    int row_off, rows;                                 // entries of plan.seg_rows
    int tile0, causal, sole;                           // causal: private; sole: its rows have no other segment
};
struct PlanTile {
    int segment, m0, m, keys;                          // M range, keys some of its rows can see
};
// An item carries what the kernels need of its tile and segment, so that one load leads to the data.
struct alignas(16) PlanItem {
    int page_off, row_off, m0, m;
    int keys, start, kv_head, block0;                  // start: position of key 0, -1 when every row sees every key
    int blocks, slot, direct, pad;                     // slot: first partial record; direct: writes the output itself
};
struct alignas(16) PlanSlots {
    int first, records, step, pad;                     // partial records of (tile, KV head): every step-th holds a row;
};                                                     // first -1: the item wrote the output
struct PlanLink {
    int tile0, index;                                  // a segment's first tile, a row's place in the segment
};

struct Plan {
    PlanHeader head;
    std::vector<int> row_position, row_page, row_slot, chain_off, pages, cta_off;
    std::vector<int> merges;                           // row * kv_heads + KV head of what no single item writes
    std::vector<PlanRow> seg_rows;
    std::vector<PlanLink> chain;
    std::vector<PlanSegment> segments;
    std::vector<PlanTile> tiles;
    std::vector<PlanSlots> slots;                      // [tile][kv_head]
    std::vector<PlanItem> items;
    int partials = 0;                                  // partial records in all
};

void make_plan(const PlanShape &shape, const std::vector<PlanMember> &members, Plan &plan);

}  // namespace satori
