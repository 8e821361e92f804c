// batch_plan.cpp -- the work of one decode step over a paged cache (host code only).
#include "paged.h"

#include <algorithm>

namespace satori {

namespace {

// Pages that several members share are read once for all of them when that saves at least this many key
// reads (tokens times members but one); shorter runs stay with each member, because a segment of its own
// costs every one of its rows another partial record to merge (about half a microsecond of a step).
constexpr int kShareTokens = 256;

struct Builder {
    const PlanShape &shape;
    const std::vector<PlanMember> &members;
    Plan &plan;
    std::vector<int> order, row0;                      // members by table; first row of a member
    struct Place {
        int segment, index;
    };
    std::vector<std::vector<Place>> places;            // per member: its segments, and its first row's place in each

    void segment(int lo, int hi, int page0, int page1, int keys, bool causal)
    {
        PlanSegment s = {};
        const PlanMember &first = members[order[lo]];
        s.page_off = (int)plan.pages.size();
        s.keys = keys;
        s.start = page0 * shape.page_tokens;
        s.row_off = (int)plan.seg_rows.size();
        s.causal = causal;
        plan.pages.insert(plan.pages.end(), first.pages + page0, first.pages + page1);
        for (int i = lo; i < hi; ++i) {
            const int b = order[i];
            places[b].push_back({(int)plan.segments.size(), s.rows});
            for (int r = 0; r < members[b].rows; ++r) plan.seg_rows.push_back({row0[b] + r, plan.row_position[row0[b] + r]});
            s.rows += members[b].rows;
        }
        plan.segments.push_back(s);
    }

    // Members order[lo..hi) share their pages before `shared`, of which [from, shared) is in no segment yet.
    void walk(int lo, int hi, int from, int shared)
    {
        while (hi - lo > 1) {
            // New tokens lie in pages of their member alone, so the common part is full pages of old tokens.
            int common = shared;
            const PlanMember &a = members[order[lo]], &z = members[order[hi - 1]];
            while (common < a.n_pages && common < z.n_pages && a.pages[common] == z.pages[common]) ++common;
            if ((long long)(common - from) * shape.page_tokens * (hi - lo - 1) >= kShareTokens) {
                segment(lo, hi, from, common, (common - from) * shape.page_tokens, false);
                from = common;
            }
            // The next pages tell the groups apart (the members are sorted by table).
            int end = lo + 1;
            while (end < hi && common < members[order[lo]].n_pages && common < members[order[end]].n_pages &&
                   members[order[end]].pages[common] == members[order[lo]].pages[common])
                ++end;
            walk(lo, end, from, common);
            lo = end;
            shared = common;
        }
        if (hi - lo == 1) {
            const PlanMember &m = members[order[lo]];
            segment(lo, hi, from, m.n_pages, m.length - from * shape.page_tokens, true);
        }
    }
};

}  // namespace

void make_plan(const PlanShape &shape, const std::vector<PlanMember> &members, Plan &plan)
{
    const int n = (int)members.size();
    plan.row_position.clear();
    plan.row_page.clear();
    plan.row_slot.clear();
    plan.chain_off.assign(1, 0);
    plan.chain.clear();
    plan.seg_rows.clear();
    plan.pages.clear();
    plan.segments.clear();
    plan.tiles.clear();
    plan.slots.clear();
    plan.items.clear();
    plan.partials = 0;

    Builder b{shape, members, plan, {}, std::vector<int>((size_t)n), std::vector<std::vector<Builder::Place>>((size_t)n)};
    std::vector<int> alone;                            // members that share no segment
    for (int i = 0; i < n; ++i) {
        b.row0[i] = (int)plan.row_position.size();
        const PlanMember &m = members[i];
        for (int r = 0; r < m.rows; ++r) {
            const int pos = m.length - m.rows + r;
            plan.row_position.push_back(pos);
            plan.row_page.push_back(m.pages[pos / shape.page_tokens]);
            plan.row_slot.push_back(pos % shape.page_tokens);
        }
        // Rows that fill tiles of their own gain nothing from a shared segment (its keys are read once per tile
        // either way); with all their keys in one segment most of their tiles need no merge.
        if (m.rows * shape.group >= shape.tile_m)
            alone.push_back(i);
        else if (m.rows > 0)
            b.order.push_back(i);
    }
    std::stable_sort(b.order.begin(), b.order.end(), [&](int x, int y) {
        return std::lexicographical_compare(members[x].pages, members[x].pages + members[x].n_pages, members[y].pages,
                                            members[y].pages + members[y].n_pages);
    });
    const int sharing = (int)b.order.size();
    b.walk(0, sharing, 0, 0);
    b.order.insert(b.order.end(), alone.begin(), alone.end());
    for (int i = sharing; i < (int)b.order.size(); ++i) b.walk(i, i + 1, 0, 0);
    for (int i = 0; i < n; ++i)
        if (b.places[i].size() == 1) plan.segments[b.places[i][0].segment].sole = 1;

    long long total = 0;
    for (int s = 0; s < (int)plan.segments.size(); ++s) {
        PlanSegment &seg = plan.segments[s];
        seg.tile0 = (int)plan.tiles.size();
        const int m_all = seg.rows * shape.group;
        for (int m0 = 0; m0 < m_all; m0 += shape.tile_m) {
            PlanTile t = {s, m0, std::min(shape.tile_m, m_all - m0), seg.keys};
            if (seg.causal) {      // the tile's last row sees the most keys
                const PlanRow &row = plan.seg_rows[seg.row_off + (m0 + t.m - 1) / shape.group];
                t.keys = row.position + 1 - seg.start;
            }
            const int blocks = (t.keys + shape.block - 1) / shape.block;
            total += shape.kv_heads * shape.cost(t.m, blocks);
            plan.tiles.push_back(t);
        }
    }
    for (int i = 0; i < n; ++i)
        for (int r = 0; r < members[i].rows; ++r) {
            for (const Builder::Place &at : b.places[i])
                plan.chain.push_back({plan.segments[at.segment].tile0, at.index + r});
            plan.chain_off.push_back((int)plan.chain.size());
        }
    plan.slots.resize(plan.tiles.size() * (size_t)shape.kv_heads);

    // Deal the blocks to the CTAs in order: segment, KV head, tile, so that tiles that read the same keys
    // run at about the same time.
    // A CTA's border may cut a tile's keys into one more item, whose cost the budget has to hold.
    const long long budget = (total + shape.ctas - 1) / shape.ctas + shape.item_cost;
    plan.cta_off.assign(1, 0);
    long long room = budget;
    for (const PlanSegment &seg : plan.segments) {
        const int tiles = (seg.rows * shape.group + shape.tile_m - 1) / shape.tile_m;
        for (int h = 0; h < shape.kv_heads; ++h)
            for (int t = seg.tile0; t < seg.tile0 + tiles; ++t) {
                const PlanTile &tile = plan.tiles[t];
                const int cost = shape.block_cost(tile.m);
                const int blocks = (tile.keys + shape.block - 1) / shape.block;
                PlanSlots &slots = plan.slots[(size_t)t * shape.kv_heads + h];
                slots.first = plan.partials;
                int items = 0;
                for (int at = 0; at < blocks;) {
                    if (room < shape.item_cost + cost && (int)plan.cta_off.size() < shape.ctas) {
                        plan.cta_off.push_back((int)plan.items.size());
                        room += budget;
                        if (room < shape.item_cost + cost) room = shape.item_cost + cost;
                    }
                    long long take = (room - shape.item_cost) / cost;
                    if ((int)plan.cta_off.size() == shape.ctas) take = blocks - at;      // the last CTA takes the rest
                    take = std::max<long long>(1, std::min<long long>(take, blocks - at));
                    plan.items.push_back({seg.page_off, seg.row_off, tile.m0, tile.m, tile.keys, seg.causal ? seg.start : -1,
                                          h, at, (int)take, 0, 0, 0});
                    ++items;
                    at += (int)take;
                    room -= take == blocks ? shape.cost(tile.m, blocks) : take * cost + shape.item_cost;
                }
                // One item holds every key its rows can see: it writes the rows' outputs.  (Tiles that an
                // item works on in two halves of its blocks leave two records.)
                const bool halves = shape.slots_per_item > 1 && tile.m <= shape.solo_m && blocks > 1;
                const bool direct = seg.sole && items == 1 && !halves;
                for (size_t i = plan.items.size() - (size_t)items; i < plan.items.size(); ++i) {
                    PlanItem &item = plan.items[i];
                    item.direct = direct;
                    item.slot = direct ? -1 : plan.partials;
                    if (!direct) plan.partials += shape.slots_per_item;
                }
                slots.records = plan.partials - slots.first;
                slots.step = tile.m <= shape.solo_m ? 1 : shape.slots_per_item;
                if (direct) slots.first = -1;
            }
    }
    // Rows whose outputs come from several items: all of those with several segments, and of the others those in
    // a tile that was cut.
    plan.merges.clear();
    for (int i = 0; i < n; ++i)
        if (b.places[i].size() > 1)
            for (int r = 0; r < members[i].rows * shape.kv_heads; ++r) plan.merges.push_back(b.row0[i] * shape.kv_heads + r);
    for (const PlanSegment &seg : plan.segments) {
        if (!seg.sole) continue;
        const int tiles = (seg.rows * shape.group + shape.tile_m - 1) / shape.tile_m;
        for (int h = 0; h < shape.kv_heads; ++h)
            for (int t = seg.tile0, next = 0; t < seg.tile0 + tiles; ++t) {
                const PlanTile &tile = plan.tiles[t];
                if (plan.slots[(size_t)t * shape.kv_heads + h].first < 0) continue;
                const int end = (tile.m0 + tile.m - 1) / shape.group + 1;
                for (next = std::max(next, tile.m0 / shape.group); next < end; ++next)
                    plan.merges.push_back(plan.seg_rows[seg.row_off + next].row * shape.kv_heads + h);
            }
    }
    while ((int)plan.cta_off.size() <= shape.ctas) plan.cta_off.push_back((int)plan.items.size());
    plan.head.rows = (int)plan.row_position.size();
    plan.head.segments = (int)plan.segments.size();
    plan.head.items = (int)plan.items.size();
    plan.head.merges = (int)plan.merges.size();
}

}  // namespace satori
