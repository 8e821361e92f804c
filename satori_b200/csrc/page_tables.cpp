// page_tables.cpp -- page numbers, reference counts and sequences of a paged cache (host code only).
#include "paged.h"

#include <algorithm>

namespace satori {

namespace {
// A sequence id is its slot and a generation, so that the id of a removed sequence is not taken for the
// next one in its slot.
constexpr int kSlotBits = 20, kSlotMask = (1 << kSlotBits) - 1, kGenerations = 1 << 11;
}  // namespace

size_t type_size(int type)
{
    return type == SATORI_F32 ? 4 : type == SATORI_F16 || type == SATORI_BF16 ? 2 : 0;
}

int PageTables::top() const
{
    int n = pages();
    while (n > 0 && refs_[n - 1] == 0) --n;
    return n;
}

PageSequence *PageTables::find(int id)
{
    const int slot = id & kSlotMask;
    if (id < 0 || slot >= (int)sequences_.size()) return nullptr;
    PageSequence &s = sequences_[slot];
    return s.live && s.generation == id >> kSlotBits ? &s : nullptr;
}

bool PageTables::room_for_sequences(int n) const
{
    return (size_t)n <= unused_.size() + (size_t)(kSlotMask + 1) - sequences_.size();
}

int PageTables::add()
{
    int slot;
    if (!unused_.empty()) {
        slot = unused_.back();
        unused_.pop_back();
    } else {
        slot = (int)sequences_.size();
        sequences_.emplace_back();
        unused_.reserve(sequences_.size());            // remove() must not fail
    }
    PageSequence &s = sequences_[slot];
    s.live = true;
    s.length = 0;
    s.pages.clear();
    ++s.version;
    return s.generation << kSlotBits | slot;
}

int PageTables::take()
{
    while (refs_[hint_] != 0) ++hint_;
    refs_[hint_] = 1;
    --free_;
    return hint_++;
}

void PageTables::release(int page)
{
    if (--refs_[page] == 0) {
        ++free_;
        hint_ = std::min(hint_, page);
    }
}

void PageTables::remove(int id)
{
    PageSequence &s = sequences_[id & kSlotMask];
    for (int page : s.pages) release(page);
    s.pages.clear();
    s.length = 0;
    s.live = false;
    s.generation = (s.generation + 1) % kGenerations;
    ++s.version;
    unused_.push_back(id & kSlotMask);
}

void PageTables::compact(std::vector<int> &moves)
{
    const int live = pages() - free_;
    std::vector<int> to;
    moves.clear();
    moves.reserve(2 * (size_t)std::min(live, free_));
    int hole = 0;
    for (int page = live; page < pages(); ++page) {
        if (refs_[page] == 0) continue;
        while (refs_[hole] != 0) ++hole;
        if (to.empty()) to.assign((size_t)pages(), -1);
        to[page] = hole;
        moves.push_back(page);
        moves.push_back(hole);
        ++hole;
    }
    if (moves.empty()) return;
    for (size_t i = 0; i < moves.size(); i += 2) std::swap(refs_[moves[i]], refs_[moves[i + 1]]);
    for (PageSequence &s : sequences_) {
        bool changed = false;
        for (int &page : s.pages)
            if (to[page] >= 0) {
                page = to[page];
                changed = true;
            }
        if (changed) ++s.version;
    }
    hint_ = live;
}

}  // namespace satori
