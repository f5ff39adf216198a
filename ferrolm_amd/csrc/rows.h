// The host-side plan of a set of rows over a paged cache (RowArgs): which
// tokens a row sees, how the attention is cut into items, which rows share a
// page's group of four tokens, and the children of each drafted row. Host code
// only.
#pragma once
#include "internal.h"

#include <algorithm>
#include <cstring>
#include <functional>
#include <vector>

namespace fg {

struct RowSeq {
    int n = 0, pos = 0;
    const uint32_t* blocks = nullptr;
    int n_blocks = 0;
    const int32_t* parents = nullptr;  // nullptr: a chain
};

// Longest tree: its masks hold a bit per row and token of the tree.
constexpr int kTreeRows = 4096;
// Workgroups that an attention launch is cut into at most, where it has not many more row groups: one a CU. More cost
// more in the merge than they gain; cut into even parts of each context, us of a tree over a long fp8 context in 256, 384, 512 workgroups 149, 196, 170,
// of trees of 16 sequences 70, 82, 79; one token over 32000 fp8 tokens (8 heads, workgroups of four waves) in
// 256, 512, 1024 21.9, 23.6, 33.4, eight chains of 5 17.5, 19.6, 25.0, one token of 16 sequences 22.7, 20.9, 24.9.
constexpr int kTreeWorkgroups = 256;

// A workgroup takes pieces of consecutive contexts until its share is full, so that ragged ones end together; a piece
// costs it this many pages besides its own (queries, the first loads, the join). us of a layer at 0 to 6000 cached
// tokens, 32 heads over 8 of 128 channels, with one piece of even length a workgroup and with 16, 32, 48 pages:
// trees of 22 tokens, 16 sequences 73, 67, 63, 68, 8 sequences 37, 40, 37, 37, 40 sequences 137, 103, 100, 108; one
// token of 16 sequences 26, 28, 24, 25; four prompt chunks of 300 128, 122, 114, 126.
constexpr int kPieceCost = 32;

struct RowPlan {
    int n_seqs = 0, rows = 0, n_wi = 0, n_items = 0, n_quads = 0, longest = 0, deepest = 0, most_rows = 0;
    uint32_t top_block = 0;  // the highest block id
    int64_t tokens = 0;  // cached tokens of all sequences, rows among them
    int qt = 1, rw = 1, pw = 1;
    int parts = 0;        // most parts of a row's context
    bool unused = false;  // some row is unused
    bool rooted = true;  // every sequence's rows hang on its first
    std::vector<int32_t> seqs, btab, items, mrec, quads, rpos, cstart, clist, parent;
    std::vector<uint16_t> masks;
    size_t o_seqs = 0, o_btab = 0, o_items = 0, o_mrec = 0, o_quads = 0, o_rpos = 0, o_masks = 0, o_cstart = 0,
           o_clist = 0, o_parent = 0, words = 0;
};

// Checked by the caller: n >= 0, parents[i] in [-2, i), a block for every position.
inline void plan_rows(RowPlan& P, const RowSeq* in, int n_seqs, int nh, int nkv, int hd, bool cached) {
    P = RowPlan();
    P.n_seqs = n_seqs;
    const int G = std::max(1, nh / nkv), qm = attn_qmax(hd), rps = std::max(1, qm / G);  // rows of a slot
    int most_q = 1, most_slots = 1;
    for (int s = 0; s < n_seqs; s++) {
        const RowSeq& q = in[s];
        const int row0 = P.rows, L = q.pos + q.n, page0 = q.pos / 16, pages = (L + 15) / 16;
        bool chain = true;
        for (int i = 0; q.parents && i < q.n; i++) chain = chain && q.parents[i] == i - 1;
        const int tp = chain ? 0 : pages - page0;
        const int32_t rec[kSeqWords] = {row0, q.n, q.pos, (int32_t)P.btab.size(), chain ? -1 : (int32_t)P.masks.size(),
                                        tp, (int32_t)P.tokens, L};
        P.seqs.insert(P.seqs.end(), rec, rec + kSeqWords);
        for (int b = 0; cached && b < pages; b++) {
            P.btab.push_back((int32_t)q.blocks[b]);
            P.top_block = std::max(P.top_block, q.blocks[b]);
        }
        // ancestors, depths, children
        const int aw = (q.n + 63) / 64;
        std::vector<uint64_t> anc(chain ? 0 : (size_t)q.n * aw, 0);
        std::vector<int> depth(q.n), kids(q.n + 1, 0);
        for (int i = 0; i < q.n; i++) {
            const int p = chain ? i - 1 : q.parents[i];
            depth[i] = p >= 0 ? depth[p] + 1 : 0;
            P.parent.push_back(std::max(p, -1));
            if (p >= 0) kids[p + 1]++;
            P.rooted = P.rooted && (i == 0 ? p == -1 : p != -1);
            P.unused = P.unused || p == -2;
            if (p != -2) P.deepest = std::max(P.deepest, depth[i] + 1);
            P.rpos.push_back(q.pos + depth[i]);
            if (chain || p == -2) continue;
            uint64_t* a = &anc[(size_t)i * aw];
            if (p >= 0) std::memcpy(a, &anc[(size_t)p * aw], aw * 8);
            a[i / 64] |= 1ull << (i % 64);
        }
        P.rooted = P.rooted && q.n > 0;
        P.most_rows = std::max(P.most_rows, q.n);
        for (int i = 0; i < q.n; i++) kids[i + 1] += kids[i];
        const int c0 = (int)P.clist.size();
        for (int i = 0; i < q.n; i++) P.cstart.push_back(c0 + kids[i]);
        P.clist.resize(c0 + kids[q.n]);
        for (int i = 0; i < q.n; i++) {
            const int p = chain ? i - 1 : q.parents[i];
            if (p >= 0) P.clist[c0 + kids[p]++] = row0 + i;
        }
        auto dead = [&](int i) { return !chain && q.parents[i] == -2; };
        for (int i = 0; !chain && i < q.n; i++)
            for (int x = 0; x < tp; x++) {
                uint32_t m = 0;
                for (int b = 0; b < 16 && !dead(i); b++) {
                    const int j = (page0 + x) * 16 + b - q.pos;
                    if (j < 0 || (j < q.n && (anc[(size_t)i * aw + j / 64] >> (j % 64) & 1))) m |= 1u << b;
                }
                P.masks.push_back((uint16_t)m);
            }
        // groups of four tokens
        for (int t = q.pos / 4 * 4; cached && t < L; t += 4) {
            int used = 0;
            for (int b = 0; b < 4; b++)
                if (t + b >= q.pos && t + b < L && !dead(t + b - q.pos)) used |= 1 << b;
            if (!used) continue;
            const int32_t qr[4] = {row0 + t - q.pos, (int32_t)q.blocks[t / 16], t % 16 / 4, used};
            P.quads.insert(P.quads.end(), qr, qr + 4);
        }
        if (cached) P.n_quads += (q.n + 6) / 4;  // at most, wherever the rows start
        for (int i = 0; i < q.n; i++) {
            const int32_t mr[4] = {i % rps * G, 0, 0, dead(i) ? 1 : 0};
            P.mrec.insert(P.mrec.end(), mr, mr + 4);
        }
        if (q.n) {
            most_q = std::max(most_q, std::min(q.n, rps) * G);
            most_slots = std::max(most_slots, (q.n + rps - 1) / rps);
        }
        P.longest = std::max(P.longest, L);
        P.rows += q.n;
        P.tokens += L;
    }
    P.cstart.push_back((int32_t)P.clist.size());
    P.qt = most_q <= 16 ? 1 : qm / 16;
    P.rw = std::min(4, most_slots);
    P.pw = P.rw <= 2 ? 4 : 2;
    // items: rw slots of rows x a part of the pages that they see
    auto group_pages = [&](const RowSeq& q, int r0) {
        const bool chain = P.seqs[(&q - in) * kSeqWords + 4] < 0;
        const int last = chain ? q.pos + std::min(q.n, r0 + P.rw * rps) : q.pos + q.n;
        return (last + 15) / 16;
    };
    struct Group {
        int seq, row0, pages, np, wi;
    };
    struct Piece {
        int group, p0, p1;
        bool head;  // the first of its workgroup
    };
    std::vector<Group> groups;
    for (int s = 0; cached && s < n_seqs; s++)
        for (int r0 = 0; r0 < in[s].n; r0 += P.rw * rps) groups.push_back(Group{s, r0, group_pages(in[s], r0), 0, 0});
    // Pieces of the groups' pages for workgroups of at most `budget` pages, a piece's fixed cost among them, in whole
    // rounds of a workgroup's waves; how many workgroups that takes.
    const int step = P.rw > 1 ? 4 * P.pw : 2 * P.pw, most_wgs = std::max(1, kTreeWorkgroups / std::max(1, nkv));
    // More groups than places: whole ones, a workgroup each, longest first, unless there are few and that leaves
    // places idle for long (with 4 groups a place, two chunks of 2047 took 306 us in shared pieces, 281 whole).
    // Workgroups of smaller heads run two on a CU, so theirs stay whole (trees of 16 sequences at 64 channels 50 us,
    // 68 in pieces).
    const int64_t n = (int64_t)groups.size();
    bool whole = n > 2 * most_wgs || (n > most_wgs && P.rw > 1 && hd < 128);
    std::vector<Piece> pieces;
    auto cut = [&](int budget, bool keep) {
        int wgs = 0, left = 0;
        for (int g = 0; g < (int)groups.size(); g++)
            for (int p = 0, n = groups[g].pages; p < n;) {
                const bool head = whole || left < kPieceCost + step;
                if (head) {
                    wgs++;
                    left = budget;
                }
                const int take = std::min({n - p, kPartPages, whole ? kPartPages : (left - kPieceCost) / step * step});
                if (keep) pieces.push_back(Piece{g, p, p + take, head});
                left -= kPieceCost + (take + step - 1) / step * step;
                p += take;
            }
        return wgs;
    };
    int64_t total = 0;
    for (const Group& g : groups) total += g.pages;
    int lo = kPieceCost + std::max(step, (int)(total / most_wgs)), hi = lo;
    while (!whole && cut(hi, false) > most_wgs) hi *= 2;
    while (!whole && lo < hi) {
        const int mid = (lo + hi) / 2;
        if (cut(mid, false) <= most_wgs)
            hi = mid;
        else
            lo = mid + 1;
    }
    if (!whole && n > most_wgs) {
        std::vector<int> len, place(most_wgs, 0);
        for (const Group& g : groups) len.push_back(g.pages);
        std::sort(len.begin(), len.end(), std::greater<int>());
        for (int p : len) *std::min_element(place.begin(), place.end()) += p + kPieceCost;
        whole = 4 * (int64_t)*std::max_element(place.begin(), place.end()) < 5 * (int64_t)hi;
    }
    cut(hi, true);
    for (const Piece& x : pieces) groups[x.group].np++;
    for (Group& g : groups) {
        const RowSeq& q = in[g.seq];
        const int slots = std::min(P.rw, (q.n - g.row0 + rps - 1) / rps);
        g.wi = P.n_wi;
        P.n_wi += g.np * slots;
        P.parts = std::max(P.parts, g.np);
        for (int i = g.row0; i < std::min(q.n, g.row0 + P.rw * rps); i++) {
            int32_t* mr = &P.mrec[(size_t)(P.seqs[g.seq * kSeqWords] + i) * 4];
            mr[1] = g.wi + (i - g.row0) / rps * g.np;
            mr[2] = g.np;
        }
    }
    // the launch's items, longest first where they are whole (what is left at the end is short), then those that
    // follow one in its workgroup; capacities in steps, so that the layout (and a captured step) lasts while contexts
    // grow
    std::vector<int> heads;
    for (int i = 0; i < (int)pieces.size(); i++)
        if (pieces[i].head) heads.push_back(i);
    if (whole)
        std::stable_sort(heads.begin(), heads.end(),
                         [&](int a, int b) { return pieces[a].p1 - pieces[a].p0 > pieces[b].p1 - pieces[b].p0; });
    P.n_items = ((int)heads.size() + 15) / 16 * 16;
    const size_t more = whole ? 0 : (std::max(groups.size(), pieces.size() - heads.size()) + 15) / 16 * 16;
    P.items.assign((P.n_items + more) * kItemWords, -1);
    std::vector<int> at(groups.size(), 0);  // parts of a group so far
    std::vector<int> part(pieces.size());
    for (int i = 0; i < (int)pieces.size(); i++) part[i] = at[pieces[i].group]++;
    int follow = P.n_items;
    auto emit = [&](int i, int slot, int next) {
        const Piece& x = pieces[i];
        const Group& g = groups[x.group];
        const int32_t* sr = &P.seqs[(size_t)g.seq * kSeqWords];
        const int slots = std::min(P.rw, (in[g.seq].n - g.row0 + rps - 1) / rps);
        const int32_t rec[kItemWords] = {g.seq, g.row0, x.p0, x.p1, g.wi + part[i], g.np, slots, g.np == 1,
                                         sr[0], sr[1], sr[2], sr[3], sr[4], sr[5], next, 0};
        std::copy(rec, rec + kItemWords, P.items.begin() + (size_t)slot * kItemWords);
    };
    for (int k = 0; k < (int)heads.size(); k++)
        for (int i = heads[k], slot = k;; i++) {
            const bool last = whole || i + 1 == (int)pieces.size() || pieces[i + 1].head;
            const int next = last ? -1 : follow++;
            emit(i, slot, next);
            if (last) break;
            slot = next;
        }
    auto place = [&](size_t n) {
        const size_t r = P.words;
        P.words += (n + 63) / 64 * 64;
        return r;
    };
    P.quads.resize((size_t)P.n_quads * 4, 0);
    P.n_wi = (P.n_wi + 15) / 16 * 16;
    P.btab.resize((P.btab.size() + 255) / 256 * 256, 0);
    P.o_seqs = place(P.seqs.size());
    P.o_btab = place(P.btab.size());
    P.o_items = place(P.items.size());
    P.o_mrec = place(P.mrec.size());
    P.o_quads = place(P.quads.size());
    P.o_rpos = place(P.rpos.size());
    P.o_masks = place((P.masks.size() + 1) / 2);
    P.o_cstart = place(P.cstart.size());
    P.o_clist = place(P.clist.size());
    P.o_parent = place(P.parent.size());
}

inline void pack_rows(const RowPlan& P, int32_t* h) {
    auto cp = [&](size_t off, const std::vector<int32_t>& v) {
        if (!v.empty()) std::memcpy(h + off, v.data(), v.size() * 4);
    };
    cp(P.o_seqs, P.seqs);
    cp(P.o_btab, P.btab);
    cp(P.o_items, P.items);
    cp(P.o_mrec, P.mrec);
    cp(P.o_quads, P.quads);
    cp(P.o_rpos, P.rpos);
    cp(P.o_cstart, P.cstart);
    cp(P.o_clist, P.clist);
    cp(P.o_parent, P.parent);
    if (!P.masks.empty()) std::memcpy(h + P.o_masks, P.masks.data(), P.masks.size() * 2);
}

inline RowArgs row_args(const RowPlan& P, const int32_t* d) {
    RowArgs a;
    a.seqs = d + P.o_seqs;
    a.btab = d + P.o_btab;
    a.items = d + P.o_items;
    a.mrec = d + P.o_mrec;
    a.quads = d + P.o_quads;
    a.rpos = d + P.o_rpos;
    a.masks = (const uint16_t*)(d + P.o_masks);
    a.cstart = d + P.o_cstart;
    a.clist = d + P.o_clist;
    a.parent = d + P.o_parent;
    a.n_seqs = P.n_seqs;
    a.rows = P.rows;
    a.n_items = P.n_items;
    a.n_wi = P.n_wi;
    a.n_quads = P.n_quads;
    a.longest = P.longest;
    a.most_rows = P.most_rows;
    a.unused = P.unused;
    a.parts = P.parts;
    a.qt = P.qt;
    a.rw = P.rw;
    a.pw = P.pw;
    return a;
}

}  // namespace fg
