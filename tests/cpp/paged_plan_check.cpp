// Checks and cuts one step over a paged cache, as lumen_page_batch_new does: reads
//   pages page h_kv d bf16 n_head causal rows keys slots stride n_seq  then per sequence  q kv first (stride page numbers)      (first -1: none given)
// and prints the status; if it is 0: tokens max_pos shared write_shared can_append, the slot and the position of every new token, then items
// (seq kvh row0 rows key0 key1 part) and joins (seq kvh row0 rows part splits), one per line.
#include <cstdio>

#include "paged_plan.cuh"

int main() {
    lumen::PagedGeom g;
    lumen::PagedShape shape;
    int bf16, n_head, causal, stride, n_seq;
    if (std::scanf("%d %d %d %d %d %d %d %d %d %d %d %d", &g.pages, &g.page, &g.h_kv, &g.d, &bf16, &n_head, &causal, &shape.rows, &shape.keys, &shape.slots, &stride, &n_seq) != 12)
        return 1;
    g.dtype = bf16 ? LUMEN_BF16 : LUMEN_F32;
    std::vector<int32_t> q, kv, first, tables;
    bool given = false;
    for (int s = 0; s < n_seq; ++s) {
        int a, b, c, t;
        if (std::scanf("%d %d %d", &a, &b, &c) != 3) return 1;
        q.push_back(a); kv.push_back(b); first.push_back(c);
        given = given || c != -1;
        for (int i = 0; i < stride; ++i) {
            if (std::scanf("%d", &t) != 1) return 1;
            tables.push_back(t);
        }
    }
    lumen::PagedPlan p;
    std::string why;
    const int rc = lumen::paged_layout(g, (size_t)n_head, (size_t)n_seq, q.data(), kv.data(), given ? first.data() : nullptr, tables.data(), (size_t)stride, causal, p, why);
    std::printf("%d\n", rc);
    if (rc) return std::fprintf(stderr, "%s\n", why.c_str()), 0;
    std::vector<int> live;
    for (int s = 0; s < n_seq; ++s)
        if (p.seqs[(size_t)s].q_len) live.push_back(s);
    lumen::paged_cut(p, g, shape, live);
    std::printf("%d %lld %d %d %d\n", p.tokens, p.max_pos, p.shared, p.write_shared, p.can_append);
    for (int t = 0; t < p.tokens; ++t) std::printf("token %d %d\n", p.tok_slot[(size_t)t], p.tok_pos[(size_t)t]);
    for (const auto &i : p.items) std::printf("item %d %d %d %d %d %d %d\n", i.seq, i.kvh, i.row0, i.rows, i.key0, i.key1, i.part);
    for (const auto &j : p.joins) std::printf("join %d %d %d %d %d %d\n", j.seq, j.kvh, j.row0, j.rows, j.part, j.splits);
    return 0;
}
