// Host build of the cache's addressing rules, for tests/test_kv4_layout.py.
#include "kv4_layout.h"

extern "C" {
void p_seq(int rows, int width, int shift, int cu0, int cu1, int len, int* out) {
    tb::Kv4Rows r{nullptr, nullptr, nullptr, 1, width, rows};
    const tb::Kv4Seq s = tb::kv4_seq(r, shift, cu0, cu1, len);
    out[0] = s.first; out[1] = s.n; out[2] = s.len; out[3] = s.pos0; out[4] = s.bad;
}
int p_span(int pos0, int pos1, int len, int window, int sinks, int shift, int most, int* chunks) {
    const tb::Kv4Span s = tb::kv4_span(pos0, pos1, len, window, sinks, shift);
    const int n = tb::kv4_span_chunks(s);
    for (int i = 0; i < n && i < most; ++i) chunks[i] = tb::kv4_span_chunk(s, i);
    return n;
}
int p_sees(int pos, int tok, int window, int sinks) { return tb::kv4_sees(pos, tok, window, sinks); }
int p_slot_ok(int width, int slot) {
    tb::Kv4Rows r{nullptr, nullptr, nullptr, 1, width, 1};
    return tb::kv4_slot_ok(r, slot);
}
int p_page_ok(int pages, int page) {
    tb::Kv4Cache c{};
    c.num_pages = pages;
    return tb::kv4_page_ok(c, page);
}
unsigned long long p_offset(unsigned long long stride, int shift, int dim, int page, int head) {
    tb::Kv4Cache c{};
    c.page_stride = stride; c.page_shift = shift; c.dim = dim;
    return tb::kv4_block_offset(c, page, head);
}
}
