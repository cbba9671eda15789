// Host build of where a sequence's rows lie, for tests/test_kv4_rows.py.
#include "kv4_layout.h"

extern "C" void p_rows_seq(int rows, int width, int shift, int cu0, int cu1, int len, int* out) {
    tb::Kv4Rows r{nullptr, nullptr, nullptr, 1, width, rows};
    const tb::Kv4Seq s = tb::kv4_rows_seq(r, shift, cu0, cu1, len);
    out[0] = s.first; out[1] = s.n; out[2] = s.len; out[3] = s.pos0; out[4] = s.bad; out[5] = s.cut;
}
