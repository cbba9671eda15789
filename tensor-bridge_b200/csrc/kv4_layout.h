// kv4_layout.h -- where a token's keys and values lie in a paged cache of
// block-scaled FP4, and which pages and rows a call may touch.  Plain
// functions of integers for host and device: the kernels address the cache
// through them, and a CPU test walks them over bad pages and lengths.
//
// One page holds page_size tokens of every KV head; within a page the heads
// follow one another, and a head's block is one contiguous run
//   [K codes: page_size x D/2][K scales: page_size x D/16]
//   [V codes: page_size x D/2][V scales: page_size x D/16]
// of E2M1 codes (two per byte, the first value in the HIGH nibble) and E4M3
// scale bytes (one per 16 values): the layout of tb_decode_nvfp4, token by
// token.  A block of 16 tokens is 18 D bytes, so with page_size >= 16 every
// part starts on a 16-byte boundary and 16 tokens of any part can be moved by
// a bulk copy.
#pragma once

#include <cstddef>
#include <cstdint>

#if defined(__CUDACC__)
#define TB_KV4_HD __host__ __device__ __forceinline__
#else
#define TB_KV4_HD inline
#endif

namespace tb {

struct Kv4Cache {
    uint8_t* data;
    unsigned long long page_stride;  // bytes from one page to the next
    int num_pages;
    int page_shift;                  // log2(page_size)
    int heads;
    int dim;
    float k_scale, v_scale;
};

// The rows of a call: row cu[b] + i belongs to sequence b, and is its token
// number lens[b] - (cu[b+1] - cu[b]) + i.
struct Kv4Rows {
    const int* cu;
    const int* lens;
    const int* table;  // [batch x width] page numbers
    int batch;
    int width;
    int rows;          // rows that the caller's arrays hold
};

TB_KV4_HD uint32_t kv4_codes_bytes(const Kv4Cache& c) { return static_cast<uint32_t>(c.dim / 2) << c.page_shift; }
TB_KV4_HD uint32_t kv4_scales_bytes(const Kv4Cache& c) { return static_cast<uint32_t>(c.dim / 16) << c.page_shift; }
TB_KV4_HD uint32_t kv4_head_bytes(const Kv4Cache& c) { return 2u * (kv4_codes_bytes(c) + kv4_scales_bytes(c)); }

// Rows [first, first + n) of a sequence and its length.  Whatever cu and lens
// hold, first and n stay inside the caller's rows and len inside the table.
struct Kv4Seq {
    int first, n;
    int len;      // tokens of the sequence that the table has pages for
    int pos0;     // position of row `first`; negative where n > length
    bool bad;     // the length is negative or passes the table
    bool cut;     // cu decreases, or some of the rows lie outside the caller's
};

// The rows as clamped, the last of them the sequence's last token.
TB_KV4_HD Kv4Seq kv4_seq(const Kv4Rows& r, int page_shift, int cu0, int cu1, int len) {
    Kv4Seq s;
    s.first = cu0 < 0 ? 0 : cu0 > r.rows ? r.rows : cu0;
    const int end = cu1 < s.first ? s.first : cu1 > r.rows ? r.rows : cu1;
    s.n = end - s.first;
    const long long room = static_cast<long long>(r.width) << page_shift;
    s.bad = len < 0 || len > room;
    s.len = len < 0 ? 0 : len > room ? static_cast<int>(room) : len;
    s.pos0 = (len < 0 ? 0 : len) - s.n;
    s.cut = cu0 < 0 || cu1 < cu0 || cu1 > r.rows;
    return s;
}

// The same with each row at its own token: rows behind the caller's arrays are
// the sequence's last tokens, those inside come before them.  The position of
// row `first` is len - (cu1 - first); where that is below -2^31 + 4096 (then all
// rows inside are before the sequence) it is held there, so that what the
// kernels add and subtract stays in 32 bits.
TB_KV4_HD Kv4Seq kv4_rows_seq(const Kv4Rows& r, int page_shift, int cu0, int cu1, int len) {
    Kv4Seq s = kv4_seq(r, page_shift, cu0, cu1, len);
    if (s.n > 0) {
        const long long pos0 = (len < 0 ? 0ll : len) - (static_cast<long long>(cu1) - s.first);
        constexpr int kLeast = -0x7FFFFFFF - 1 + 4096;
        s.pos0 = pos0 < kLeast ? kLeast : static_cast<int>(pos0);
    }
    return s;
}

// True if table slot `slot` exists and holds the number of a page.
TB_KV4_HD bool kv4_slot_ok(const Kv4Rows& r, int slot) { return slot >= 0 && slot < r.width; }
TB_KV4_HD bool kv4_page_ok(const Kv4Cache& c, int page) { return page >= 0 && page < c.num_pages; }

// Byte offset of head `head`'s block in page `page`.
TB_KV4_HD unsigned long long kv4_block_offset(const Kv4Cache& c, int page, int head) {
    return static_cast<unsigned long long>(page) * c.page_stride +
           static_cast<unsigned long long>(head) * kv4_head_bytes(c);
}

// The tokens that rows at positions [pos0, pos0 + n) of a sequence can see,
// in chunks of 2^shift tokens: the chunks of the first `sinks` tokens, then
// those from the oldest token in the first row's window to the last row.
// `sink` chunks [0, sink), then [low, end); never empty for a sequence with
// rows (one chunk, all of it masked, where nothing is visible).
struct Kv4Span {
    int sink, low, end;
};

TB_KV4_HD Kv4Span kv4_span(int pos0, int pos1, int len, int window, int sinks, int shift) {
    Kv4Span s;
    int stop = pos1 + 1 < len ? pos1 + 1 : len;
    if (stop < 0) stop = 0;
    int first = 0;
    if (window > 0 && pos0 >= window) first = pos0 - window + 1;
    if (first > stop) first = stop;
    const int mask = (1 << shift) - 1;
    s.low = first >> shift;
    s.end = (stop >> shift) + ((stop & mask) != 0);
    const int nsink = sinks < 0 ? 0 : sinks;
    const int want = (nsink >> shift) + ((nsink & mask) != 0);
    s.sink = want < s.low ? want : s.low;
    if (s.end <= s.low && s.sink == 0) s.end = s.low + 1;
    return s;
}

TB_KV4_HD int kv4_span_chunks(const Kv4Span& s) { return s.sink + (s.end > s.low ? s.end - s.low : 0); }
TB_KV4_HD int kv4_span_chunk(const Kv4Span& s, int i) { return i < s.sink ? i : i - s.sink + s.low; }

// Whether the row at position pos sees token `tok`.
TB_KV4_HD bool kv4_sees(int pos, int tok, int window, int sinks) {
    return tok <= pos && (window <= 0 || pos - tok < window || tok < sinks);
}

}  // namespace tb
