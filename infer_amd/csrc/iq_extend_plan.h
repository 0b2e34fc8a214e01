// iq_extend_plan.h -- how the new tokens of sequences are split into units, a
// block of a sequence's tokens each (or `span` of them, for a 16-bit cache):
// arithmetic shared by extend_kernel (iq_kv8.hip), its host side and the CPU
// tests (plain C++: g++ compiles it on its own).  Also the way of threads
// through a block's older rows.
#pragma once

#include <algorithm>
#include <cstdint>

#include "iq_attn_plan.h"

namespace iq {

// A sequence's rows starts[b] .. starts[b + 1] as they count: inside the T that
// there are, none for a length outside the table, and no more than fit behind it.
struct NewTokens {
    int32_t row, count;
};
IQ_HD NewTokens new_tokens(int32_t s0, int32_t s1, int32_t len, int32_t T, int32_t cap) {
    s0 = s0 < 0 ? 0 : s0 > T ? T : s0;
    s1 = s1 > T ? T : s1;
    if (len < 0 || len >= cap || s1 <= s0) return {s0, 0};
    const int32_t n = s1 - s0, room = cap - len;
    return {s0, n < room ? n : room};
}

// How many units `count` tokens behind `len` touch.
IQ_HD uint32_t units_of(int32_t len, int32_t count, PageDiv span_div) {
    return count > 0 ? page_of(uint32_t(len + count - 1), span_div) - page_of(uint32_t(len), span_div) + 1 : 0;
}

// A run of new tokens inside one unit: its first, their number, the unit's first token.
struct Unit {
    int32_t tok, count, begin;
    int32_t row;  // of the first token's q, k, v
};
// The nth unit of a sequence; count 0 if it has none such.
IQ_HD Unit unit_at(uint32_t nth, int32_t len, NewTokens n, int32_t span, PageDiv span_div) {
    const int64_t begin = (int64_t(page_of(uint32_t(len < 0 ? 0 : len), span_div)) + nth) * span;
    const int64_t tok = begin < len ? len : begin, past = int64_t(len) + n.count, end = begin + span;
    Unit u{0, 0, 0, 0};
    if (len < 0 || tok >= past) return u;
    u.tok = int32_t(tok);
    u.count = int32_t((past < end ? past : end) - tok);
    u.begin = int32_t(begin);
    u.row = int32_t(n.row + (tok - len));
    return u;
}

// At most so many units of all sequences whose rows do not overlap: n tokens
// touch at most (n - 1) / span + 2.
inline int64_t max_units(int64_t T, int64_t B, int64_t span) { return T / span + 2 * std::min(B, T); }

// The 16-byte pieces of rows, `per` each, dealt to threads in turn.  Row and
// piece apart: a block may have 2^27 rows of 16 pieces and more, whose product
// passes 32 bits, while a row (below 0x7fff0000) with a step stays inside them.
struct Piece {
    int32_t row, col;
};
IQ_HD Piece piece_of(int32_t n, int32_t per) { return {n / per, n % per}; }
// The piece `step` (piece_of(threads, per)) behind p.
IQ_HD Piece piece_behind(Piece p, Piece step, int32_t per) {
    p.row += step.row;
    p.col += step.col;
    if (p.col >= per) {
        p.col -= per;
        p.row++;
    }
    return p;
}

}  // namespace iq
