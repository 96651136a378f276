// Format of K/V pages held in 4 bits, shared by the append (pool_q4.cu), the expansion
// (pool_q4.cu) and the decode (decode_q4.cu).
//
// A group is 64 dims of one token of one KV head.  With low = min x and s = bf16((max - low) / 15),
// a value is held as n = rint((x - low) / s) in 0..15 (0 when s is 0) and stands for n * s + low;
// low is a bf16 input value, so it is held exactly.  4.5 bits a value.  A group with a NaN or an
// infinity, or whose values span 2^60 or more (the decode multiplies scales by 2^64), is stored with
// s = low = NaN and reads back as NaN.
//
// A page of one KV head is one block of 18 * D bytes (1152 or 2304: a multiple of 128):
//   K codes  [token 16][c 4][group D/64][word 2]           32-bit words: 8 dims of a token each;
//            dim = 64 group + 16 c + 8 word + e, nibble e at bit 4 (e / 2) + 16 (e % 2)
//   V codes  [token / 8][g 8][c 4][group][word 2][token % 2] 16-bit pieces: 4 dims of a token each;
//            token = 8 (token / 8) + 2 c + token % 2, dim = 64 group + 8 g + 4 word + i, nibble i at bit 4 i
//   params   [token 16][K, V][group][scale, low]           bf16
// The orders are those in which a warp's lane 4 g + c feeds m16n8k16 fragments: every lane's codes
// of a page are whole 16-byte (D = 64: 8-byte) vectors, consecutive over the lanes, and
// (word >> 4 i) & 0x000F000F is one A-operand register's pair of codes.
#pragma once

#include "lf_common.cuh"

namespace lf {
namespace q4 {

constexpr int kPage = LF_PAGE_SIZE;
constexpr int kGroup = 64;
constexpr float kMaxSpan = 1152921504606846976.f;      // 2^60

template <int D>
struct Fmt {
    static_assert(D == 64 || D == 128, "head_dim 64 or 128");
    static constexpr int NG = D / kGroup;              // groups of a row
    static constexpr int kKBytes = 8 * D;              // K codes of a page
    static constexpr int kVOff = 8 * D;
    static constexpr int kParOff = 16 * D;
    static constexpr int kBlockBytes = 18 * D;
};

}  // namespace q4
}  // namespace lf
