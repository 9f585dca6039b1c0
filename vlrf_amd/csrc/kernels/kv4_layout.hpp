// kv4_layout.hpp - where the 4-bit KV cache (VLRF_HIP_KV_Q4_0) keeps what; no HIP
// in it, so that the host and its tests use the same arithmetic.
//
// A head's row of d elements is nb = d / 32 GGUF Q4_0 blocks: an f16 scale and 32
// codes, byte j holding elements 2j (low nibble) and 2j + 1 (high nibble).  The
// device keeps codes and scales apart and orders both for the 16x16x32 matrix
// instruction, whose lane l supplies 8 of the 32 values that a product adds up, of
// row l % 16, as group l / 16; any order will do that both operands share.
//   K   scores add up a block's elements: group L takes elements 8L .. 8L + 7, a
//       32-bit word of the block.  A row's words stand as [L][block], so that a
//       lane's words of all blocks are one load.
//   V   outputs add up keys, 32 at a time: group L takes keys 4L .. 4L + 3 and
//       16 + 4L .. 16 + 4L + 3 (slots 0..3 and 4..7), the keys whose weights the
//       score products leave in its lanes.  Codes stand as [L][i][block][slot], the
//       byte of elements 2i and 2i + 1 of a block, one run of all blocks a lane.
//   scales of K and V: [L][block][slot] f16 for 32 keys, those of a lane's keys.
// Heads follow one another; max_seq is rounded up to whole groups of 32 keys.
#pragma once

#include <cstddef>

#if defined(__HIPCC__)
#define VH_KV4_FN __host__ __device__ inline
#else
#define VH_KV4_FN inline
#endif

namespace vlrf_hip {
namespace kv4 {

constexpr int kKeys = 32;   // keys of a group, and elements of a block

VH_KV4_FN size_t groups(int max_seq) { return ((size_t)max_seq + kKeys - 1) / kKeys; }
VH_KV4_FN size_t head_codes(int max_seq, int d) { return groups(max_seq) * kKeys * (d / 2); }    // bytes
VH_KV4_FN size_t head_scales(int max_seq, int d) { return groups(max_seq) * kKeys * (d / 32); }  // f16 values

VH_KV4_FN int lane_group(int key) { return (key % 16) / 4; }                    // L of a key (any key: its place in its 32)
VH_KV4_FN int slot(int key) { return key % 4 + 4 * ((key % kKeys) / 16); }
VH_KV4_FN int key_of(int L, int slot) { return 4 * L + slot % 4 + 16 * (slot / 4); }

// Within a head: byte offset of word L of a block of key t's K row, of the byte of
// elements 2i, 2i + 1 of a block of its V row, and index of the block's scale.
VH_KV4_FN size_t k_word(int t, int L, int block, int d) { return (size_t)t * (d / 2) + 4 * (L * (d / 32) + block); }
VH_KV4_FN size_t v_byte(int t, int i, int block, int d) {
    return (size_t)(t / kKeys) * (kKeys * (d / 2)) + 8 * ((lane_group(t) * 16 + i) * (d / 32) + block) + slot(t);
}
VH_KV4_FN size_t scale(int t, int block, int d) {
    return (size_t)(t / kKeys) * d + 8 * (lane_group(t) * (d / 32) + block) + slot(t);
}

}  // namespace kv4
}  // namespace vlrf_hip
