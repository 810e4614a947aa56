// How a row of logits is laid out over the CTAs, warps and steps of the
// sampling kernel, shared by the kernel, its launcher and their host check.
#pragma once

#include <stdint.h>

namespace walsh {

constexpr int kSampleMaxVocab = 1 << 18;
constexpr int kSampleThreads = 512, kSampleWarps = kSampleThreads / 32;

// CTAs per row: one when the rows alone occupy every SM (the barriers and scalar
// steps of a row are paid per CTA), else more while a thread still has eight
// tokens.  Rows of 50257 tokens: 64 in float32 with top-p 27.4 us on 4 CTAs each (47
// on one, 27.2 on two, 53 on 8), with top-k 50 21.2 (21.1, 16.2, 31.6); 256 in
// float32 with top-p 73.9 us on one, read again from L2, 70.3 on two, held; with
// top-k 50 31.7 and 43.0, plain 46 and 50; 256 in bf16 with top-p 56.9 on one, held,
// 70.8 on two.
inline int sample_cluster(int64_t rows, int vocab) {
  int cs = 1;
  while (cs < 8 && rows * cs < 148 && vocab / cs > kSampleThreads * 8) cs *= 2;
  return cs;
}

// 16-byte chunks (of vec elements) that a row covers which starts mis elements
// behind a chunk's boundary, of a CTA's contiguous part of them, and of a warp's part of n
constexpr int sample_chunks(int vocab, int mis, int vec) { return (mis + vocab + vec - 1) / vec; }
constexpr int sample_cta_chunks(int chunks, int cs) { return (chunks + cs - 1) / cs; }
constexpr int sample_warp_chunks(int n) { return n > kSampleWarps ? (n + kSampleWarps - 1) / kSampleWarps : 1; }
// steps of 32 chunks that n chunks take
constexpr int sample_steps(int n) { return (n + 31) / 32; }

// of the largest part of a warp: a row of float32 in one CTA, starting off a boundary
constexpr int kSampleSteps = sample_steps(sample_warp_chunks(sample_cta_chunks(sample_chunks(kSampleMaxVocab, 3, 4), 1)));

}  // namespace walsh
