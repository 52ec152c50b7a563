// Launchers of castle_vocab.hip: cross entropy of hidden rows against a vocabulary, without its logits.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace castle {

enum { kMeanLoss = 0, kSumLoss = 1, kEachLoss = 2 };

struct VocabArgs {
  const void *x, *w;       // rows: x[r] = x + r * ld_x, D elements; w [V][ld_w]
  int64_t ld_x, ld_w;
  const int64_t* target;   // row r: target[(r / n) * target_ld + r % n]
  int64_t n, target_ld, ignore;
  int R, V, D, reduction;
};
// What a forward pass leaves for its backward pass, in this order, 256-byte aligned each: VocabHead, rank [R] (place of a row among those that count, or -1), by rank their targets [R],
// lse [R] and in 16 bits the rows themselves, of up to the next multiple of 64 elements (a launch less in the backward pass: 256 rows of 512 over 32000, forward and backward, 85 us,
// so 79).
struct VocabHead {
  int32_t count;
  float inv_count;
  uint32_t arrived;   // workgroups of the forward pass that have their sums there
};
int64_t vocab_state_bytes(int64_t R, int D, int es);
int64_t vocab_fwd_bytes(const VocabArgs& a, int es);
int64_t vocab_bwd_bytes(const VocabArgs& a, int es, bool need_x, bool need_w);
int launch_vocab_fwd(const VocabArgs& a, int dtype, void* loss, void* state, void* workspace, hipStream_t stream);
// dloss: one element of the type, or one for each row (kEachLoss); dx [R][D] and dw [V][D] contiguous, nullptr: not wanted
int launch_vocab_bwd(const VocabArgs& a, int dtype, const void* dloss, const void* state, void* dx, void* dw, void* workspace, hipStream_t stream);

}  // namespace castle
