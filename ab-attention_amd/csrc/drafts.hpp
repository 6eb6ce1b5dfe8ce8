// Calls of the operators of drafted tokens: the tree, and its verification.
#pragma once

#include "layout.hpp"

namespace ab {

// The trees of `batch` sequences, whose new tokens are the packed rows offsets[b] ..
// offsets[b + 1]. parents: place among the sequence's new tokens, or a number that is
// no earlier place (a token that follows the cached ones).
struct TreeCall {
    const int32_t *parents, *lengths, *offsets;
    int32_t* positions;
    uint64_t* near;  // bit j: token 64 (i / 64) + j is on the line from the cached tokens to token i
    int32_t* above;  // the last token of that line before 64 (i / 64), or -1
    int32_t batch, tokens;
};

// Where a sequence's verification stands between its two kernels.
struct VerifyState {
    double less;     // drawn drafts: what is left of p is max(p - less q, 0)
    int32_t last;    // the last kept token's place
    int32_t next;    // the first place that has not been looked at
    int32_t counts;  // kept tokens
    int32_t gone;    // drafts turned down behind the last kept token
};

struct VerifyCall {
    const void *target, *draft;  // draft: or none
    int64_t target_row, draft_row;
    const void* tokens;
    bool wide;  // tokens and next are 64-bit integers
    const int32_t *parents, *offsets;
    const float* uniforms;
    int32_t *path, *counts;
    void* next;
    int32_t batch, rows, vocab, parts;
    int32_t type;  // 0 bf16, 1 fp16, 2 fp32
    VerifyState* state;  // [batch]
    double* sums;        // [batch][parts]
    int32_t times;       // a part is so many times kVerifyStep tokens of the vocabulary
};

int launch_tree(const TreeCall& call, hipStream_t stream);
int launch_verify(const VerifyCall& call, hipStream_t stream);
constexpr int kVerifyStep = 1024;   // tokens of the vocabulary that a wave takes at a time
constexpr int kVerifyParts = 256;   // of a vocabulary, at most

}  // namespace ab
