// C ABI of the log probabilities of given tokens (logprobs_kernel.h).  Declarations: include/ternaspmm.h.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>

#include "../../include/ternaspmm.h"
#include "host_util.h"
#include "logprobs_kernel.h"

using namespace terna;

namespace {

bool logprobs_shape_ok(int M, int V, int top)
{
    return M >= 1 && launch_fits(M, kLogprobThreads) && V >= 1 && V <= 1 << 19 && top >= 0 && top <= kLogprobMaxTop && top <= V;
}

// Workgroups of a row: enough that the rows together give every CU two, while each keeps two pieces a thread.
int logprobs_splits(int M, int V)
{
    int splits = 1;
    while (2 * splits <= kLogprobThreads && M * splits < 512 && V / (2 * splits) >= 4 * 2 * kLogprobThreads) splits *= 2;
    return splits;
}
// Blocks of 2^shift pieces that a row can have (its start need not be aligned).
int logprobs_blocks(int V, int fp32, int shift)
{
    const int pieces = V / (fp32 ? 4 : 8) + 2;
    return (pieces + (1 << shift) - 1) >> shift;
}
int logprobs_shift(int V, int fp32) { return logprobs_blocks(V, fp32, 4) <= kLogprobBlocks ? 4 : 6; }
static_assert(((1 << 19) / 4 + 2 + 63) / 64 <= kLogprobBlocks);

}  // namespace

extern "C" {

long long ternaspmm_token_logprobs_workspace_bytes(int M, int V, int fp32, int top)
{
    if (!logprobs_shape_ok(M, V, top)) return -1;
    const int splits = logprobs_splits(M, V);
    return splits == 1 ? 0 : 4ll * M * (3ll * splits + (top ? logprobs_blocks(V, fp32, logprobs_shift(V, fp32)) : 0));
}

int ternaspmm_token_logprobs(const void* logits, long long row, int fp32, const long long* targets, float* logprob, float* entropy, long long* top_ids,
                             float* top_logprobs, int top, void* workspace, int M, int V, terna_stream stream)
{
    if (!logprobs_shape_ok(M, V, top) || !logits || !entropy || (targets && !logprob) || (top && (!top_ids || !top_logprobs)) ||
        (reinterpret_cast<uintptr_t>(workspace) & 3) || (reinterpret_cast<uintptr_t>(logits) & (fp32 ? 3 : 1)) || row < 0)
        return -1;
    const int shift = logprobs_shift(V, fp32);
    LogprobArgs a{logits, targets, logprob, entropy, top_ids, top_logprobs, static_cast<float*>(workspace), row, M, V, top, workspace ? logprobs_splits(M, V) : 1,
                  logprobs_blocks(V, fp32, shift), shift};
    hipStream_t st = static_cast<hipStream_t>(stream);
    launch(fp32 ? terna_logprobs_kernel<float> : terna_logprobs_kernel<uint16_t>, dim3(M * a.splits), dim3(kLogprobThreads), 0, st, a);
    if (a.splits > 1) launch(fp32 ? terna_logprobs_merge_kernel<float> : terna_logprobs_merge_kernel<uint16_t>, dim3(M), dim3(kLogprobThreads), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) die("ternaspmm_token_logprobs", e, __LINE__);
    return 0;
}

}  // extern "C"
