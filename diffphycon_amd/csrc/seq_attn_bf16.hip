// bf16 kernels of seq_attn.h
#include "seq_attn.h"

namespace dpc {
namespace seqattn {
int fwd_bf16(const Params& p, int grid, hipStream_t s) { return fwd<__bf16>(p, grid, s); }
int bwd_bf16(const Params& pq, int gq, const Params& pk, int gk, hipStream_t s) { return bwd<__bf16>(pq, gq, pk, gk, s); }
}  // namespace seqattn
}  // namespace dpc
