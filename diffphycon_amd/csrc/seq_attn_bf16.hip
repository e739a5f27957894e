// bf16 kernels of seq_attn.h
#include "seq_attn.h"

namespace dpc {
namespace seqattn {
int fwd_bf16(const Params& p, hipStream_t s) { return fwd<__bf16>(p, s); }
int bwd_bf16(const Params& pq, const Params& pk, hipStream_t s) { return bwd<__bf16>(pq, pk, s); }
}  // namespace seqattn
}  // namespace dpc
