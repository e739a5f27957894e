// f16 kernels of seq_attn.h
#include "seq_attn.h"

namespace dpc {
namespace seqattn {
int fwd_f16(const Params& p, hipStream_t s) { return fwd<_Float16>(p, s); }
int bwd_f16(const Params& pq, const Params& pk, hipStream_t s) { return bwd<_Float16>(pq, pk, s); }
}  // namespace seqattn
}  // namespace dpc
