// f32 kernels of seq_attn.h
#include "seq_attn.h"

namespace dpc {
namespace seqattn {
int fwd_f32(const Params& p, hipStream_t s) { return fwd<float>(p, s); }
int bwd_f32(const Params& pq, const Params& pk, hipStream_t s) { return bwd<float>(pq, pk, s); }
}  // namespace seqattn
}  // namespace dpc
