// f32 kernels of seq_attn.h
#include "seq_attn.h"

namespace dpc {
namespace seqattn {
int fwd_f32(const Params& p, int grid, hipStream_t s) { return fwd<float>(p, grid, s); }
int bwd_f32(const Params& pq, int gq, const Params& pk, int gk, hipStream_t s) { return bwd<float>(pq, gq, pk, gk, s); }
}  // namespace seqattn
}  // namespace dpc
