// f16 kernels of seq_attn.h
#include "seq_attn.h"

namespace dpc {
namespace seqattn {
int fwd_f16(const Params& p, int grid, hipStream_t s) { return fwd<_Float16>(p, grid, s); }
int bwd_f16(const Params& pq, int gq, const Params& pk, int gk, hipStream_t s) { return bwd<_Float16>(pq, gq, pk, gk, s); }
}  // namespace seqattn
}  // namespace dpc
