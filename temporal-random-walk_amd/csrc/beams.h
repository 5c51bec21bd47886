// beams.h -- implementations of beam search behind the C ABI.
#ifndef TRW_BEAMS_H
#define TRW_BEAMS_H

#include "operators.h"

namespace trw {
namespace ops {

uint64_t beam_select_workspace(const trw_beam_select_params& p);
void beam_select(const trw_beam_select_params& p, hipStream_t stream);
void beam_reorder(const trw_beam_reorder_params& p, hipStream_t stream);

}  // namespace ops
}  // namespace trw
#endif  // TRW_BEAMS_H
