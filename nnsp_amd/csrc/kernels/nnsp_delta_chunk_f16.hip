// nnsp_delta_chunk_f16.hip -- the gated delta rule in chunks, _Float16 tensors.
#include "nnsp_delta_chunk.h"

extern "C" int nnspk_launch_delta_chunk_f16(const nnsp_delta_args* a, void* stream) {
    return launch_chunk<_Float16>(*a, (hipStream_t)stream);
}
