// nnsp_delta_chunk_f16.hip -- the gated delta rule in chunks, _Float16 tensors.
#include "nnsp_delta_chunk.h"

extern "C" int nnspk_launch_delta_chunk_f16(const nnsp_delta_args* a, int split, void* stream) {
    return launch_chunk<_Float16>(*a, split, (hipStream_t)stream);
}
extern "C" long long nnspk_delta_split_bytes_f16(const nnsp_delta_args* a) { return chunk_plan<_Float16>(*a).bytes(); }
