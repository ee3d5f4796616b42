// Attention whose rows see every token of their sequence: a decoder's rows over an encoder's states, or an encoder's own.
//
// The causal kernel's tiles with one mask less: only the last tile has an edge.  What bounds it: of 40 sequences of 90 to 6404 states (32 heads of 128 on 8) 46.7 us, 151 MB
// (3.3 TB/s; a copy moves 5.1), issue slots before the memory; of 4096 rows over 6404 states 1045 us, 430 Gflop, in 22 bits 1075: the rate of a large fp16 product of the
// library here (1.12 Pflop/s), at clocks that fall to 1.9 to 2.2 GHz; of five chunks of up to 187 rows over 1025 to 1601 60.5 us, the items' starts
// and ends.  One row over 1500 states, 20 heads of 64, 10.7.
#include "attention_device.h"

namespace qproj {

hipError_t launch_attention_all(const AttentionJob &j, hipStream_t s) {
    if (rows_apart(j, false)) return launch_as(j, AllApartArgs{}, s);
    return launch_as(j, AllArgs{}, s);
}

}  // namespace qproj
