// Attention whose rows see every token of their sequence: a decoder's rows over an encoder's states, or an encoder's own.
#include "attention_device.h"

namespace qproj {

hipError_t launch_attention_all(const AttentionJob &j, hipStream_t s) {
    if (rows_apart(j)) return launch_as(j, AllApartArgs{}, s);
    return launch_as(j, AllArgs{}, s);
}

}  // namespace qproj
