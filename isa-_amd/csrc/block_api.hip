// Version and errors of libisa_block_hip.so.
#include "block_common.hpp"

namespace isa_block {
char* error_buffer() {
    static thread_local char text[kErrorBytes] = "";
    return text;
}
}  // namespace isa_block

extern "C" int isa_block_abi_version(void) { return ISA_BLOCK_ABI_VERSION; }
extern "C" const char* isa_block_last_error(void) { return isa_block::error_buffer(); }
