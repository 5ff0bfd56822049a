// Version and build information of libinet_policy.so (include/inet_policy.h).
#include "../../../include/inet_policy.h"

#ifndef INET_SRC_HASH
#define INET_SRC_HASH "unknown"
#endif

extern "C" {

int32_t inet_policy_abi_version(void) { return INET_POLICY_ABI_VERSION; }

const char* inet_policy_build_info(void) { return "libinet_policy gfx950 abi=1 src=" INET_SRC_HASH; }

}  // extern "C"
