// What every call of an attention plan writes, from whatever host thread, has to be atomic (compiled only).
#include <type_traits>

#include "../darknet_b200/csrc/attention.h"

static_assert(std::is_same<decltype(dnb_attention_plan::kernel), std::atomic<const char *>>::value, "every forward writes it");
