// The dense-block operators of libontovae_hip.so (gfx950): 8-bit products, group norm with an activation, dropout.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "ontovae_ops.h"
#include "ontovae_dropout.h"
#include "ontovae_groupnorm.h"
#include "ontovae_int8.h"
