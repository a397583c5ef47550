// The declarations live in ck/b200/block_scale_ops.hpp.
#pragma once
#include "ck/b200/block_scale_ops.hpp"
