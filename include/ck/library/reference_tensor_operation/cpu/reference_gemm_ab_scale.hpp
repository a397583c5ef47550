// The definitions live in ck/b200/block_scale_reference.hpp.
#pragma once
#include "ck/b200/block_scale_reference.hpp"
