// The Newton-Schulz iteration's products of both parts of their operands.
#include "oz_newton_schulz_tiles.hpp"

template void ozn::launch_products<true>(hipStream_t, Phase, int, const Shapes&, const Ends&, const Pass&);
