"""Elementwise optimizers for what the orthogonalized ones leave over (embeddings, the output layer, 1-D parameters):
``AdamW`` over many tensors at once with states in 32 or in 8 bits, its functional forms ``adamw_step`` and
``adamw_step_8bit``, and the block quantiser of the 8-bit states."""

from emerging_optimizers_b200.scalar_optimizers.adamw import *  # noqa: F401,F403
from emerging_optimizers_b200.scalar_optimizers.quantization import *  # noqa: F401,F403
