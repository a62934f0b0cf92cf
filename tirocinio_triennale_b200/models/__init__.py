from .gpt2 import GPT2, GPT2Config  # noqa: F401
from .adamw import AdamW  # noqa: F401
from .muon import Muon, muon_with_adamw  # noqa: F401
