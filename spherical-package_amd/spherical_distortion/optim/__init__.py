from .adamw import AdamW  # noqa: F401
from .muon import Muon  # noqa: F401
