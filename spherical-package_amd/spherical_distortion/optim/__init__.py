from .adamw import AdamW  # noqa: F401
