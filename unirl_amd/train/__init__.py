"""The optimizer step that follows a policy's backward."""

from .optim import AdamW

__all__ = ["AdamW"]
