"""Drop-in replacement of the reference's ``src.model`` package (same public names)."""
from .chassis import KVCache, WalshConfig
from .mhc import SinkhornKnopp, mHCResidualStream, mHCWalsh
from .paged import PagedKVCache

__all__ = ["WalshConfig", "KVCache", "mHCWalsh", "mHCResidualStream", "SinkhornKnopp", "PagedKVCache"]
