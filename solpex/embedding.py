"""Alias: `solpex.embedding` -> `unet_amd.embedding` (the MI355X-native implementation)."""
from unet_amd.embedding import *  # noqa: F401,F403
from unet_amd import embedding as _impl

globals().update({k: v for k, v in vars(_impl).items() if not k.startswith("__")})
