"""Alias: `solpex.adapters` -> `unet_amd.adapters` (the MI355X-native implementation)."""
from unet_amd.adapters import *  # noqa: F401,F403
from unet_amd import adapters as _impl

globals().update({k: v for k, v in vars(_impl).items() if not k.startswith("__")})
