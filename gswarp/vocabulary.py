"""Alias of :mod:`gswarp_amd.vocabulary`."""

from gswarp_amd.vocabulary import *  # noqa: F401,F403
from gswarp_amd.vocabulary import __all__  # noqa: F401
