from . import channel, instance, rms  # noqa: F401
