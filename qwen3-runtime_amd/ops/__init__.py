"""Device ops. ``HipOps`` is the only implementation the engine has; ``Int8Weight`` is a weight that its products take."""


def __getattr__(name):
    if name in ("HipOps", "OpsError"):
        from . import hip

        return getattr(hip, name)
    if name == "Int8Weight":
        from .int8 import Int8Weight

        return Int8Weight
    raise AttributeError(name)
