"""Import path beside the reference's modules: ``from triturus.route import route``."""
from triturus_amd.route import Routes, route, route_grad  # noqa: F401
