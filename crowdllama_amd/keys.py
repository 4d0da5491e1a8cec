"""Peer identity keys (reference parity: internal/keys/keys.go:16-140).

Stable keyfile => stable PeerID across restarts, exactly like the
reference's libp2p ed25519 identities. The keyfile stores a 32-byte
ed25519 seed (0600, dir 0700); the peer id is derived from the ed25519
PUBLIC key (mesh/crypto.py peer_id_from_pub), so any peer shown the key
can verify it hashes to the claimed id — and the mesh handshake
(mesh/wire.py secure_open/secure_accept) proves possession of the private
half.
"""

from __future__ import annotations

import os
import threading
from dataclasses import dataclass

from .mesh import crypto

_KEY_LOCK = threading.Lock()

COMPONENTS = ("dht", "worker", "consumer")


@dataclass(frozen=True)
class Identity:
    seed: bytes     # ed25519 private seed (32 B)
    pub: bytes      # ed25519 public key (32 B)
    peer_id: str    # hash of pub (crypto.peer_id_from_pub)


def default_key_path(component: str) -> str:
    base = os.environ.get("CROWDLLAMA_KEY_DIR",
                          os.path.join(os.path.expanduser("~"),
                                       ".crowdllama-amd"))
    return os.path.join(base, f"{component}.key")


def get_or_create_key(path: str) -> bytes:
    """Load (or create, 0600) a 32-byte identity seed."""
    with _KEY_LOCK:
        if os.path.exists(path):
            with open(path, "rb") as f:
                seed = f.read()
            if len(seed) != 32:
                raise ValueError(f"corrupt key file {path}: {len(seed)} bytes")
            return seed
        os.makedirs(os.path.dirname(path) or ".", mode=0o700, exist_ok=True)
        seed = os.urandom(32)
        fd = os.open(path, os.O_WRONLY | os.O_CREAT | os.O_EXCL, 0o600)
        with os.fdopen(fd, "wb") as f:
            f.write(seed)
        return seed


def identity_from_seed(seed: bytes) -> Identity:
    pub = crypto.ed25519_public(seed)
    return Identity(seed=seed, pub=pub, peer_id=crypto.peer_id_from_pub(pub))


def load_identity(component: str, key_path: str | None = None) -> Identity:
    path = key_path or default_key_path(component)
    return identity_from_seed(get_or_create_key(path))


def peer_id_from_key(seed: bytes) -> str:
    """Peer id for a seed (derives the ed25519 public key)."""
    return identity_from_seed(seed).peer_id


def load_peer_id(component: str, key_path: str | None = None) -> tuple[str, bytes]:
    path = key_path or default_key_path(component)
    seed = get_or_create_key(path)
    return peer_id_from_key(seed), seed
