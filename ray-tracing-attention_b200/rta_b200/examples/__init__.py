"""Small programs that use the package as a server would."""
